"""What the calls on a paged KV cache compute, in plain numpy: block tables request by request, attention in 64 bits."""
import numpy as np

U = 2.0 ** -24          # half a step of fp32


def pages(x, page):
    return -(-x // page)


class Ring:
    """The free pages: `state` = (first, count) of a ring of n entries."""

    def __init__(self, entries, head, count):
        self.entries, self.head, self.count = np.array(entries, np.int32), head, count


def tables(new, lens, table, ring, page, maxLen, rows):
    """One step.  Returns the outputs of mg_paged_tables; table, ring and lens are copied, not changed."""
    n, nP = len(new), len(ring.entries)
    table, entries = table.copy(), ring.entries.copy()
    why, need, give, total = 0, 0, 0, 0
    for a, l in zip(new, lens):
        if l < 0 or l > maxLen or a < -1 or a > maxLen or (a > 0 and l + a > maxLen):
            why |= 4
            continue
        total += max(int(a), 0)
        if a < 0:
            give += pages(int(l), page)
        else:
            need += pages(int(l) + int(a), page) - pages(int(l), page)
    if not (0 <= ring.head < nP and 0 <= ring.count <= nP) or give > nP - min(max(ring.count, 0), nP):
        why |= 8
    if need > max(ring.count, 0):
        why |= 1
    if total > rows:
        why |= 2
    slots, positions = np.full(rows, -1, np.int32), np.full(rows, -1, np.int32)
    if why:
        return dict(lensOut=lens.copy(), table=table, ring=entries, ringState=np.array([ring.head, ring.count], np.int32),
                    rowStart=np.zeros(n + 1, np.int32), slots=slots, positions=positions, counts=np.array([0, 0, 0, why], np.int32))
    lensOut, rowStart, taken, given, at = lens.copy(), [0], 0, [], 0
    for r in range(n):
        l, a = int(lens[r]), int(new[r])
        for pos in range(l, l + max(a, 0)):
            if pos % page == 0:
                table[r, pos // page] = entries[(ring.head + taken) % nP]
                taken += 1
            p = int(table[r, pos // page])
            slots[at] = p * page + pos % page if 0 <= p < nP else -1
            positions[at] = pos
            at += 1
        if a < 0:
            given += table[r, :pages(l, page)].tolist()
        lensOut[r] = 0 if a < 0 else l + a
        rowStart.append(at)
    for i, p in enumerate(given):
        entries[(ring.head + ring.count + i) % nP] = p
    return dict(lensOut=lensOut, table=table, ring=entries,
                ringState=np.array([(ring.head + taken) % nP, ring.count - taken + len(given)], np.int32),
                rowStart=np.array(rowStart, np.int32), slots=slots, positions=positions,
                counts=np.array([at, taken, len(given), 0], np.int32))


def sees(i, j, length, window, prefix):
    return (j < length) & (((j <= i) & ((window == 0) | (j > i - window))) | (j < prefix))


def attention(q, K, V, table, rowStart, lens, page, group, hd, scale=0.0, cap=0.0, slopes=None, window=0, prefix=None):
    """(out, bound) in 64 bits, rows [rowStart[-1], heads * hd]; K, V [nPages * page, kvHeads * hd].

    bound: how far an fp32 computation may be off at each element.  With A the greatest scale * sum_d |q_d k_d| of the row, a
    score is off by at most (hd + 4) u A for its sum and its scaling and 8 u A for operands held to 22 bits, with a cap by
    another 8 u cap, with slopes by another 4 u (greatest bias); an exponential by that (twice: numerator and sum) and
    2^-20 for 2^x and the probabilities' two terms, a sum over n positions by (n / 8 + 64) u (lanes, tiles and splits
    add at most every eighth term to one register in a row), all relative to sum_j p_j |v_j|."""
    heads = q.shape[1] // hd
    nPages = K.shape[0] // page
    scale = scale or 1.0 / np.sqrt(hd)
    out = np.zeros((int(rowStart[-1]), q.shape[1]))
    bound = np.zeros_like(out)
    for r in range(len(lens)):
        r0, r1, n = int(rowStart[r]), int(rowStart[r + 1]), int(lens[r])
        if r1 == r0 or n == 0:
            continue
        j = np.arange(n)
        p = table[r][j // page].astype(np.int64)
        held = (p >= 0) & (p < nPages)
        j, at = j[held], (p * page + j % page)[held]
        i = (n - (r1 - r0) + np.arange(r1 - r0))[:, None]
        mask = sees(i, j, n, window, int(prefix[r]) if prefix is not None else 0)
        for h in range(heads):
            c = slice(h // group * hd, h // group * hd + hd)
            qh = q[r0:r1, h * hd:(h + 1) * hd].astype(np.float64)
            k, v = K[at][:, c].astype(np.float64), V[at][:, c].astype(np.float64)
            with np.errstate(all="ignore"):
                s = scale * (qh @ k.T)
                A = np.where(mask & np.isfinite(s), scale * (np.abs(qh) @ np.abs(k).T), 0).max(1, initial=0.0)
                off = (hd + 12) * U * A
                if cap:
                    s = cap * np.tanh(s / cap)
                    off = off + 8 * U * cap
                if slopes is not None:
                    bias = float(slopes[h]) * np.abs(i - j)
                    s = s - bias
                    off = off + 4 * U * np.where(mask, np.abs(bias), 0).max(1, initial=0.0)
                s = np.where(mask, s, -np.inf)
                m = s.max(1, initial=-np.inf, keepdims=True)
                e = np.where(mask, np.exp(s - np.where(np.isinf(m), 0, m)), 0)
                l = e.sum(1, keepdims=True)
                w = np.divide(e, l, out=np.zeros_like(e), where=l > 0)
                o, size = np.zeros((r1 - r0, hd)), np.zeros((r1 - r0, hd))
                fine = np.isfinite(v).all(1)
                o = w[:, fine] @ v[fine]
                size = w[:, fine] @ np.abs(v[fine])
                for b in np.nonzero(~fine)[0]:                 # a value that is no number counts where its position is seen
                    o += np.where(mask[:, b:b + 1], w[:, b:b + 1] * v[b], 0)
            out[r0:r1, h * hd:(h + 1) * hd] = o
            n8 = (len(j) / 8 + 64) * U
            bound[r0:r1, h * hd:(h + 1) * hd] = size * (2 * off[:, None] + 2.0 ** -20 + 2 * n8) + 1e-30
    return out, bound
