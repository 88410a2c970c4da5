"""A paged KV cache in 8 bits on the GPU: rows quantized as they are stored (equal to the plain model's), rows of any format read back,
attention over the pages (against 64 bits on the values that the pools stand for, to the bounds derived in paged_model.attention: the two
further products by scales are within its terms)."""
import numpy as np
import pytest

from mongoose_amd import engine as E
from tests import paged_model as P
from tests import paged_q8_model as Q
from tests.paged_q8_model import Case8
from tests.test_gpu_paged import Case, _ok, _synced, bufs, rt  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
U = P.U


# ---------------------------------------------------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------------------------------------------------
def _store(hip, bufs, heads, kv, hd, page, nPages, x, pad, slots, pos, cos, sin, K0, V0, rows=None):
    """(q, K pool, V pool) after a call on rows of one projection, K0 and V0 the pools' bytes before."""
    rows = len(x) if rows is None else rows
    ld = x.shape[1]
    dx, dK, dV, dq = bufs.up(x), bufs.up(K0), bufs.up(V0), bufs.up(np.full((len(x), heads * hd + pad), 7.25, np.float32))
    h = E.NewHIPPaged(hip, heads, kv, hd, page, nPages, 8, 1, max(rows, 1), 64)
    assert h is not None and h.PoolBytes() == K0.size, E.last_error()
    base = dx.DevicePtr()
    _ok(h.Store(base, base + heads * hd * 4, base + (heads + kv) * hd * 4, ld, ld, ld, dq, heads * hd + pad, dK, dV, bufs.up(slots), bufs.up(pos), rows, bufs.up(cos),
                bufs.up(sin), len(cos)))
    _synced()
    h.Close()
    assert np.array_equal(bufs.down(dx, x), x, equal_nan=True)
    return bufs.down(dq, np.zeros((len(x), heads * hd + pad), np.float32)), bufs.down(dK, K0), bufs.down(dV, V0)


def _turned(y, c, s):
    """Rows of heads [.., hd] turned, in 64 bits."""
    y = y.astype(np.float64)
    a, b = y[..., :y.shape[-1] // 2], y[..., y.shape[-1] // 2:]
    return np.concatenate((a * c - b * s, a * s + b * c), -1)


@pytest.mark.parametrize("heads,kv,hd,page,rows,pad", [(14, 2, 64, 16, 1, 0), (32, 8, 128, 8, 33, 0), (8, 8, 64, 32, 7, 12), (4, 1, 128, 128, 300, 4), (1, 1, 64, 8, 5, 0),
                                                       (30, 10, 128, 16, 9, 8), (128, 1, 64, 64, 3, 0), (6, 3, 64, 8, 130, 0)])
def test_store(hip, bufs, heads, kv, hd, page, rows, pad):
    """Equal to the model to the bit, in rows and scales; some rows have no position, one past the tables, no slot or a slot past the pools.
    Rows of every size, among them zeros, one element that is not zero, and ties."""
    print(f"store8 {heads}/{kv}/{hd} page={page} rows={rows}", flush=True)
    rng = np.random.default_rng(rows + hd)
    nPages, far, ld = -(-rows // page) + 3, 50, (heads + 2 * kv) * hd + pad
    n = nPages * page
    x = (rng.standard_normal((rows, ld)) * np.exp2(rng.integers(-60, 60, (rows, 1)))).astype(np.float32)
    if rows > 12:
        v = x[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
        v[7] = 0.0
        v[8] = 0.0
        v[8, 3] = -1e-3
        v[9] = np.float32(2.0 ** -9) * (rng.integers(-127, 127, kv * hd) + 0.5)          # all but the largest half-way
        v[9, ::hd] = 127 * 2.0 ** -9
        v[10] = np.float32(1e-44) * rng.integers(-3, 4, kv * hd)                         # the least fp32 numbers there are
        v[11] = np.float32(3e38) * rng.choice([-1, 1], kv * hd)
        x[12, heads * hd:(heads + kv) * hd] = 0.0
    slots = rng.permutation(n)[:rows].astype(np.int32)
    pos = rng.integers(0, far, rows).astype(np.int32)
    bad = {1: (0, -1), 2: (1, -1), 3: (0, n), 4: (1, far), 5: (1, -(1 << 31)), 6: (0, -(1 << 31))}
    for t, (which, value) in bad.items():
        if t < rows:
            (slots, pos)[which][t] = value
    ang = np.arange(far)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2.0 / hd)
    c, s = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qs, ss = (rng.integers(-128, 128, (n, kv, hd)).astype(np.int8) for _ in range(2)), (rng.standard_normal((n, kv)).astype(np.float32) for _ in range(2))
    (K0, V0), (Ks, Vs) = qs, ss
    got, K, V = _store(hip, bufs, heads, kv, hd, page, nPages, x, pad, slots, pos, c, s, Q.pool(K0, Ks, page), Q.pool(V0, Vs, page))
    assert (got[:, heads * hd:] == 7.25).all()
    for t in range(rows):
        if not 0 <= pos[t] < far:
            assert (got[t] == 7.25).all()
            continue
        cc, sn = c[pos[t]].astype(np.float64), s[pos[t]].astype(np.float64)
        q = x[t, :heads * hd].reshape(heads, hd)
        off = np.concatenate((2 * U * (np.abs(q[:, :hd // 2] * cc) + np.abs(q[:, hd // 2:] * sn)), 2 * U * (np.abs(q[:, :hd // 2] * sn) + np.abs(q[:, hd // 2:] * cc))), 1)
        assert (np.abs(got[t, :heads * hd].reshape(heads, hd) - _turned(q, cc, sn)) <= off).all(), t
        if 0 <= slots[t] < n:
            K0[slots[t]], Ks[slots[t]] = Q.held(_turned(x[t, heads * hd:(heads + kv) * hd].reshape(kv, hd), cc, sn).astype(np.float32))
            V0[slots[t]], Vs[slots[t]] = Q.held(x[t, (heads + kv) * hd:(heads + 2 * kv) * hd].reshape(kv, hd))
    for name, data, q, scale in (("K", K, K0, Ks), ("V", V, V0, Vs)):
        gq, gs = Q.from_pool(data, n, kv, hd, page)
        assert np.array_equal(gs, scale), (name, np.argwhere(gs != scale)[:5].tolist())
        assert np.array_equal(gq, q), (name, np.argwhere(gq != q)[:5].tolist(), gq[gq != q][:5], q[gq != q][:5])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_row_with_a_value_that_is_no_number(hip, bufs, hd, value):
    """Its scale is a NaN, so that it reads back as one; the other heads' rows are as ever."""
    x = np.random.default_rng(1).standard_normal((2, 9 * hd)).astype(np.float32)
    x[1, 3 * hd + 5] = value                # k of head 0
    x[1, 8 * hd + hd - 1] = value           # v of head 2
    one, zero = np.ones((1, hd // 2), np.float32), np.zeros((1, hd // 2), np.float32)
    blank = Q.pool(np.zeros((8, 3, hd), np.int8), np.zeros((8, 3), np.float32), 8)
    _, K, V = _store(hip, bufs, 3, 3, hd, 8, 1, x, 0, np.array([4, 2], np.int32), np.zeros(2, np.int32), one, zero, blank, blank)
    for data, first, odd in ((K, 3, 0), (V, 6, 2)):
        q, s = Q.from_pool(data, 8, 3, hd, 8)
        for t, slot in enumerate((4, 2)):
            wq, ws = Q.held(x[t, first * hd:(first + 3) * hd].reshape(3, hd))
            assert np.array_equal(s[slot], ws, equal_nan=True) and np.array_equal(q[slot], wq)
        assert np.isnan(s[2, odd]) and np.isfinite(np.delete(s[2], odd)).all()


# ---------------------------------------------------------------------------------------------------------------------
# load
# ---------------------------------------------------------------------------------------------------------------------
def _load(c, rows=None, pad=0, n=None, starts=None, lens=None, stream=None):
    """The rows read back, [bound, kv * hd + pad] each, 7.25 where nothing was written."""
    bound = c.bound if rows is None else rows
    width = c.kv * c.hd
    like = np.full((max(bound, 1), width + pad), 7.25, np.float32), np.full((max(bound, 1), width + 2 * pad), 7.25, np.float32)
    k, v = c.b.up(like[0]), c.b.up(like[1])
    _ok(c.h.Load(c.d["K"], c.d["V"], c.d["table"], c.b.up(starts) if starts is not None else c.d["rowStart"], c.b.up(lens) if lens is not None else c.d["lens"],
                 len(c.new) if n is None else n, bound, k, width + pad, v, width + 2 * pad, stream))
    _synced()
    return c.b.down(k, like[0]), c.b.down(v, like[1])


def _rows_want(c, name):
    """The last new[r] positions of every request, as fp32 (a product of a whole number and a scale is rounded once)."""
    rows = getattr(c, name)
    out = np.zeros((c.rows, c.kv * c.hd), np.float32)
    for r in range(len(c.new)):
        for t in range(int(c.new[r])):
            j = int(c.lens[r]) - int(c.new[r]) + t
            page = int(c.table[r, j // c.page]) if j >= 0 else -1
            if 0 <= page < c.nPages:
                out[c.rowStart[r] + t] = rows[page * c.page + j % c.page].astype(np.float32)
    return out


def _make(fmt, hip, bufs, heads, kv, hd, page, new, lens, **more):
    return Case8(hip, bufs, heads, kv, hd, page, new, lens, **more) if fmt == 8 else Case(hip, bufs, heads, kv, hd, fmt, page, new, lens, **more)


def _check_load(c, pad=0):
    c.upload()
    got = _load(c, pad=pad)
    width = c.kv * c.hd
    for name, g in zip("KV", got):
        assert (g[c.rows:] == 7.25).all() and (g[:, width:] == 7.25).all()
        assert np.array_equal(g[:c.rows, :width], _rows_want(c, name)), name


@pytest.mark.parametrize("fmt", [0, 1, 8])
@pytest.mark.parametrize("kv,hd,page,new,lens,pad", [
    (1, 64, 8, [1], [1], 0), (2, 64, 16, [1, 5, 40], [100, 5, 333], 4), (8, 128, 64, [200, 1], [200, 900], 0), (3, 128, 32, [0, 7, 0, 0, 33, 1, 0], [9, 70, 0, 3, 33, 64, 5], 8),
    (10, 128, 8, [3] * 70, [3 + 5 * r for r in range(70)], 0), (1, 128, 16, [1] * 4096, [1 + r % 60 for r in range(4096)], 0), (4, 64, 4096, [4000, 4097], [4100, 9000], 0)])
def test_load(hip, bufs, fmt, kv, hd, page, new, lens, pad):
    print(f"load fmt={fmt} {kv}/{hd} page={page} {len(new)} requests", flush=True)
    _check_load(_make(fmt, hip, bufs, kv, kv, hd, page, new, lens, seed=page, rowsMore=5), pad)


@pytest.mark.parametrize("fmt", [0, 1, 8])
def test_load_through_pages_that_are_gone(hip, bufs, fmt):
    """Zeros there; rows ahead of a request's first position (more rows than positions) are zeros too."""
    c = _make(fmt, hip, bufs, 2, 2, 64, 16, [100, 60, 50], [160, 60, 70], seed=3)
    c.table[0, [5, 7, 9]] = [-1, c.nPages, 0x7fffffff]
    c.table[1, :] = -(1 << 31)
    c.lens[2] = 30
    _check_load(c)


@pytest.mark.parametrize("fmt", [0, 1, 8])
def test_load_of_lengths_that_do_not_fit(hip, bufs, fmt):
    """Row starts that run backwards or pass the rows, lengths past the handle's: nothing is read or written outside."""
    c = _make(fmt, hip, bufs, 2, 2, 64, 16, [5, 1, 4], [60, 33, 60], seed=2)
    c.upload()
    for starts in ([7, 2, 9, -5], [-(1 << 31), 0x7fffffff, 3, 8], [0, 5, 6, 4000], [3, 4, 5, 6]):
        for lens in ([60, 33, 1 << 30], [-4, 33, 0x7fffffff], [-(1 << 31), 0, 10]):
            for g in _load(c, starts=np.array(starts, np.int32), lens=np.array(lens, np.int32)):
                assert np.isfinite(g).all()
    got = _load(c, starts=np.array([3, 4, 5, 6], np.int32))
    assert all((g[:3] == 7.25).all() and (g[6:] == 7.25).all() and (g[3:6] != 7.25).any(1).all() for g in got)


def test_load_of_nothing(hip, bufs):
    c = Case8(hip, bufs, 2, 2, 64, 8, [1], [9])
    _ok(c.h.Load(None, None, None, None, None, 0, 5, None, 0, None, 0))
    _ok(c.h.Load(None, None, None, None, None, 1, 0, None, 0, None, 0))


def test_load_refuses(hip, bufs):
    c = Case8(hip, bufs, 2, 2, 64, 8, [4], [9])
    c.upload()
    d, out = c.d, bufs.up(np.zeros((4, 256), np.float32))
    p = out.DevicePtr()

    def load(k=p, ldk=256, v=p + 512, ldv=256, K=d["K"], n=1, rows=4):
        return c.h.Load(K, d["V"], d["table"], d["rowStart"], d["lens"], n, rows, k, ldk, v, ldv)

    assert load() == 0
    for args, why in ((dict(n=2), "nReqs"), (dict(n=-1), "nReqs"), (dict(rows=-1), "rows"), (dict(k=p + 4), "16 bytes"), (dict(K=None), "16 bytes"), (dict(ldk=124), "smaller"),
                      (dict(ldv=258), "multiple of 4"), (dict(v=p + 256), "overlaps vOut"), (dict(v=p, ldv=128), "overlaps vOut"), (dict(k=d["K"]), "what is read"), (dict(v=d["table"]), "what is read")):
        assert load(**args) == -2 and why in E.last_error(), (args, E.last_error())
    _synced()


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 8, 128), (8, 8, 64), (6, 2, 128), (71, 1, 64), (40, 1, 128), (128, 1, 64)])
@pytest.mark.parametrize("page", [8, 16, 64, 128])
def test_single_tokens(hip, bufs, heads, kv, hd, page):
    lens = [1, 2, 7, 8, 9, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 1000, 2049]
    print(f"tokens8 {heads}/{kv}/{hd} page={page}", flush=True)
    Case8(hip, bufs, heads, kv, hd, page, [1] * len(lens), lens, seed=page).check()


@pytest.mark.parametrize("heads,kv,hd,n", [(14, 2, 64, 500), (32, 8, 128, 9001), (4, 1, 64, 20011), (3, 3, 128, 4097)])
def test_one_long_request(hip, bufs, heads, kv, hd, n):
    print(f"long8 {heads}/{kv}/{hd} n={n}", flush=True)
    Case8(hip, bufs, heads, kv, hd, 32, [1], [n], seed=n, rowsMore=2, ld=8).check()


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 8, 128), (4, 4, 64), (9, 3, 128)])
@pytest.mark.parametrize("page", [8, 16, 128])
def test_chunks_and_tokens(hip, bufs, heads, kv, hd, page):
    new, cached = [1, 5, 17, 33, 64, 1, 130, 2, 200], [300, 0, 40, 3, 64, 0, 70, 900, 129]
    print(f"chunks8 {heads}/{kv}/{hd} page={page}", flush=True)
    Case8(hip, bufs, heads, kv, hd, page, new, [a + b for a, b in zip(new, cached)], seed=page).check()


@pytest.mark.parametrize("heads,kv,hd,new,length", [(4, 1, 128, 700, 2300), (7, 1, 64, 513, 513), (2, 2, 64, 300, 1111), (8, 1, 128, 130, 900)])
def test_long_chunks(hip, bufs, heads, kv, hd, new, length):
    print(f"long chunk8 {heads}/{kv}/{hd} {new} of {length}", flush=True)
    Case8(hip, bufs, heads, kv, hd, 16, [new, 1], [length, 600], seed=new).check()


def test_requests_without_rows_or_length(hip, bufs):
    Case8(hip, bufs, 8, 2, 64, 16, [0, 1, 0, 0, 3, 0, 40, 0], [0, 1, 77, 0, 3, 16, 90, 0], rowsMore=37, ld=4).check()


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("window,prefix", [(1, False), (7, False), (64, False), (130, True), (1000, False), (0, True), (100000, False)])
def test_windows_and_prefixes(hip, bufs, heads, kv, hd, window, prefix):
    new, lens = [1, 1, 3, 70, 200, 40, 1], [900, 5, 64, 70, 450, 333, 300]
    print(f"window8 {window} prefix {prefix} {heads}/{kv}/{hd}", flush=True)
    Case8(hip, bufs, heads, kv, hd, 8, new, lens, seed=window).check(window=window, prefix=[3, 5, 62, 70, 260, 0, 300] if prefix else None)


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("cap,slopes,window,prefix", [(50.0, False, 0, False), (2.0, False, 0, False), (0.0, True, 0, False), (30.0, True, 90, True)])
def test_changed_scores(hip, bufs, heads, kv, hd, cap, slopes, window, prefix):
    new, lens = [1, 3, 70, 200, 1, 1], [900, 64, 70, 450, 2, 129]
    sl = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32) if slopes else None
    Case8(hip, bufs, heads, kv, hd, 32, new, lens, seed=int(cap), peak=4.0).check(cap=cap, slopes=sl, window=window, prefix=[3, 62, 70, 260, 1, 40] if prefix else None)


@pytest.mark.parametrize("scale", [1.0, 1e-3])
def test_scale(hip, bufs, scale):
    Case8(hip, bufs, 8, 2, 64, 16, [1, 90, 1], [700, 300, 33]).check(scale=scale)


@pytest.mark.parametrize("lo,hi", [(-12, 12), (-60, -20), (30, 50), (-90, 80)])
@pytest.mark.parametrize("new", [[1, 60, 1], [3, 1, 90]])
def test_positions_of_very_different_size(hip, bufs, lo, hi, new):
    """Scales that differ from position to position by up to 2^170: a weight is a probability times one, and neither a large one that comes
    late nor one that the row gives no weight may cost the others their digits."""
    c = Case8(hip, bufs, 8, 2, 128, 16, new, [600, 140, 400], seed=8, peak=2.0)
    size = np.exp2(c.rng.integers(lo, hi, (c.nPages * c.page, 1))).astype(np.float32)
    c.set_rows("V", np.float32(c.V) * size)
    c.check()


def test_rows_of_q_and_keys_of_any_size(hip, bufs):
    c = Case8(hip, bufs, 8, 2, 128, 16, [1, 60, 1], [600, 140, 40], seed=8)
    c.q *= np.exp2(c.rng.integers(-30, 2, (c.q.shape[0], 1))).astype(np.float32)
    c.set_rows("K", np.float32(c.K) * np.exp2(c.rng.integers(-8, 2, (c.nPages * c.page, 1))).astype(np.float32))
    c.check()


@pytest.mark.parametrize("new", [1, 3, 150])
def test_pages_that_are_gone_hide_their_positions(hip, bufs, new):
    c = Case8(hip, bufs, 8, 2, 128, 16, [new, new, new], [333, 200, 160], seed=new)
    c.table[0, [0, 3, 4, 5, 11]] = [-1, c.nPages, -(1 << 31), 0x7fffffff, -7]
    c.table[1, :] = -1
    c.table[2, 10 - -(-new // 16):10] = -1
    c.check()


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("name", ["K", "V"])
def test_rows_that_are_no_numbers_count_where_they_are_seen(hip, bufs, heads, kv, hd, name):
    """A K or V row of one KV head whose scale is a NaN reaches that head's results of the tokens that see its position, and no other."""
    for new, lens, window, bad in [([70, 3, 1], [70, 90, 300], 0, [(0, 41), (1, 88), (2, 7)]), ([40, 3, 1], [140, 90, 300], 20, [(0, 99), (0, 120), (1, 66), (1, 67), (2, 270), (2, 290)])]:
        c = Case8(hip, bufs, heads, kv, hd, 8, new, lens, seed=3)
        x = np.float32(getattr(c, name)).reshape(-1, kv, hd)
        for r, j in bad:
            x[c.where(r, j), 1] = np.nan
        c.set_rows(name, x)
        c.upload()
        c.plan(window)
        c.attend()
        _synced()
        got = c.result()[:c.rows].reshape(c.rows, heads, hd)
        odd = np.zeros((c.rows, heads), bool)
        for r, j in bad:
            i = c.lens[r] - c.new[r] + np.arange(c.new[r])
            odd[c.rowStart[r]:c.rowStart[r + 1], heads // kv:2 * (heads // kv)] |= ((j <= i) & ((window == 0) | (j > i - window)))[:, None]
        x = np.nan_to_num(getattr(c, name))
        setattr(c, name, x)
        want, bound = (a.reshape(c.rows, heads, hd) for a in c.want(window=window))
        assert np.isnan(got[odd]).all()
        assert (np.abs(got - want) <= bound)[~odd].all(), np.argwhere(~(np.abs(got - want) <= bound) & ~odd[..., None])[:5].tolist()
        c.h.Close()


@pytest.mark.parametrize("around", [1, 32])
@pytest.mark.parametrize("new,length,bad", [(1, 300, 299), (1, 300, 40), (3, 90, 88), (70, 70, 41), (70, 200, 160), (70, 200, 3)])
def test_a_row_that_is_no_number_under_no_weight(hip, bufs, new, length, bad, around):
    """A probability that fp32 holds as 0, times a scale that is a NaN: the rows that see the position have it, the others have not."""
    c = Case8(hip, bufs, 8, 2, 64, 8, [new, 70], [length, 75], seed=bad)
    c.q[:] = 1.0
    x = np.float32(c.K)
    for pos in range(bad // around * around, min(bad // around * around + around, length)):
        x[c.where(0, pos)] = -100.0                  # a score of -800, the others' within 10 of 0
    c.set_rows("K", x)
    x = np.float32(c.V)
    x[c.where(0, bad)] = np.nan
    c.set_rows("V", x)
    c.upload()
    c.plan()
    c.attend()
    _synced()
    got = c.result()[:c.rows]
    sees = length - new + np.arange(new) >= bad
    assert np.isnan(got[:new][sees]).all() and np.isfinite(got[:new][~sees]).all() and np.isfinite(got[new:]).all()
    c.h.Close()


def test_the_same_call_gives_the_same_bits(hip, bufs):
    c = Case8(hip, bufs, 32, 8, 128, 16, [1, 300, 1, 17], [5000, 900, 333, 2000], seed=9)
    c.upload()
    c.plan()
    outs = []
    for _ in range(4):
        c.b.put(c.d["out"], c.out0)
        c.attend()
        _synced()
        outs.append(c.result())
    assert all(np.array_equal(outs[0], o) for o in outs[1:])


def test_offsets_past_32_bits(hip, bufs):
    """A pool of 4.7 GB an array: rows and scales past 32 bits, attended to, stored and read back."""
    heads, kv, hd, page, nPages = 8, 8, 128, 64, 70000
    c = Case8(hip, bufs, heads, kv, hd, page, [1, 70], [300, 200], seed=6, spare=0)
    big = E.NewHIPPaged(hip, heads, kv, hd, page, nPages, 8, 2, 71, c.maxLen)
    size, slots, first = big.PoolBytes(), nPages * page, nPages - c.nPages
    assert size > 1 << 32
    pools = [E.lib.tw_gpu_alloc(size) for _ in range(2)]
    assert all(pools)
    c.upload()
    for p, name in zip(pools, "KV"):
        E.KZero(p, size)
        E.KSync()
        for a, at in ((c.q8[name], first * page * kv * hd), (Q.pool(c.q8[name], c.scales[name], page)[c.q8[name].size:], slots * kv * hd + first * page * kv * 4)):
            a = np.ascontiguousarray(a)
            E.lib.tw_gpu_upload(p + at, a.ctypes.data, a.nbytes)
    table = bufs.up(np.where((c.table >= 0) & (c.table < c.nPages), c.table + first, -1).astype(np.int32))
    d = c.d
    _ok(big.Plan(d["rowStart"], d["lens"], 2, 71))
    _ok(big.Attention(d["q"], c.ldq, pools[0], pools[1], table, d["out"], c.ldo))
    _synced()
    c.compare(c.result(), *c.want())
    # the second request's last row, stored anew and read back
    x = np.random.default_rng(1).standard_normal((1, 3 * kv * hd)).astype(np.float32)
    dx, qo, k, v = bufs.up(x), bufs.up(np.zeros((1, kv * hd), np.float32)), bufs.up(np.zeros((71, kv * hd), np.float32)), bufs.up(np.zeros((71, kv * hd), np.float32))
    p0, one, zero = dx.DevicePtr(), np.ones(64, np.float32), np.zeros(64, np.float32)
    slot = c.where(1, 199) + first * page
    _ok(big.Store(p0, p0 + 4096, p0 + 8192, x.shape[1], x.shape[1], x.shape[1], qo, kv * hd, pools[0], pools[1], bufs.up(np.array([slot], np.int32)),
                  bufs.up(np.zeros(1, np.int32)), 1, bufs.up(one), bufs.up(zero), 1))
    _ok(big.Load(pools[0], pools[1], table, d["rowStart"], d["lens"], 2, 71, k, kv * hd, v, kv * hd))
    _synced()
    for t, name, at in ((k, "K", kv * hd), (v, "V", 2 * kv * hd)):
        want = _rows_want(c, name)
        want[70] = Q.values(*Q.held(x[0, at:at + kv * hd].reshape(kv, hd))).astype(np.float32).reshape(-1)
        assert np.array_equal(bufs.down(t, want), want)
    big.Close()
    for p in pools:
        E.lib.tw_gpu_free(p)


def test_a_captured_step(hip, bufs, rt):
    """Tables, plan, store, attention and the new rows read back, captured once and replayed as the requests grow, on a stream of its own,
    against the same calls made eagerly on another handle and another copy of everything, and against the model."""
    heads, kv, hd, page, n, rows, maxLen, nPages = 8, 2, 64, 8, 5, 64, 200, 130
    rng = np.random.default_rng(12)
    ang = np.arange(maxLen)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2.0 / hd)
    cos, sin = bufs.up(np.cos(ang).astype(np.float32)), bufs.up(np.sin(ang).astype(np.float32))
    ld = (heads + 2 * kv) * hd
    blank = Q.pool(rng.integers(-128, 128, (nPages * page, kv, hd)).astype(np.int8), np.full((nPages * page, kv), np.nan, np.float32), page)

    def server():
        s = {"h": E.NewHIPPaged(hip, heads, kv, hd, page, nPages, 8, n, rows, maxLen)}
        for name, a in dict(new=np.zeros(n, np.int32), lens=np.zeros(n, np.int32), table=np.full((n, 25), -1, np.int32), ring=np.arange(nPages, dtype=np.int32)[::-1],
                            state=np.array([0, nPages], np.int32), rowStart=np.zeros(n + 1, np.int32), slots=np.zeros(rows, np.int32), pos=np.zeros(rows, np.int32),
                            counts=np.zeros(4, np.int32), x=np.zeros((rows, ld), np.float32), K=blank, V=blank, out=np.zeros((rows, heads * hd), np.float32),
                            k=np.zeros((rows, kv * hd), np.float32), v=np.zeros((rows, kv * hd), np.float32)).items():
            s[name] = bufs.up(a)
        return s

    def step(s, stream):
        x, h = s["x"].DevicePtr(), s["h"]
        _ok(h.Tables(s["new"], n, s["lens"], s["lens"], s["table"], s["ring"], s["state"], s["state"], rows, s["rowStart"], s["slots"], s["pos"], s["counts"], stream))
        _ok(h.Plan(s["rowStart"], s["lens"], n, rows, 0, None, stream))
        _ok(h.Store(x, x + heads * hd * 4, x + (heads + kv) * hd * 4, ld, ld, ld, x, ld, s["K"], s["V"], s["slots"], s["pos"], rows, cos, sin, maxLen, stream))
        _ok(h.Attention(x, ld, s["K"], s["V"], s["table"], s["out"], heads * hd, 0.0, 0.0, None, stream))
        _ok(h.Load(s["K"], s["V"], s["table"], s["rowStart"], s["lens"], n, rows, s["k"], kv * hd, s["v"], kv * hd, stream))

    a, b, stream = server(), server(), rt.stream()
    graph = rt.capture(stream, lambda: step(a, stream))
    lens = np.zeros(n, np.int64)
    for t in range(8):
        new = np.array([[30, 1, 0, 17, 5], [1, 1, 1, 1, 1], [1, 20, 1, -1, 0], [1, 1, 40, 0, 1], [-1, 1, 1, 9, 1], [60, 1, 1, 1, 1], [1, -1, 1, 1, 3], [1, 1, 1, 1, 1]][t], np.int32)
        x = rng.standard_normal((rows, ld)).astype(np.float32)
        for s in (a, b):
            bufs.put(s["new"], new)
            bufs.put(s["x"], x)
            for name, width in (("out", heads * hd), ("k", kv * hd), ("v", kv * hd)):
                bufs.put(s[name], np.full((rows, width), 7.25, np.float32))
        E.KSync()
        rt.replay(graph, stream)
        step(b, None)
        _synced()
        for name, width in (("out", heads * hd), ("k", kv * hd), ("v", kv * hd)):
            assert np.array_equal(*(bufs.down(s[name], np.zeros((rows, width), np.float32)) for s in (a, b))), (t, name)
        lens = np.where(new < 0, 0, lens + np.maximum(new, 0))
        start = np.concatenate(([0], np.cumsum(np.maximum(new, 0))))
        K, V = (Q.from_pool(bufs.down(a[w], blank), nPages * page, kv, hd, page) for w in ("K", "V"))
        table, slots = bufs.down(a["table"], np.zeros((n, 25), np.int32)), bufs.down(a["slots"], np.zeros(rows, np.int32))
        q = bufs.down(a["x"], x)[:, :heads * hd]
        got = bufs.down(a["out"], np.zeros((rows, heads * hd), np.float32))
        want, bound = P.attention(q, Q.values(*K).reshape(-1, kv * hd), Q.values(*V).reshape(-1, kv * hd), table, start, lens, page, heads // kv, hd)
        assert (np.abs(got[:start[-1]] - want) <= bound).all() and (got[start[-1]:] == 7.25).all()
        for name, (q8, scale), at in (("k", K, heads), ("v", V, heads + kv)):
            back = bufs.down(a[name], np.zeros((rows, kv * hd), np.float32))
            mine = slots[:start[-1]]
            assert np.array_equal(back[:start[-1]], Q.values(q8[mine], scale[mine]).astype(np.float32).reshape(-1, kv * hd)) and (back[start[-1]:] == 7.25).all()
            if name == "v":
                assert np.array_equal(q8[mine], Q.held(x[:start[-1], at * hd:(at + kv) * hd].reshape(-1, kv, hd))[0])
