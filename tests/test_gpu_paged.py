"""Several requests out of one paged KV cache on the GPU: block tables and slot maps (equal to the plain model's), rotary
positions with rows stored by slot, attention over the pages (against 64 bits, to bounds derived in paged_model.attention)."""
import ctypes

import numpy as np
import pytest

from mongoose_amd import engine as E
from tests import paged_model as P

pytestmark = pytest.mark.gpu
U = P.U


class Runtime:
    """Streams and graphs of the HIP runtime that the library itself runs on."""

    def __init__(self):
        self.lib = ctypes.CDLL("libamdhip64.so.7")

    def call(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = ctypes.c_void_p()
        self.call("hipStreamCreateWithFlags", ctypes.byref(s), 1)
        return s

    def capture(self, stream, fn):
        g, ex = ctypes.c_void_p(), ctypes.c_void_p()
        self.call("hipStreamBeginCapture", stream, 0)
        fn()
        self.call("hipStreamEndCapture", stream, ctypes.byref(g))
        self.call("hipGraphInstantiate", ctypes.byref(ex), g, None, None, ctypes.c_size_t(0))
        return ex

    def replay(self, ex, stream):
        self.call("hipGraphLaunch", ex, stream)
        self.call("hipStreamSynchronize", stream)


@pytest.fixture(scope="module")
def rt(hip):
    return Runtime()


class Bufs:
    """Device buffers of one test."""

    def __init__(self, hip):
        self.hip, self.live = hip, []

    def up(self, a):
        a = np.ascontiguousarray(a)
        t = self.hip.UploadRawBytes(a if a.size else np.zeros(16, np.uint8))
        assert t is not None
        self.live.append(t)
        return t

    def down(self, t, like):
        like = np.asarray(like)
        return self.hip.DownloadRawBytes(t, like.nbytes).view(like.dtype).reshape(like.shape).copy()

    def put(self, t, a, at=0):
        a = np.ascontiguousarray(a)
        E.lib.tw_gpu_upload(t.DevicePtr() + at, a.ctypes.data, a.nbytes)

    def free(self):
        for t in self.live:
            t.Release()


@pytest.fixture
def bufs(hip):
    b = Bufs(hip)
    yield b
    b.free()


def _ok(rc):
    assert rc == 0, E.last_error()


def _synced():
    E.KSync()
    assert E.HIPCheck() == 0


# ---------------------------------------------------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------------------------------------------------
class Step:
    """A step's arrays on the device, and the call."""

    def __init__(self, hip, bufs, page, nPages, maxReqs, maxRows, maxLen):
        self.b, self.page, self.maxLen = bufs, page, maxLen
        self.h = E.NewHIPPaged(hip, 2, 1, 64, page, nPages, 0, maxReqs, maxRows, maxLen)
        assert self.h is not None, E.last_error()
        self.width = self.h.TableWidth()
        assert self.width == P.pages(maxLen, page)

    def run(self, new, lens, table, ring, rows, inPlace):
        b, n = self.b, len(new)
        want = P.tables(new, lens, table, ring, self.page, self.maxLen, rows)
        state = np.array([ring.head, ring.count], np.int32)
        d = {k: b.up(v) for k, v in dict(new=new, lens=lens, table=table, ring=ring.entries, state=state).items()}
        o = {k: b.up(np.full(want[k].shape, -99, np.int32)) for k in ("lensOut", "ringState", "rowStart", "slots", "positions", "counts")}
        if inPlace:
            o["lensOut"], o["ringState"] = d["lens"], d["state"]
        _ok(self.h.Tables(d["new"], n, d["lens"], o["lensOut"], d["table"], d["ring"], d["state"], o["ringState"], rows, o["rowStart"],
                          o["slots"], o["positions"], o["counts"]))
        _synced()
        got = {k: b.down(t, want[k]) for k, t in {**o, "table": d["table"], "ring": d["ring"]}.items()}
        for k in want:
            assert np.array_equal(got[k], want[k]), (k, np.argwhere(got[k] != want[k])[:4].tolist(), got["counts"].tolist())
        if not inPlace:
            assert np.array_equal(b.down(d["lens"], lens), lens) and np.array_equal(b.down(d["state"], state), state)
        return want


def _filled(rng, lens, page, width, nPages, free, head):
    """A table whose requests hold their pages (other entries: no pages), and the ring of `free` others."""
    order = rng.permutation(nPages).astype(np.int32)
    table, at = rng.integers(-(1 << 31), 0, (len(lens), width)).astype(np.int32), 0
    for r, l in enumerate(lens):
        k = P.pages(int(l), page)
        table[r, :k] = order[at:at + k]
        at += k
    entries = np.full(nPages, -5, np.int32)
    assert at + free <= nPages
    entries[(head + np.arange(free)) % nPages] = order[at:at + free]
    return table, P.Ring(entries, head, free)


@pytest.mark.parametrize("inPlace", [True, False])
@pytest.mark.parametrize("n,page,most,rows", [(1, 16, 1, 1), (3, 8, 5, 40), (64, 16, 1, 64), (65, 16, 1, 128), (100, 8, 40, 5000), (300, 128, 9, 1024), (300, 128, 9, 1500),
                                             (1000, 16, 3, 3000), (1025, 32, 1, 1025), (4096, 8, 2, 8200), (2, 64, 3000, 6001)])
def test_tables(hip, bufs, n, page, most, rows, inPlace):
    print(f"tables n={n} page={page} most={most} rows={rows} inPlace={inPlace}", flush=True)
    rng = np.random.default_rng(n + page)
    maxLen = 700 + most
    lens = rng.integers(0, 700, n).astype(np.int32)
    new = rng.integers(0, most + 1, n).astype(np.int32)
    new[rng.random(n) < 0.2] = -1
    lens[rng.random(n) < 0.1] = 0
    nPages = int(sum(P.pages(int(l) + max(int(a), 0), page) for l, a in zip(lens, new))) + 40
    free = nPages - int(sum(P.pages(int(l), page) for l in lens))
    step = Step(hip, bufs, page, nPages, n, rows, maxLen)
    table, ring = _filled(rng, lens, page, step.width, nPages, free, nPages - 3)       # the ring's end is crossed
    want = step.run(new, lens, table, ring, rows, inPlace)
    assert want["counts"][3] == (0 if np.maximum(new, 0).sum() <= rows else 2)


def test_tables_step_after_step(hip, bufs):
    """Requests come, grow, end and come again, through the state that the calls hand on; every page is in one place at any time."""
    rng = np.random.default_rng(3)
    n, page, nPages, maxLen, rows = 24, 8, 260, 120, 300
    step = Step(hip, bufs, page, nPages, n, rows, maxLen)
    lens = np.zeros(n, np.int32)
    table, ring = _filled(rng, lens, page, step.width, nPages, nPages, 17)
    for t in range(25):
        new = rng.integers(0, 12, n).astype(np.int32)
        new[(lens + new > maxLen) | ((rng.random(n) < 0.1) & (lens > 0))] = -1
        got = step.run(new, lens, table, ring, rows, bool(t % 2))
        assert got["counts"][3] == 0
        lens, table = got["lensOut"], got["table"]
        ring = P.Ring(got["ring"], int(got["ringState"][0]), int(got["ringState"][1]))
        held = [int(table[r, e]) for r in range(n) for e in range(P.pages(int(lens[r]), page))]
        free = [int(ring.entries[(ring.head + i) % nPages]) for i in range(ring.count)]
        assert sorted(held + free) == list(range(nPages))


@pytest.mark.parametrize("inPlace", [True, False])
@pytest.mark.parametrize("what,why", [("pages", 1), ("rows", 2), ("long", 4), ("negative", 4), ("new", 4), ("head", 8), ("count", 8), ("given", 8), ("huge", 7)])          # (69 requests of 57 pages and 900 rows, 1,000 pages free)
def test_tables_that_do_not_fit_change_nothing(hip, bufs, what, why, inPlace):
    rng = np.random.default_rng(5)
    n, page, rows, maxLen = 70, 16, 2000, 1000
    lens, new = rng.integers(1, 500, n).astype(np.int32), rng.integers(0, 20, n).astype(np.int32)
    step = Step(hip, bufs, page, 4000, n, rows, maxLen)
    table, ring = _filled(rng, lens, page, step.width, 4000, 1000, 3990)
    if what == "pages":
        ring.count = 3
    elif what == "rows":
        new[:] = 29
    elif what == "long":
        lens[69], new[69] = 990, 11
    elif what == "negative":
        lens[3] = -1
    elif what == "new":
        new[40] = -2
    elif what == "head":
        ring.head = 4000
    elif what == "count":
        ring.count = 4001
    elif what == "given":
        new[0], ring.count = -1, 4000
    elif what == "huge":
        new[:], lens[:], new[1] = 900, 0, 0x7fffffff
    got = step.run(new, lens, table, ring, rows, inPlace)
    assert got["counts"][3] == why


def test_tables_with_entries_that_are_no_page(hip, bufs):
    """A page that is gone (-1, or past the pool) leaves its rows without a slot; nothing is read or written through it."""
    lens, new = np.array([13, 16, 0], np.int32), np.array([4, 1, 3], np.int32)
    step = Step(hip, bufs, 8, 10, 3, 8, 32)
    table = np.array([[3, -1, -9, -9], [7, 10, -9, -9], [-9] * 4], np.int32)
    got = step.run(new, lens, table, P.Ring([1, 0x7fffffff, 2, 4, 5, 6, 8, 9, 0, 0], 0, 8), 8, False)
    assert got["slots"].tolist() == [-1, -1, -1, 8, -1, 16, 17, 18] and got["counts"][3] == 0


def test_tables_of_no_requests(hip, bufs):
    step = Step(hip, bufs, 16, 4, 4, 2048, 64)
    for rows in (0, 5, 2000):
        got = step.run(np.zeros(0, np.int32), np.zeros(0, np.int32), np.zeros((0, 4), np.int32), P.Ring([3, 2, 1, 0], 1, 4), rows, True)
        assert got["counts"].tolist() == [0, 0, 0, 0]


# ---------------------------------------------------------------------------------------------------------------------
# store
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,hd,half,rows,pad,inPlace", [(14, 2, 64, 0, 1, 0, False), (32, 8, 128, 1, 33, 0, False), (8, 8, 64, 1, 7, 12, True),
                                                               (4, 1, 128, 0, 300, 4, True), (1, 1, 64, 0, 5, 0, False), (30, 10, 128, 1, 9, 8, False)])
def test_store(hip, bufs, heads, kv, hd, half, rows, pad, inPlace):
    """Rows are columns of one projection; some rows have no position, one past the tables, no slot, or a slot past the pools.
    A turned element a c - b s is off by at most 2 u (|a c| + |b s|) (two products, one difference), a stored one by half a
    step of the cache's format more."""
    rng = np.random.default_rng(rows)
    page, nPages, far = 8, 60, 50
    ld = (heads + 2 * kv) * hd + pad
    x = rng.standard_normal((rows, ld)).astype(np.float32)
    kind = np.float16 if half else np.float32
    K0, V0 = (rng.standard_normal((nPages * page, kv * hd)).astype(kind) for _ in range(2))
    slots = rng.permutation(nPages * page)[:rows].astype(np.int32)
    pos = rng.integers(0, far, rows).astype(np.int32)
    bad = {1: (0, -1), 2: (1, -1), 3: (0, nPages * page), 4: (1, far), 5: (1, -(1 << 31)), 6: (0, -(1 << 31))}
    for t, (which, value) in bad.items():
        if t < rows:
            (slots, pos)[which][t] = value
    ang = np.arange(far)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2.0 / hd)
    c, s = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qOut0 = rng.standard_normal((rows, heads * hd + pad)).astype(np.float32)
    dx, dK, dV, dq = bufs.up(x), bufs.up(K0), bufs.up(V0), bufs.up(qOut0)
    h = E.NewHIPPaged(hip, heads, kv, hd, page, nPages, half, 1, rows, 64)
    base = dx.DevicePtr()
    out, ldo = (base, ld) if inPlace else (dq, heads * hd + pad)
    _ok(h.Store(base, base + heads * hd * 4, base + (heads + kv) * hd * 4, ld, ld, ld, out, ldo, dK, dV, bufs.up(slots), bufs.up(pos), rows, bufs.up(c), bufs.up(s), far))
    _synced()
    got = bufs.down(dx, x)[:, :heads * hd] if inPlace else bufs.down(dq, qOut0)[:, :heads * hd]
    K, V, xAfter = bufs.down(dK, K0), bufs.down(dV, V0), bufs.down(dx, x)
    if not inPlace:
        assert np.array_equal(xAfter, x) and np.array_equal(bufs.down(dq, qOut0)[:, heads * hd:], qOut0[:, heads * hd:])
    else:
        assert np.array_equal(xAfter[:, heads * hd:], x[:, heads * hd:])
    wantK, wantV, boundK = K0.astype(np.float64), V0.copy(), np.zeros(K0.shape)

    def turned(y, p):
        y = y.astype(np.float64).reshape(-1, 2, hd // 2)
        a, b, cc, ss = y[:, 0], y[:, 1], c[p].astype(np.float64), s[p].astype(np.float64)
        r = np.stack((a * cc - b * ss, a * ss + b * cc), 1).reshape(-1)
        return r, 2 * U * np.stack((abs(a * cc) + abs(b * ss), abs(a * ss) + abs(b * cc)), 1).reshape(-1)

    for t in range(rows):
        before = (x if inPlace else qOut0)[t, :heads * hd]
        if not 0 <= pos[t] < far:
            assert np.array_equal(got[t], before)
            continue
        r, b = turned(x[t, :heads * hd], pos[t])
        assert (np.abs(got[t] - r) <= b).all(), t
        if 0 <= slots[t] < nPages * page:
            r, b = turned(x[t, heads * hd:(heads + kv) * hd], pos[t])
            wantK[slots[t]], boundK[slots[t]] = r, b + (2.0 ** -11 * (np.abs(r) + b) + 2.0 ** -25 if half else 0)
            wantV[slots[t]] = x[t, (heads + kv) * hd:(heads + 2 * kv) * hd].astype(kind)
    assert (np.abs(K - wantK) <= boundK).all() and np.array_equal(V, wantV)
    h.Close()


def test_store_overflows_to_infinity_in_fp16(hip, bufs):
    x = np.full((1, 3 * 64), 7e4, np.float32)
    z = np.zeros((1, 32), np.float32)
    h = E.NewHIPPaged(hip, 1, 1, 64, 8, 1, 1, 1, 1, 1)
    K = bufs.up(np.zeros(512, np.float16))
    V = bufs.up(np.zeros(512, np.float16))
    d = bufs.up(x)
    one, q = bufs.up(z + 1), bufs.up(np.zeros(64, np.float32))
    p = d.DevicePtr()
    _ok(h.Store(p, p + 256, p + 512, 192, 192, 192, q, 64, K, V, bufs.up(np.zeros(1, np.int32)), bufs.up(np.zeros(1, np.int32)), 1, one, bufs.up(z), 1))
    _synced()
    assert np.isinf(bufs.down(K, np.zeros(64, np.float16))).all() and np.isinf(bufs.down(V, np.zeros(64, np.float16))).all()
    assert (bufs.down(q, np.zeros(64, np.float32)) == np.float32(7e4)).all()


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
class Case:
    """Requests of given new and total lengths over a shuffled pool.  What no request holds -- other pages, the ends of last pages,
    unused table entries -- is NaN or no page."""

    def __init__(self, hip, bufs, heads, kv, hd, half, page, new, lens, seed=0, spare=3, peak=1.5, rowsMore=0, ld=0):
        rng = np.random.default_rng(seed)
        self.rng, self.b, self.hip = rng, bufs, hip
        self.heads, self.kv, self.hd, self.half, self.page, self.group = heads, kv, hd, half, page, heads // kv
        self.new, self.lens = np.array(new, np.int32), np.array(lens, np.int32)
        self.kind = np.float16 if half else np.float32
        n, held = len(new), [P.pages(int(l), page) for l in lens]
        self.nPages, self.maxLen = sum(held) + spare, max(1, max(lens))
        self.width = P.pages(self.maxLen, page)
        order, at = rng.permutation(self.nPages).astype(np.int32), 0
        self.table = rng.choice([-1, -(1 << 31), self.nPages, 0x7fffffff], (n, self.width)).astype(np.int32)
        self.K, self.V = (np.full((self.nPages * page, kv * hd), np.nan, self.kind) for _ in range(2))
        for r in range(n):
            self.table[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
            j = np.arange(lens[r])
            where = self.table[r][j // page] * page + j % page
            self.K[where], self.V[where] = (rng.standard_normal((lens[r], kv * hd)).astype(self.kind) for _ in range(2))
        self.rowStart = np.concatenate(([0], np.cumsum(self.new))).astype(np.int32)
        self.rows = int(self.rowStart[-1])
        self.bound, self.ldq, self.ldo = self.rows + rowsMore, heads * hd + ld, heads * hd + 2 * ld
        self.q = (peak * rng.standard_normal((max(self.bound, 1), self.ldq))).astype(np.float32)
        self.h = E.NewHIPPaged(hip, heads, kv, hd, page, self.nPages, half, max(n, 1), max(self.bound, 1), self.maxLen)
        assert self.h is not None, E.last_error()

    def where(self, r, j):
        """Row of the pools that holds position j of request r."""
        return int(self.table[r, j // self.page]) * self.page + j % self.page

    def upload(self):
        up = self.b.up
        self.out0 = np.full((max(self.bound, 1), self.ldo), 7.25, np.float32)
        self.d = {"q": up(self.q), "K": up(self.K), "V": up(self.V), "table": up(self.table), "rowStart": up(self.rowStart), "lens": up(self.lens), "out": up(self.out0)}

    def plan(self, window=0, prefix=None, stream=None):
        self.dprefix = self.b.up(np.array(prefix, np.int32)) if prefix is not None else None
        _ok(self.h.Plan(self.d["rowStart"], self.d["lens"], len(self.new), self.bound, window, self.dprefix, stream))

    def attend(self, scale=0.0, cap=0.0, slopes=None, stream=None):
        d = self.d
        self.dslopes = self.b.up(slopes) if slopes is not None else None
        _ok(self.h.Attention(d["q"], self.ldq, d["K"], d["V"], d["table"], d["out"], self.ldo, scale, cap, self.dslopes, stream))

    def result(self):
        return self.b.down(self.d["out"], self.out0)

    def want(self, scale=0.0, cap=0.0, slopes=None, window=0, prefix=None):
        return P.attention(self.q[:, :self.heads * self.hd], self.K, self.V, self.table, self.rowStart, self.lens, self.page, self.group, self.hd, scale, cap, slopes,
                           window, prefix)

    def compare(self, got, want, bound):
        width = self.heads * self.hd
        assert (got[self.rows:] == 7.25).all() and (got[:, width:] == 7.25).all(), "written outside its rows"
        g = got[:self.rows, :width].astype(np.float64)
        fine = np.isfinite(want)
        assert np.array_equal(fine, np.isfinite(g)), np.argwhere(fine != np.isfinite(g))[:5].tolist()
        off = np.abs(g[fine] - want[fine])
        worst = float((off / bound[fine]).max(initial=0.0))
        print(f"  worst {worst:.3f} of the bound, largest difference {off.max(initial=0.0):.2e}", flush=True)
        assert worst <= 1.0

    def check(self, scale=0.0, cap=0.0, slopes=None, window=0, prefix=None):
        self.upload()
        self.plan(window, prefix)
        self.attend(scale, cap, slopes)
        _synced()
        self.compare(self.result(), *self.want(scale, cap, slopes, window, prefix))
        self.h.Close()


SHAPES = [(14, 2, 64, 0), (14, 2, 64, 1), (32, 8, 128, 1), (8, 2, 128, 0), (4, 4, 64, 1), (3, 3, 128, 0), (40, 2, 128, 1), (32, 1, 64, 0), (17, 1, 128, 1)]


@pytest.mark.parametrize("page", [8, 16, 128])
@pytest.mark.parametrize("heads,kv,hd,half", SHAPES)
def test_one_token_a_request(hip, bufs, heads, kv, hd, half, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 1023]
    print(f"tokens {heads}/{kv}/{hd} half={half} page={page}", flush=True)
    Case(hip, bufs, heads, kv, hd, half, page, [1] * len(lens), lens, seed=page).check()


@pytest.mark.parametrize("heads,kv,hd,half", [(14, 2, 64, 0), (8, 2, 128, 1), (32, 8, 128, 1), (4, 4, 64, 1), (3, 3, 128, 0)])
@pytest.mark.parametrize("length", [3000, 9001, 40000])
def test_one_long_request(hip, bufs, heads, kv, hd, half, length):
    print(f"long {heads}/{kv}/{hd} half={half} length={length}", flush=True)
    Case(hip, bufs, heads, kv, hd, half, 64, [1], [length], seed=length).check()


@pytest.mark.parametrize("page", [8, 32, 4096])
@pytest.mark.parametrize("heads,kv,hd,half", SHAPES)
def test_chunks(hip, bufs, heads, kv, hd, half, page):
    """Fresh prompts, chunks behind cached positions, drafted tokens, single tokens; odd lengths."""
    new = [1, 2, 3, 5, 31, 32, 33, 64, 100, 129, 1, 7]
    cached = [0, 0, 40, 63, 0, 1, 95, 64, 300, 0, 700, 129]
    print(f"chunks {heads}/{kv}/{hd} half={half} page={page}", flush=True)
    Case(hip, bufs, heads, kv, hd, half, page, new, [a + b for a, b in zip(new, cached)], seed=page).check()


@pytest.mark.parametrize("heads,kv,hd,half,new,length", [(4, 1, 128, 1, 700, 2300), (7, 1, 64, 1, 513, 513), (2, 2, 64, 0, 300, 1111), (8, 1, 128, 0, 130, 900)])
def test_long_chunks(hip, bufs, heads, kv, hd, half, new, length):
    print(f"long chunk {heads}/{kv}/{hd} half={half} {new} of {length}", flush=True)
    Case(hip, bufs, heads, kv, hd, half, 16, [new, 1], [length, 600], seed=new).check()


@pytest.mark.parametrize("half", [0, 1])
def test_requests_without_rows_or_length(hip, bufs, half):
    Case(hip, bufs, 8, 2, 64, half, 16, [0, 1, 0, 0, 3, 0, 40, 0], [0, 1, 77, 0, 3, 16, 90, 0], rowsMore=37, ld=4).check()


def test_nothing_to_do(hip, bufs):
    c = Case(hip, bufs, 8, 2, 64, 1, 16, [0, 0], [0, 30], rowsMore=5)
    c.check()
    h = E.NewHIPPaged(hip, 8, 2, 64, 16, 4, 1, 2, 8, 64)
    one = bufs.up(np.zeros(64, np.int32))
    assert h.Attention(one, 512, one, one, one, one, 512) == -4 and "plan" in E.last_error()
    _ok(h.Plan(one, None, 0, 8))
    _ok(h.Attention(None, 0, None, None, None, None, 0))
    _ok(h.Plan(one, one, 2, 0))
    _ok(h.Attention(None, 0, None, None, None, None, 0))
    _synced()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("window,prefix", [(1, False), (7, False), (64, False), (130, True), (1000, False), (0, True), (100000, False)])
def test_windows_and_prefixes(hip, bufs, heads, kv, hd, half, window, prefix):
    new, lens = [1, 1, 3, 70, 200, 40, 1], [900, 5, 64, 70, 450, 333, 300]
    print(f"window {window} prefix {prefix} {heads}/{kv}/{hd} half={half}", flush=True)
    Case(hip, bufs, heads, kv, hd, half, 8, new, lens, seed=window).check(window=window, prefix=[3, 5, 62, 70, 260, 0, 300] if prefix else None)


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("cap,slopes,window,prefix", [(50.0, False, 0, False), (2.0, False, 0, False), (0.0, True, 0, False), (30.0, True, 90, True)])
def test_changed_scores(hip, bufs, heads, kv, hd, half, cap, slopes, window, prefix):
    new, lens = [1, 3, 70, 200, 1, 1], [900, 64, 70, 450, 2, 129]
    print(f"cap {cap} slopes {slopes} {heads}/{kv}/{hd} half={half}", flush=True)
    sl = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32) if slopes else None
    Case(hip, bufs, heads, kv, hd, half, 32, new, lens, seed=int(cap), peak=4.0).check(cap=cap, slopes=sl, window=window, prefix=[3, 62, 70, 260, 1, 40] if prefix else None)


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("scale", [1.0, 1e-3])
def test_scale(hip, bufs, half, scale):
    """scale 1: scores of tens, nearly one position a row; small: nearly the mean of all."""
    Case(hip, bufs, 8, 2, 64, half, 16, [1, 90, 1], [700, 300, 33]).check(scale=scale)


@pytest.mark.parametrize("half", [0, 1])
def test_values_of_any_size(hip, bufs, half):
    """Rows of q and of the cache from tiny to large: nothing of the operands' range may be lost on the way into the products."""
    c = Case(hip, bufs, 8, 2, 128, half, 16, [1, 60, 1], [600, 140, 40], seed=8)
    c.q *= np.exp2(c.rng.integers(-30, 2, (c.q.shape[0], 1))).astype(np.float32)
    big = 3 if half else 40
    with np.errstate(over="ignore", invalid="ignore"):
        c.V = (c.V * np.exp2(c.rng.integers(-8, big, (1, c.V.shape[1])))).astype(c.kind)
        c.K = (c.K * np.exp2(c.rng.integers(-8, 2, (1, c.K.shape[1])))).astype(c.kind)
    c.check()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_pages_that_are_gone_hide_their_positions(hip, bufs, half, new):
    """Table entries of a request that are no page, first, last and in between; a request whose pages are all gone is zeros."""
    c = Case(hip, bufs, 8, 2, 128, half, 16, [new, new, new], [333, 200, 160], seed=new)
    c.table[0, [0, 3, 4, 5, 11]] = [-1, c.nPages, -(1 << 31), 0x7fffffff, -7]
    c.table[1, :] = -1
    c.table[2, 10 - -(-new // 16):10] = -1                         # the pages of its new tokens
    c.check()
    assert (c.result()[new:2 * new] == 0.0).all() if c.ldo == 1024 else True


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_values_that_are_no_numbers_count_where_they_are_seen(hip, bufs, heads, kv, hd, half, value):
    """A value row that is not finite reaches the tokens that see its position, and no other: neither the earlier tokens of its
    own chunk nor, with a window, the later ones."""
    for new, lens, window, bad in [([70, 3], [70, 90], 0, [(0, 41), (1, 88)]), ([40, 3], [140, 90], 20, [(0, 99), (0, 120), (1, 66), (1, 67)])]:
        c = Case(hip, bufs, heads, kv, hd, half, 8, new, lens, seed=3)
        for r, j in bad:
            c.V[c.where(r, j), 5::7] = value
        c.check(window=window)


@pytest.mark.parametrize("half", [0, 1])
def test_scores_that_are_no_numbers(hip, bufs, half):
    """A key of infinities or NaN behind the causal mask changes nothing; one that is seen makes its rows' results what the formula gives."""
    c = Case(hip, bufs, 8, 2, 64, half, 8, [70, 3], [100, 33], seed=4)
    c.K[c.where(0, 80)] = np.nan                                    # seen by positions 80 .. 99 of request 0 only
    c.K[c.where(1, 32)] = np.inf
    c.upload()
    c.plan()
    c.attend()
    _synced()
    want, bound = c.want()
    clean = np.ones(c.rows, bool)
    clean[50:70] = False
    clean[72] = False
    got = c.result()
    assert np.isnan(got[50:70]).all()
    assert (np.abs(got[:c.rows] - want)[clean] <= bound[clean]).all()
    h2 = Case(hip, bufs, 8, 2, 64, half, 8, [2], [40], seed=4)      # a score of minus infinity has no weight
    h2.q[:] = np.abs(h2.q)
    h2.K[h2.where(0, 7)] = -np.inf
    h2.V[h2.where(0, 7)] = 3.0
    h2.check()


def test_offsets_past_32_bits(hip, bufs):
    """A pool of 4.6 GB an array, the request's pages at its end."""
    heads, kv, hd, page, nPages = 8, 8, 128, 64, 35000
    row = kv * hd * 2
    pools = [E.lib.tw_gpu_alloc(nPages * page * row) for _ in range(2)]
    assert all(pools)
    for p in pools:
        E.KZero(p, nPages * page * row)
    c = Case(hip, bufs, heads, kv, hd, 1, page, [1, 70], [300, 200], seed=6, spare=0)
    big = E.NewHIPPaged(hip, heads, kv, hd, page, nPages, 1, 2, 71, c.maxLen)
    c.upload()
    first = nPages - c.nPages
    for p, a in zip(pools, (c.K, c.V)):
        a = np.ascontiguousarray(a)
        E.lib.tw_gpu_upload(p + first * page * row, a.ctypes.data, a.nbytes)
    table = np.where((c.table >= 0) & (c.table < c.nPages), c.table + first, -1).astype(np.int32)
    d = c.d
    _ok(big.Plan(d["rowStart"], d["lens"], 2, 71))
    _ok(big.Attention(d["q"], c.ldq, pools[0], pools[1], bufs.up(table), d["out"], c.ldo))
    _synced()
    c.compare(c.result(), *c.want())
    # and a row stored into the last slot
    x = np.random.default_rng(1).standard_normal((1, 3 * kv * hd)).astype(np.float32)
    dx, qo = bufs.up(x), bufs.up(np.zeros((1, kv * hd), np.float32))
    p0 = dx.DevicePtr()
    one, zero = np.ones(64, np.float32), np.zeros(64, np.float32)
    _ok(big.Store(p0, p0 + 4096, p0 + 8192, x.shape[1], x.shape[1], x.shape[1], qo, kv * hd, pools[0], pools[1],
                  bufs.up(np.array([nPages * page - 1], np.int32)), bufs.up(np.zeros(1, np.int32)), 1, bufs.up(one), bufs.up(zero), 1))
    _synced()
    for p, a in zip(pools, (x[0, kv * hd:2 * kv * hd], x[0, 2 * kv * hd:])):
        back = np.empty(kv * hd, np.float16)
        E.lib.tw_gpu_download(back.ctypes.data, p + (nPages * page - 1) * row, back.nbytes)
        assert np.array_equal(back, a.astype(np.float16))
    big.Close()
    for p in pools:
        E.lib.tw_gpu_free(p)


def test_lengths_that_do_not_fit_are_cut(hip, bufs):
    """rowStart and lens that pass the call's rows, the handle's maxLen, or run backwards: rows outside stay, nothing is read outside."""
    c = Case(hip, bufs, 8, 2, 64, 1, 16, [5, 1, 4], [60, 33, 60], seed=2)
    c.upload()
    rows = c.b.up(np.array([0, 5, 6, 4000], np.int32))
    lens = c.b.up(np.array([60, 33, 1 << 30], np.int32))
    _ok(c.h.Plan(rows, lens, 3, c.bound))
    c.attend()
    _synced()
    want, bound = c.want()
    got = c.result()
    assert (np.abs(got[:6] - want[:6]) <= bound[:6]).all() and np.isfinite(got).all()
    for bad in ([7, 2, 9, -5], [-(1 << 31), 0x7fffffff, 3, 8]):
        _ok(c.h.Plan(c.b.up(np.array(bad, np.int32)), c.b.up(np.array([-4, 33, 10], np.int32)), 3, c.bound))
        c.attend()
        _synced()


@pytest.mark.parametrize("half", [0, 1])
def test_the_same_call_gives_the_same_bits(hip, bufs, half):
    c = Case(hip, bufs, 32, 8, 128, half, 16, [1, 300, 1, 17], [5000, 900, 333, 2000], seed=9)
    c.upload()
    c.plan()
    outs = []
    for _ in range(4):
        c.b.put(c.d["out"], c.out0)
        c.attend()
        _synced()
        outs.append(c.result())
    assert all(np.array_equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("half", [0, 1])
def test_a_captured_step(hip, bufs, rt, half):
    """Tables, plan, store and attention of a step captured once and replayed as the requests grow, on a stream of its own,
    against the same calls made eagerly on another handle and another copy of everything; lengths stay on the device."""
    heads, kv, hd, page, n, rows, maxLen, nPages = 8, 2, 64, 8, 5, 64, 200, 130
    rng = np.random.default_rng(12)
    ang = np.arange(maxLen)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2.0 / hd)
    cos, sin = bufs.up(np.cos(ang).astype(np.float32)), bufs.up(np.sin(ang).astype(np.float32))
    kind, ld = (np.float16 if half else np.float32), (heads + 2 * kv) * hd

    def server():
        s = {"h": E.NewHIPPaged(hip, heads, kv, hd, page, nPages, half, n, rows, maxLen)}
        for name, a in dict(new=np.zeros(n, np.int32), lens=np.zeros(n, np.int32), table=np.full((n, 25), -1, np.int32), ring=np.arange(nPages, dtype=np.int32)[::-1],
                            state=np.array([0, nPages], np.int32), rowStart=np.zeros(n + 1, np.int32), slots=np.zeros(rows, np.int32), pos=np.zeros(rows, np.int32),
                            counts=np.zeros(4, np.int32), x=np.zeros((rows, ld), np.float32), K=np.full((nPages * page, kv * hd), np.nan, kind),
                            V=np.full((nPages * page, kv * hd), np.nan, kind), out=np.zeros((rows, heads * hd), np.float32)).items():
            s[name] = bufs.up(a)
        return s

    def step(s, stream):
        x, h = s["x"].DevicePtr(), s["h"]
        _ok(h.Tables(s["new"], n, s["lens"], s["lens"], s["table"], s["ring"], s["state"], s["state"], rows, s["rowStart"], s["slots"], s["pos"], s["counts"], stream))
        _ok(h.Plan(s["rowStart"], s["lens"], n, rows, 0, None, stream))
        _ok(h.Store(x, x + heads * hd * 4, x + (heads + kv) * hd * 4, ld, ld, ld, x, ld, s["K"], s["V"], s["slots"], s["pos"], rows, cos, sin, maxLen, stream))
        _ok(h.Attention(x, ld, s["K"], s["V"], s["table"], s["out"], heads * hd, 0.0, 0.0, None, stream))

    a, b, stream = server(), server(), rt.stream()
    graph = rt.capture(stream, lambda: step(a, stream))
    lens, k, v = np.zeros(n, np.int64), [np.zeros((0, kv * hd))] * n, [np.zeros((0, kv * hd))] * n
    for t in range(8):
        new = np.array([[30, 1, 0, 17, 5], [1, 1, 1, 1, 1], [1, 20, 1, -1, 0], [1, 1, 40, 0, 1], [-1, 1, 1, 9, 1], [60, 1, 1, 1, 1], [1, -1, 1, 1, 3], [1, 1, 1, 1, 1]][t], np.int32)
        x = rng.standard_normal((rows, ld)).astype(np.float32)
        for s in (a, b):
            bufs.put(s["new"], new)
            bufs.put(s["x"], x)
            bufs.put(s["out"], np.full((rows, heads * hd), 7.25, np.float32))
        E.KSync()
        rt.replay(graph, stream)
        step(b, None)
        _synced()
        got, eager = (bufs.down(s["out"], np.zeros((rows, heads * hd), np.float32)) for s in (a, b))
        assert np.array_equal(got, eager), t
        lens = np.where(new < 0, 0, lens + np.maximum(new, 0))
        assert bufs.down(a["counts"], np.zeros(4, np.int32))[3] == 0
        assert np.array_equal(bufs.down(a["lens"], np.zeros(n, np.int32)), lens)
        # against the model, from the pools as the store left them
        K, V = (bufs.down(a[w], np.zeros((nPages * page, kv * hd), kind)) for w in ("K", "V"))
        start = np.concatenate(([0], np.cumsum(np.maximum(new, 0))))
        q = bufs.down(a["x"], x)[:, :heads * hd]
        want, bound = P.attention(q, K, V, bufs.down(a["table"], np.zeros((n, 25), np.int32)), start, lens, page, heads // kv, hd)
        assert (np.abs(got[:start[-1]] - want) <= bound).all() and (got[start[-1]:] == 7.25).all()


def test_two_handles_on_two_streams(hip, bufs, rt):
    """Two requests' batches at once, each with a handle and a stream of its own."""
    cs = [Case(hip, bufs, 32, 8, 128, 1, 16, [1, 200], [9000, 700], seed=20 + k) for k in range(2)]
    ss = [rt.stream() for _ in cs]
    for c in cs:
        c.upload()
    E.KSync()
    for _ in range(3):
        for c, s in zip(cs, ss):
            c.plan(stream=s)
            c.attend(stream=s)
    for s in ss:
        rt.call("hipStreamSynchronize", s)
    for c in cs:
        c.compare(c.result(), *c.want())
