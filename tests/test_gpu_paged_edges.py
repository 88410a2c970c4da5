"""Attention over a paged KV cache at the edges of its arguments: values that are no numbers at positions that a row does not
see, infinities where it does; rows of q from tiny to huge; the largest window; arguments that overlap; plans that did not run or
were written over; more requests, tiles and shares than one round of the plan or of a join takes.  Against 64 bits, as test_gpu_paged."""
import numpy as np
import pytest

from mongoose_amd import engine as E
from tests import paged_model as P
from tests.test_gpu_paged import Case, bufs, rt  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def _check(c, **what):
    """As Case.check; what is no number is the infinity, or the NaN, that the formula gives.  The model leaves whole positions with a value
    that is no number out of its bound: here it is relative to sum_j p_j |v_j| over all the finite v_j of a column."""
    c.upload()
    c.plan(what.get("window", 0), what.get("prefix"))
    c.attend(what.get("scale", 0.0), what.get("cap", 0.0), what.get("slopes"))
    E.KSync()
    assert E.HIPCheck() == 0
    want, _ = c.want(**what)
    V = c.V
    c.V = np.where(np.isfinite(V), V, 0).astype(c.kind)
    _, bound = c.want(**what)
    c.V = V
    got = c.result()
    odd = ~np.isfinite(want)
    g = got[:c.rows, :c.heads * c.hd][odd]
    same = (g == want[odd]) | (np.isnan(g) & np.isnan(want[odd]))
    assert same.all(), (np.argwhere(odd)[~same][:5].tolist(), g[~same][:5], want[odd][~same][:5])
    c.compare(got, want, bound)
    c.h.Close()


# ---------------------------------------------------------------------------------------------------------------------
# values that are no numbers at positions that a row does not see
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("heads,kv,hd,new,lens,window,bad", [
    (32, 1, 64, 70, 70, 0, (41,)), (40, 1, 128, 70, 70, 0, (41, 69)), (71, 1, 64, 33, 80, 0, (60, 79)), (128, 2, 128, 20, 100, 0, (81, 83)),
    (32, 1, 128, 40, 140, 20, (82, 99, 120)), (71, 1, 64, 12, 300, 33, (256, 260, 295)), (4, 1, 128, 41, 141, 20, (113, 119, 120)), (16, 4, 64, 41, 141, 20, (113, 119, 120))])
def test_hidden_values_where_a_wave_of_a_wide_tile_is_one_token(hip, bufs, heads, kv, hd, new, lens, window, bad, value, half):
    """Groups of 32 heads and more, or a last token alone: the tile holds positions that its other tokens see, and this one does not."""
    print(f"hidden {heads}/{kv}/{hd} half={half} {new} of {lens} window {window}", flush=True)
    c = Case(hip, bufs, heads, kv, hd, half, 8, [new, 3], [lens, 20], seed=lens, rowsMore=300)
    for j in bad:
        c.V[c.where(0, j), j % 5::7] = value
    _check(c, window=window)


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("heads,kv,hd,n", [(4, 4, 64, 1), (8, 2, 128, 2), (40, 1, 128, 7), (32, 1, 64, 9)])
def test_hidden_values_between_a_single_tokens_prefix_and_its_window(hip, bufs, heads, kv, hd, n, value, half):
    """What lies behind the prefix and before the window shares units with both; groups of 32 and 40 in batches above 256 rows have wide tiles."""
    print(f"gap {heads}/{kv}/{hd} x {n} half={half}", flush=True)
    lens = [500 - 7 * r for r in range(n)]
    for bad in ((10, 31), (420, 435), (200,)):
        c = Case(hip, bufs, heads, kv, hd, half, 8, [1] * n, lens, seed=n)
        for j in bad:
            c.V[c.where(0, j), j % 5::7] = value
        _check(c, window=64, prefix=[10] * n)


# ---------------------------------------------------------------------------------------------------------------------
# infinite values at positions that are seen
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,kv,hd,new,lens,window,prefix", [
    (4, 4, 64, [1, 1], [200, 33], 0, None), (8, 2, 128, [1, 3], [900, 64], 0, None), (8, 2, 64, [70, 200], [70, 450], 0, None), (8, 2, 128, [130, 1, 40], [300, 129, 333], 0, None),
    (32, 1, 64, [70, 1], [300, 90], 50, None), (8, 2, 128, [3, 100], [300, 400], 90, [20, 310]), (3, 3, 128, [1], [9001], 0, None), (8, 1, 64, [60], [12000], 0, None)])
def test_infinite_values_that_are_seen_keep_their_sign(hip, bufs, heads, kv, hd, new, lens, window, prefix, half):
    """Either infinity, both in one column (no number), and NaN, at first, middle and last positions."""
    print(f"signs {heads}/{kv}/{hd} half={half} {new} of {lens}", flush=True)
    c = Case(hip, bufs, heads, kv, hd, half, 8, new, lens, seed=lens[0])
    for r, n in enumerate(lens):
        for j, first, value in ((n - 1, 0, np.inf), (n // 2, 1, -np.inf), (n // 2 + 1, 2, np.inf), (n - new[r], 2, -np.inf), (0, 3, np.inf), (n - 1, 4, np.nan), (n - 1, 5, -np.inf)):
            c.V[c.where(r, j), first::11] = value
    _check(c, window=window, prefix=prefix)


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,kv,new,lens", [(4, 4, [1, 2], [300, 80]), (8, 2, [100], [300])])
def test_infinite_values_of_small_weight(hip, bufs, heads, kv, new, lens, half):
    """Weights below what two fp16 terms hold, above the least fp32 number: the infinity counts all the same."""
    c = Case(hip, bufs, heads, kv, 64, half, 8, new, lens, seed=2, peak=9.0)
    small = 0
    for r, n in enumerate(lens):
        first = n - new[r]
        c.V[c.where(r, 5), ::9] = -np.inf
        c.V[c.where(r, first // 2), 4::9] = np.inf
        at = [c.where(r, j) for j in range(n)]
        for h in range(heads):
            col = slice(h // c.group * 64, h // c.group * 64 + 64)
            s = c.q[c.rowStart[r]:c.rowStart[r + 1], h * 64:h * 64 + 64] @ c.K[at][:first, col].astype(np.float32).T / 8
            rel = (s[:, [5, first // 2]] - s.max(1, keepdims=True)) * 1.4426950408889634
            assert rel.min() > -120
            small += int((rel < -42).sum())
    assert small > 0
    _check(c)


# ---------------------------------------------------------------------------------------------------------------------
# scales and rows of q whose factor in powers of two is no fp32 number
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("scale,size,keys", [(1e-30, 1e-12, 1.0), (1e-30, 1e-36, 1.0), (0.0, 1e-38, 1.0), (1e30, 1e30, 0.0), (1e-30, 1e30, 1.0)])
def test_scales_far_from_the_rows_of_q(hip, bufs, scale, size, keys, half):
    """Scores next to nothing, ordinary ones of a small scale and a huge q, zero keys under a scale times q that is no fp32 number."""
    for cap in (0.0, 20.0):
        c = Case(hip, bufs, 8, 2, 64, half, 16, [1, 90, 3], [300, 300, 40], seed=5)
        c.q = (c.q * size).astype(np.float32)
        c.K = (c.K * keys).astype(c.kind)
        c.check(scale=scale, cap=cap)


# ---------------------------------------------------------------------------------------------------------------------
# calls whose arguments overlap
# ---------------------------------------------------------------------------------------------------------------------
def test_overlapping_arguments_are_refused(hip, bufs):
    x = np.ones((4, 24 * 64), np.float32)
    d = bufs.up(x)
    p = d.DevicePtr()
    h = E.NewHIPPaged(hip, 8, 2, 64, 8, 4, 0, 2, 4, 32)
    K, V, z = bufs.up(np.zeros((32, 128), np.float32)), bufs.up(np.zeros((32, 128), np.float32)), bufs.up(np.zeros(64, np.int32))
    slots = bufs.up(np.arange(4, dtype=np.int32))
    c, s = bufs.up(np.ones(32, np.float32)), bufs.up(np.zeros(32, np.float32))

    def store(o, ldo):
        return h.Store(p, p + 2048, p + 2560, 768, 768, 768, o, ldo, K, V, slots, z, 4, c, s, 1)

    assert store(p, 512) == -2 and "qOut overlaps q" in E.last_error()
    assert store(p + 1024, 768) == -2 and "qOut overlaps" in E.last_error()
    E.KSync()
    assert np.array_equal(bufs.down(d, x), x)
    assert store(p, 768) == 0
    E.KSync()
    one = bufs.up(np.array([0, 1, 4], np.int32))
    assert h.Plan(one, one, 2, 4) == 0
    for out in (p, p + 256, p + 1536 * 2, K, V):
        assert h.Attention(p, 768, K, V, z, out, 768) == -2 and "out" in E.last_error(), out
    h.Close()


# ---------------------------------------------------------------------------------------------------------------------
# windows wider than any request
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("half", [0, 1])
def test_the_largest_window_is_none(hip, bufs, half):
    """Also for requests with more rows than positions, whose first rows see nothing."""
    outs = []
    for window in (0, (1 << 31) - 1):
        c = Case(hip, bufs, 8, 2, 64, half, 8, [5, 1, 90], [60, 33, 120], seed=1)
        c.lens[0], c.lens[2] = 3, 40
        c.upload()
        c.plan(window)
        c.attend()
        E.KSync()
        outs.append(c.result())
        c.h.Close()
    assert np.array_equal(*outs) and (outs[0][:2] == 0).all() and (outs[0][2:6] != 0).any(1).all() and (outs[0][6:56] == 0).all() and (outs[0][56:] != 0).any(1).all()


# ---------------------------------------------------------------------------------------------------------------------
# plans that did not run, or that another has written over
# ---------------------------------------------------------------------------------------------------------------------
def _two_batches(hip, bufs, half):
    """(case, the arguments of its plan, those of a plan of its first request alone)"""
    c = Case(hip, bufs, 8, 2, 64, half, 8, [3, 1, 90], [60, 33, 400], seed=2)
    c.upload()
    d = c.d
    return c, (d["rowStart"], d["lens"], 3, c.rows, 0, None), (d["rowStart"], d["lens"], 1, 3, 0, None)


def _got(c):
    E.KSync()
    assert E.HIPCheck() == 0
    got = c.result()
    c.b.put(c.d["out"], c.out0)
    return got


@pytest.mark.parametrize("half", [0, 1])
def test_a_plan_that_was_captured_and_has_not_run(hip, bufs, rt, half):
    c, whole, _ = _two_batches(hip, bufs, half)
    want, bound = c.want()
    stream = rt.stream()

    def step():
        assert c.h.Plan(*whole, stream) == 0
        c.attend(stream=stream)

    graph = rt.capture(stream, step)
    c.attend()
    assert (_got(c) == 7.25).all()
    for _ in range(3):
        rt.replay(graph, stream)
        c.compare(_got(c), want, bound)
        c.attend()                       # the plan is there now
        c.compare(_got(c), want, bound)
    c.h.Close()


@pytest.mark.parametrize("half", [0, 1])
def test_a_plan_of_another_batch_in_the_handle(hip, bufs, rt, half):
    c, whole, first = _two_batches(hip, bufs, half)
    want, bound = c.want()
    stream = rt.stream()
    assert c.h.Plan(*whole) == 0
    alone = rt.capture(stream, lambda: c.attend(stream=stream))

    def step():
        assert c.h.Plan(*whole, stream) == 0
        c.attend(stream=stream)

    both = rt.capture(stream, step)
    for _ in range(2):
        assert c.h.Plan(*first) == 0
        c.attend()
        got = _got(c)
        assert (np.abs(got[:3, :512] - want[:3]) <= bound[:3]).all() and (got[3:] == 7.25).all()
        rt.replay(alone, stream)         # captured behind the plan of all three
        assert (_got(c) == 7.25).all()
        rt.replay(both, stream)
        c.compare(_got(c), want, bound)
        c.attend()                       # asked for behind the plan of one
        assert (_got(c) == 7.25).all()
        rt.replay(alone, stream)
        c.compare(_got(c), want, bound)
        assert c.h.Plan(*whole[:4], 5) == 0      # the same batch, another window
        E.KSync()
        rt.replay(alone, stream)
        assert (_got(c) == 7.25).all()
    c.h.Close()


# ---------------------------------------------------------------------------------------------------------------------
# many requests, tiles and shares
# ---------------------------------------------------------------------------------------------------------------------
def _check_some(c, which, **what):
    """As Case.check for the rows of some requests."""
    c.upload()
    c.plan(what.get("window", 0))
    c.attend()
    E.KSync()
    assert E.HIPCheck() == 0
    got = c.result()
    assert np.isfinite(got).all() and (got[c.rows:] == 7.25).all()
    for r in which:
        a, b = int(c.rowStart[r]), int(c.rowStart[r + 1])
        want, bound = P.attention(c.q[a:b, :c.heads * c.hd], c.K, c.V, c.table[r:r + 1], np.array([0, b - a]), c.lens[r:r + 1], c.page, c.group, c.hd, **what)
        assert (np.abs(got[a:b, :c.heads * c.hd] - want) <= bound).all(), r
    c.h.Close()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,kv,n", [(4, 1, 1100), (2, 2, 4096), (32, 1, 1500), (8, 4, 2049)])
def test_more_requests_than_the_plan_has_threads(hip, bufs, heads, kv, n, half):
    """A token each, from 1 position up; groups of up to 16 are narrow tiles, 32 a wide one a request."""
    print(f"{n} requests {heads}/{kv} half={half}", flush=True)
    lens = np.random.default_rng(n).integers(1, 70, n)
    lens[[0, n - 1]] = 1, 600
    _check_some(Case(hip, bufs, heads, kv, 64, half, 16, [1] * n, lens, seed=n), range(n) if heads * n < 12000 else [*range(0, n, 7), n - 1])


@pytest.mark.parametrize("half", [0, 1])
def test_more_tiles_than_the_plan_has_places_for(hip, bufs, half):
    """110 rows x 128 heads each: 4,400 wide tiles."""
    lens = [110 + 3 * r for r in range(40)]
    _check_some(Case(hip, bufs, 128, 1, 64, half, 16, [110] * 40, lens, seed=1), (0, 9, 10, 37, 38, 39))


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("heads,hd,new,length", [(2, 64, 130, 33001), (4, 128, 65, 41000)])
def test_tiles_of_more_shares_than_are_joined_at_once(hip, bufs, heads, hd, new, length, half):
    print(f"shares {heads}/1/{hd} half={half} {new} of {length}", flush=True)
    Case(hip, bufs, heads, 1, hd, half, 64, [new], [length], seed=new).check()
