"""More of attention over an 8-bit paged cache: V rows whose sizes differ from stretch to stretch of positions, zeros among them.  The kernels hold a row's
weights -- probabilities times V's scales -- times a power of two that they choose from what they have seen so far.  The bound is Case8.want's: its last
term takes the largest weight of a row to be held at 2^11 or more, whatever came before it."""
import numpy as np
import pytest

from tests.paged_q8_model import Case8
from tests.test_gpu_paged import _synced, bufs  # noqa: F401  (fixtures)
from tests.test_gpu_paged_shared import make, plan

pytestmark = pytest.mark.gpu
NEW = [[1, 1], [3, 1], [80, 1]]          # narrow tiles; wide ones


def lay(c, sizes, gaps, stretch):
    """V rows of stretch s of every request (the last one: to its end) are of sizes[s], and its keys' scores gaps[s] powers of two above the others' --
    to a few powers of two, by what q and the keys have besides."""
    K, V = (np.nan_to_num(np.float32(getattr(c, n)), nan=0.0, posinf=0.0, neginf=0.0) for n in "KV")
    c.q[:] = 1.0 + 0.1 * c.q
    K *= 0.2
    up = np.log(2.0) / np.sqrt(c.hd)          # (q near ones: a key of k throughout has a score of k sqrt(hd))
    seen = np.zeros(len(V), bool)             # (rows that requests share: once)
    for r in range(len(c.lens)):
        j = np.arange(c.lens[r])
        at = c.table[r][j // c.page].astype(np.int64) * c.page + j % c.page
        j, at = j[~seen[at]], at[~seen[at]]
        seen[at] = True
        s = np.minimum(j // stretch, len(sizes) - 1)
        K[at] += (np.array(gaps)[s] * up)[:, None]
        V[at] *= np.array(sizes)[s][:, None]
    c.set_rows("K", K)
    c.set_rows("V", V)


def run(c, **what):
    c.upload()
    c.plan()
    c.attend(**what)
    _synced()
    c.compare(c.result(), *c.want(**what))
    c.h.Close()


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("stretch", [32, 64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-20])
def test_rows_of_zeros_that_hold_the_maximum(hip, bufs, new, stretch, size):
    """At the start, ahead of rows that count for little; again later, further up."""
    for hd in (64, 128):
        for gaps, sizes in (([6, 0], [0, size]), ([14, 0], [0, size]), ([0, 10, 3], [size, 0, size]), ([9, 0, 18, 0], [0, size, 0, size * 100])):
            print(f"zeros new={new} hd={hd} stretch={stretch} size={size} gaps={gaps}", flush=True)
            c = Case8(hip, bufs, 8, 2, hd, 16, new, [700, 300], seed=stretch)
            lay(c, sizes, gaps, stretch)
            run(c)


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("stretch", [32, 64, 128])
@pytest.mark.parametrize("sizes", [[1e8, 1e-28], [1e-28, 1e8], [1e10, 1e-30, 1e10], [1e-30, 1e10, 1e-30], [1e25, 1e-5, 1e-30, 0, 1e20], [0, 1e-30, 1e20, 1e30], [1e30, 0, 1e-30], [0, 0, 1e33]])
def test_sizes_that_differ_by_stretches(hip, bufs, new, stretch, sizes):
    """Ascending and descending, the scores too: small rows that move the maximum, large ones behind them."""
    n = len(sizes)
    for gaps in ([0] * n, [7 * i for i in range(n)], [7 * (n - 1 - i) for i in range(n)], [30 * (i % 2) for i in range(n)]):
        print(f"sizes new={new} stretch={stretch} {sizes} gaps={gaps}", flush=True)
        c = Case8(hip, bufs, 8, 2, 128, 16, new, [700, 300], seed=n)
        lay(c, sizes, gaps, stretch)
        run(c)


@pytest.mark.parametrize("cap,slopes,window", [(20.0, False, 0), (0.0, True, 0), (0.0, False, 300)])
@pytest.mark.parametrize("new", NEW)
def test_changed_scores_over_zeros(hip, bufs, new, cap, slopes, window):
    c = Case8(hip, bufs, 8, 2, 128, 16, new, [700, 300], seed=4)
    lay(c, [0, 1e-3, 0, 1e10], [9, 0, 15, 2], 64)
    sl = np.exp2(-np.arange(4, 12)).astype(np.float32) if slopes else None
    c.upload()
    c.plan(window)
    c.attend(cap=cap, slopes=sl)
    _synced()
    c.compare(c.result(), *c.want(cap=cap, slopes=sl, window=window))
    c.h.Close()


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("sizes,gaps", [([0, 1.0], [12, 0]), ([1e8, 1e-28], [0, 9]), ([1e-28, 1e12], [9, 0]), ([0, 1e-6, 0, 1e-6], [8, 0, 14, 0])])
def test_behind_shared_prefixes(hip, bufs, new, sizes, gaps):
    """Stretches of the shared positions, the requests' own among the last."""
    from tests.test_gpu_paged_shared import share
    c = make(8, hip, bufs, 8, 2, 64, 16, [new] * 4, [400 + new + 9 * r for r in range(4)], [0, 4], [400], seed=2)
    lay(c, sizes, gaps, 64)
    share(c, c.groups, c.shared)
    c.upload()
    plan(c, new)
    c.attend()
    _synced()
    c.compare(c.result(), *c.want())
    c.h.Close()


def test_long_requests_of_zeros_and_of_small_rows(hip, bufs):
    """What the probabilities sum up to stays a number."""
    for size in (0.0, 1e-33):
        c = Case8(hip, bufs, 4, 1, 64, 64, [1, 40], [140000, 30000], seed=6)
        lay(c, [size, 1e-2], [3, 0], 29000)
        run(c)
