"""Values that are no numbers under weights that fp32 holds as 0, in fp16 and fp32 caches: the rows that see the position have them, the others have not."""
import numpy as np
import pytest

from tests.test_gpu_paged import Case, _synced, bufs  # noqa: F401  (fixtures)
from tests.test_gpu_paged_shared import make, plan

pytestmark = pytest.mark.gpu


def without_weight(c, r, positions):
    """Scores of -800, the others' within 10 of 0."""
    c.q[:] = 1.0
    for j in positions:
        c.K[c.where(r, j)] = -100.0


def found(c, sees, value):
    """The result, of which rows `sees` of the batch see the value in columns 1, 6, .. of V's rows [kv * hd]."""
    got = c.result()[:c.rows, :c.heads * c.hd].reshape(c.rows, c.heads, c.hd)
    odd = np.zeros(got.shape, bool)
    columns = np.arange(c.kv * c.hd).reshape(c.kv, c.hd)[np.arange(c.heads) // c.group] % 5 == 1
    odd[sees] = columns
    if np.isnan(value):
        assert np.isnan(got[odd]).all(), np.argwhere(~np.isnan(got) & odd)[:5].tolist()
    else:                                                   # (no number, or the infinity)
        assert (np.isnan(got[odd]) | (got[odd] == value)).all()
    assert np.isfinite(got[~odd]).all(), np.argwhere(~np.isfinite(got) & ~odd)[:5].tolist()
    return got, odd


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("around", [1, 64])
@pytest.mark.parametrize("new,length,bad", [(1, 300, 299), (1, 300, 40), (3, 90, 88), (70, 70, 41), (70, 200, 160), (70, 200, 3), (300, 700, 399), (300, 700, 500)])
def test_under_no_weight(hip, bufs, half, value, around, new, length, bad):
    for hd in (64, 128):
        c = Case(hip, bufs, 8, 2, hd, half, 8, [new, 70], [length, 75], seed=bad)
        without_weight(c, 0, range(bad // around * around, min(bad // around * around + around, length)))
        c.V[c.where(0, bad), 1::5] = value
        c.upload()
        c.plan()
        c.attend()
        _synced()
        found(c, np.arange(new)[length - new + np.arange(new) >= bad], value)
        c.h.Close()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("window,prefix,new,length,bad", [(50, 0, 3, 300, 260), (50, 0, 150, 400, 300), (50, 40, 150, 400, 20), (50, 40, 3, 400, 39), (90, 130, 150, 400, 200), (90, 130, 2, 400, 200)])
def test_under_no_weight_in_windows(hip, bufs, half, value, window, prefix, new, length, bad):
    """Seen by some of the rows, by all (a prefix), by none (between a prefix and the windows)."""
    c = Case(hip, bufs, 8, 2, 128, half, 16, [new, 1], [length, 75], seed=bad)
    without_weight(c, 0, range(bad // 32 * 32, bad // 32 * 32 + 32))
    c.V[c.where(0, bad), 1::5] = value
    c.upload()
    c.plan(window, [prefix, 0] if prefix else None)
    c.attend()
    _synced()
    i = length - new + np.arange(new)
    found(c, np.arange(new)[((bad <= i) & (bad > i - window)) | (bad < prefix)], value)
    c.h.Close()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("bad", [5, 198, 199, 200])
def test_under_no_weight_behind_shared_prefixes(hip, bufs, half, new, bad):
    from tests.test_gpu_paged_shared import share
    c = make(half, hip, bufs, 8, 2, 64, 8, [new] * 4, [200 + new] * 4, [0, 3, 4], [200, 0], seed=3)
    without_weight(c, 0, range(bad // 32 * 32, min(bad // 32 * 32 + 32, 200 + new - 1)))
    c.V[c.where(0, bad), 1::5] = np.nan
    share(c, c.groups, c.shared)
    c.upload()
    plan(c, new)
    c.attend()
    _synced()
    sees = np.concatenate([np.arange(new)[200 + np.arange(new) >= bad] + r * new for r in (range(3) if bad < 200 else [0])])
    found(c, sees, np.nan)
    c.h.Close()
