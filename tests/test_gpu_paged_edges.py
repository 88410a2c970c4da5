"""Attention over a paged KV cache at the edges of its arguments: values that are no numbers at positions that a row does not
see.  Against 64 bits, as test_gpu_paged."""
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
