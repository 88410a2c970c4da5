"""Rows read back by the hundred million bytes: more rows than one launch may have threads for."""
import numpy as np
import pytest

from mongoose_amd import engine as E
from tests.test_gpu_paged import _ok, _synced, bufs  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_launch_has(hip, bufs):
    """Five requests of up to 2^24 positions over 16 pages of 4,096, 2^26 + 103 rows of 64 floats: those at both ends, and around the 2^26th."""
    page, nPages, kv, hd, maxLen = 4096, 16, 1, 64, 1 << 24
    rng = np.random.default_rng(3)
    h = E.NewHIPPaged(hip, 1, kv, hd, page, nPages, 0, 5, 1, maxLen)
    assert h is not None, E.last_error()
    lens = np.array([maxLen] * 4 + [100], np.int32)
    starts = np.concatenate(([0], np.cumsum(lens))).astype(np.int32)
    rows = int(starts[-1]) + 3
    table = rng.integers(0, nPages, (5, h.TableWidth())).astype(np.int32)
    pool = [rng.standard_normal((nPages * page, hd)).astype(np.float32) for _ in range(2)]
    K, V = (bufs.up(a) for a in pool)
    outs = [E.lib.tw_gpu_alloc(rows * hd * 4) for _ in range(2)]
    assert all(outs)
    spots = [0, 1 << 25, (1 << 26) - 300, rows - 200]
    mark = np.full((200, hd), 7.25, np.float32)
    for o in outs:
        for at in spots:
            E.lib.tw_gpu_upload(o + at * hd * 4, mark.ctypes.data, mark.nbytes)
    print(f"load {rows} rows", flush=True)
    _ok(h.Load(K, V, bufs.up(table), bufs.up(starts), bufs.up(lens), 5, rows, outs[0], hd, outs[1], hd))
    _synced()
    for o, x in zip(outs, pool):
        for at in spots:
            got = np.empty((200, hd), np.float32)
            E.lib.tw_gpu_download(got.ctypes.data, o + at * hd * 4, got.nbytes)
            i = at + np.arange(200)
            r = np.searchsorted(starts, i, "right") - 1
            want = np.full((200, hd), 7.25, np.float32)
            mine = r < 5
            pos = i[mine] - starts[r[mine]]
            want[mine] = x[table[r[mine], pos // page] * page + pos % page]
            assert np.array_equal(got, want), at
    for o in outs:
        E.lib.tw_gpu_free(o)
    h.Close()
