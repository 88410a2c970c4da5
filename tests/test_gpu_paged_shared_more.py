"""More of attention behind shared prefixes (HIPPaged.PlanShared): groups whose tiles are many for the workers that there are, so that a worker has
several of them and leaves a share of each; plans that differ in the most rows that a request has; requests that come and end.  Bounds as in test_gpu_paged_shared."""
import copy

import numpy as np
import pytest

from mongoose_amd import engine as E
from tests import paged_model as P
from tests import paged_q8_model as Q
from tests.test_gpu_paged import _ok, _synced, bufs, rt  # noqa: F401  (fixtures)
from tests.test_gpu_paged_shared import FORMATS, make, plan

pytestmark = pytest.mark.gpu


def want_of(c, reqs, **what):
    """What the model gives for some of the requests, and their rows."""
    s = copy.copy(c)
    s.new, s.lens, s.table = c.new[reqs], c.lens[reqs], c.table[reqs]
    rows = np.concatenate([np.arange(c.rowStart[r], c.rowStart[r + 1]) for r in reqs])
    s.q, s.rowStart = c.q[rows], np.concatenate(([0], np.cumsum(s.new))).astype(np.int32)
    return (rows, *s.want(**what))


def check_some(c, reqs, mostNew=0, **what):
    c.upload()
    plan(c, mostNew)
    c.attend(**what)
    _synced()
    got = c.result()
    assert np.isfinite(got).all()
    rows, want, bound = want_of(c, reqs, **what)
    off = np.abs(got[rows][:, :c.heads * c.hd] - want) / bound
    print(f"  worst {off.max():.3f} of the bound", flush=True)
    assert off.max() <= 1.0, np.unique(rows[np.nonzero((off > 1).any(1))[0]])[:10].tolist()
    c.h.Close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd,n,new,length,groups", [(16, 8, 64, 16, 400, 300, 1), (16, 8, 64, 16, 400, 300, 2), (6, 6, 128, 5, 1500, 333, 2), (32, 8, 128, 4, 1024, 1000, 1)])
def test_prompts_that_arrive_together(hip, bufs, fmt, heads, kv, hd, n, new, length, groups):
    """Tiles from half the workers up: a worker has the end of one and all of the next."""
    print(f"shared prompts fmt={fmt} {heads}/{kv}/{hd} {n} of {new} behind {length}, {groups} groups", flush=True)
    own = [new + (r % 3) * (groups - 1) for r in range(n)]
    starts = [0, n] if groups == 1 else [0, n // 2, n]
    c = make(fmt, hip, bufs, heads, kv, hd, 32, own, [length + x for x in own], starts, [length, length // 3][:groups], seed=n)
    check_some(c, [0, n // 2, n - 1] if heads < 32 else [2], new + 2)


@pytest.mark.parametrize("fmt,mostNew", [(0, 0), (1, 40), (8, 40)])
def test_many_requests_of_some_rows(hip, bufs, fmt, mostNew):
    """64 requests of 40 rows behind 8,001 positions: 80 tiles for 64 workers."""
    print(f"shared 64 x 40 behind 8001 fmt={fmt} mostNew={mostNew}", flush=True)
    c = make(fmt, hip, bufs, 32, 8, 128, 64, [40] * 64, [8041 + r % 7 for r in range(64)], [0, 64], [8001], seed=1)
    check_some(c, [0, 21, 63], mostNew)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd,size,new", [(32, 8, 128, 2, 1), (8, 8, 64, 2, 1), (14, 2, 64, 3, 3), (8, 8, 64, 2, 9)])
def test_many_groups_of_any_length(hip, bufs, fmt, heads, kv, hd, size, new):
    """Groups of two or three requests behind 50 to 3,000 positions: a worker has many short tiles, or a part of a long one; narrow and wide."""
    print(f"shared groups fmt={fmt} {heads}/{kv}/{hd} size={size} new={new}", flush=True)
    n = 100 if new == 1 else 70
    rng = np.random.default_rng(n + size)
    shared = np.exp(rng.uniform(np.log(50), np.log(3000), n)).astype(int)
    own = [new + int(rng.integers(0, 30)) for _ in range(n * size)]
    lens = [int(shared[r // size]) + own[r] for r in range(n * size)]
    c = make(fmt, hip, bufs, heads, kv, hd, 16, [new] * (n * size), lens, list(range(0, n * size + 1, size)), shared, seed=n)
    check_some(c, list(range(n * size)), new)


@pytest.mark.parametrize("fmt", FORMATS)
def test_few_rows_in_many_groups(hip, bufs, fmt):
    """Narrow tiles, more than workers: 60 groups of two requests, one query head a KV head, 16 KV heads."""
    rng = np.random.default_rng(4)
    shared = rng.integers(20, 900, 60)
    lens = [int(shared[r // 2]) + int(rng.integers(1, 40)) for r in range(120)]
    c = make(fmt, hip, bufs, 16, 16, 64, 8, [1] * 120, lens, list(range(0, 121, 2)), shared, seed=8)
    check_some(c, list(range(120)), 1)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scores_changed_by_distance_in_many_tiles(hip, bufs, fmt):
    slopes = np.exp2(-np.arange(1, 9)).astype(np.float32)
    c = make(fmt, hip, bufs, 8, 8, 64, 16, [150] * 40, [370 + r for r in range(40)], list(range(0, 41, 4)), [200, 60, 199, 3, 120, 210, 64, 65, 180, 1], seed=5)
    check_some(c, [0, 5, 11, 22, 39], 150, cap=30.0, slopes=slopes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("most", [(1, 0), (0, 1)])
def test_plans_for_other_numbers_of_rows_in_turn(hip, bufs, rt, fmt, most):
    """Plans of one step that differ in mostNew alone have other kinds of tiles.  Attention captured behind one does nothing on the other, and is right
    again on its own; so is an eager call behind a plan that was captured and has not run."""
    c = make(fmt, hip, bufs, 8, 2, 64, 8, [3, 1, 70, 1], [260, 233, 400, 50], [0, 3], [200], seed=2)
    c.upload()
    want, stream = c.want(), rt.stream()
    c.d["groups"], c.d["shared"] = c.b.up(c.groups), c.b.up(c.shared)

    def made(m, stream=None):
        _ok(c.h.PlanShared(c.d["rowStart"], c.d["lens"], 4, c.bound, m, c.d["groups"], c.d["shared"], 1, stream))

    def got():
        _synced()
        x = c.result()
        c.b.put(c.d["out"], c.out0)
        E.KSync()
        return x

    made(most[0])
    alone = rt.capture(stream, lambda: c.attend(stream=stream))
    E.KSync()
    rt.replay(alone, stream)
    c.compare(got(), *want)
    for _ in range(2):
        made(most[1])
        E.KSync()
        rt.replay(alone, stream)
        assert (got() == 7.25).all()
        c.attend()
        c.compare(got(), *want)
        made(most[0])
        E.KSync()
        rt.replay(alone, stream)
        c.compare(got(), *want)
    later = rt.capture(stream, lambda: made(most[1], stream))
    c.attend()
    assert (got() == 7.25).all()
    rt.replay(later, stream)
    c.attend()
    c.compare(got(), *want)
    c.h.Close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_plan_of_wide_tiles_that_has_never_run(hip, bufs, rt, fmt):
    """The first plan of a handle has no wide tiles for requests, the second has and is only captured: an eager call leaves out as it was."""
    c = make(fmt, hip, bufs, 8, 2, 64, 8, [1, 1, 80, 1], [260, 233, 400, 50], [0, 3], [200], seed=3)
    c.upload()
    want, stream = c.want(), rt.stream()
    plan(c, 1)
    E.KSync()
    d = c.d
    later = rt.capture(stream, lambda: _ok(c.h.PlanShared(d["rowStart"], d["lens"], 4, c.bound, 0, d["groups"], d["shared"], 1, stream)))
    c.attend()
    _synced()
    assert (c.result() == 7.25).all()
    rt.replay(later, stream)
    c.attend()
    _synced()
    c.compare(c.result(), *want)
    c.h.Close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_requests_behind_one_prefix_come_and_end(hip, bufs, rt, fmt):
    """Tables, plan, store and attention captured once and replayed.  Request 0 holds the prefix (whole pages); a request that comes behind it has
    those pages in its row of the table and their length; one that ends gives back its own: they go to the front of its row and its length is theirs.
    Every page is in one place at any time, and all are free at the end."""
    heads, kv, hd, page, n, rows, nPages, width, shared = 8, 2, 64, 8, 6, 48, 60, 16, 40
    maxLen, P0 = page * width, shared // page
    rng = np.random.default_rng(fmt)
    ang = np.arange(maxLen)[:, None] * 1e4 ** (-np.arange(hd // 2) * 2.0 / hd)
    cos, sin = bufs.up(np.cos(ang).astype(np.float32)), bufs.up(np.sin(ang).astype(np.float32))
    ld = (heads + 2 * kv) * hd
    h = E.NewHIPPaged(hip, heads, kv, hd, page, nPages, fmt, n, rows, maxLen)
    assert h is not None and h.TableWidth() == width
    _ok(h.Share())
    host = dict(new=np.zeros(n, np.int32), lens=np.zeros(n, np.int32), table=np.full((n, width), -1, np.int32), ring=rng.permutation(nPages).astype(np.int32),
                state=np.array([7, nPages], np.int32), rowStart=np.zeros(n + 1, np.int32), slots=np.zeros(rows, np.int32), pos=np.zeros(rows, np.int32),
                counts=np.zeros(4, np.int32), x=np.zeros((rows, ld), np.float32), K=np.zeros(h.PoolBytes(), np.uint8), V=np.zeros(h.PoolBytes(), np.uint8),
                out=np.zeros((rows, heads * hd), np.float32), groups=np.array([0, n], np.int32), shared=np.array([shared], np.int32))
    s = {name: bufs.up(a) for name, a in host.items()}
    x, stream = s["x"].DevicePtr(), rt.stream()

    def step():
        _ok(h.Tables(s["new"], n, s["lens"], s["lens"], s["table"], s["ring"], s["state"], s["state"], rows, s["rowStart"], s["slots"], s["pos"], s["counts"], stream))
        _ok(h.PlanShared(s["rowStart"], s["lens"], n, rows, 0, s["groups"], s["shared"], 1, stream))
        _ok(h.Store(x, x + heads * hd * 4, x + (heads + kv) * hd * 4, ld, ld, ld, x, ld, s["K"], s["V"], s["slots"], s["pos"], rows, cos, sin, maxLen, stream))
        _ok(h.Attention(x, ld, s["K"], s["V"], s["table"], s["out"], heads * hd, 0.0, 0.0, None, stream))

    graph = rt.capture(stream, step)
    down = lambda name: bufs.down(s[name], host[name])  # noqa: E731
    lens = np.zeros(n, np.int64)
    for t, new in enumerate([[40, 0, 0, 0, 0, 0], [0, 3, 1, 9, 0, 0], [0, 1, 1, 1, 0, 0], [0, 1, -1, 8, 5, 0], [0, 20, 7, 1, 1, 0], [0, -1, 4, -1, 1, 20], [0, 2, 1, 0, -1, 30], [0, 1, -1, 7, 3, -1],
                             [0, -1, 0, 1, 1, 0], [0, 0, 0, -1, -1, 0], [-1, 0, 0, 0, 0, 0]]):
        table, at = down("table"), lens.copy()
        for r in range(1, n):
            if new[r] > 0 and at[r] == 0:                       # comes
                table[r, :P0] = table[0, :P0]
                at[r] = shared
            elif new[r] < 0:                                    # ends
                own = -(-at[r] // page) - P0
                table[r, :own] = table[r, P0:P0 + own].copy()
                at[r] -= shared
        q = rng.standard_normal((rows, ld)).astype(np.float32)
        for name, a in (("table", table), ("lens", at.astype(np.int32)), ("new", np.array(new, np.int32)), ("x", q), ("out", np.full((rows, heads * hd), 7.25, np.float32))):
            bufs.put(s[name], a)
        E.KSync()
        rt.replay(graph, stream)
        lens = np.where(np.array(new) < 0, 0, at + np.maximum(new, 0))
        table, counts, state, ring = down("table"), down("counts"), down("state"), down("ring")
        assert counts[3] == 0 and np.array_equal(down("lens"), lens), (t, counts.tolist())
        held = [int(table[r, e]) for r in range(n) if lens[r] for e in range(P0 if r else 0, -(-int(lens[r]) // page))]
        free = [int(ring[(state[0] + i) % nPages]) for i in range(state[1])]
        assert sorted(held + free) == list(range(nPages)), t
        for r in range(1, n):
            assert lens[r] == 0 or np.array_equal(table[r, :P0], table[0, :P0])
        start = np.concatenate(([0], np.cumsum(np.maximum(new, 0))))
        pools = []
        for name in "KV":
            data = down(name)
            if fmt == 8:
                data = Q.values(*Q.from_pool(data, nPages * page, kv, hd, page))
            else:
                data = data.view(np.float16 if fmt else np.float32)
            pools.append(data.reshape(-1, kv * hd))
        got = down("out")
        want, bound = P.attention(down("x")[:, :heads * hd], *pools, table, start, lens, page, heads // kv, hd)
        assert (np.abs(got[:start[-1]] - want) <= bound).all() and (got[start[-1]:] == 7.25).all(), t
    assert down("state")[1] == nPages
    h.Close()
