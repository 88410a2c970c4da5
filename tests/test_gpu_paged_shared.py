"""Attention of requests that share their first positions (HIPPaged.PlanShared): the shared ones once a group, against the plain model of
every request by itself, in 64 bits.

The bound is paged_model.attention's: a row's result is joined from two parts as from any two shares of a tile, which its terms count."""
import numpy as np
import pytest

from mongoose_amd import engine as E
from tests.paged_q8_model import Case8
from tests.test_gpu_paged import Case, _ok, _synced, bufs, rt  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
FORMATS = [0, 1, 8]


def copy_rows(c, a, r, s):
    """Makes request r name request a's pages for the whole pages below s, and hold copies of its rows on the page where that ends."""
    c.table[r, :s // c.page] = c.table[a, :s // c.page]
    for j in range(s // c.page * c.page, s):
        x, y = c.where(a, j), c.where(r, j)
        for name in "KV":
            getattr(c, name)[y] = getattr(c, name)[x]
            if c.half == 8:
                c.q8[name][y], c.scales[name][y] = c.q8[name][x], c.scales[name][x]


def share(c, groups, lens):
    """The first lens[g] positions of requests groups[g] .. groups[g+1]-1 of a batch as those of the first of them."""
    for g, s in enumerate(lens):
        for r in range(groups[g] + 1, groups[g + 1]):
            copy_rows(c, groups[g], r, min(int(s), int(c.lens[groups[g]]), int(c.lens[r])))


def make(fmt, hip, bufs, heads, kv, hd, page, new, lens, groups, shared, **more):
    c = Case8(hip, bufs, heads, kv, hd, page, new, lens, **more) if fmt == 8 else Case(hip, bufs, heads, kv, hd, fmt, page, new, lens, **more)
    c.groups, c.shared = np.array(groups, np.int32), np.array(shared, np.int32)
    share(c, groups, shared)
    _ok(c.h.Share())
    return c


def plan(c, mostNew=0, stream=None):
    c.d["groups"], c.d["shared"] = c.b.up(c.groups), c.b.up(c.shared)
    _ok(c.h.PlanShared(c.d["rowStart"], c.d["lens"], len(c.new), c.bound, mostNew, c.d["groups"], c.d["shared"], len(c.shared), stream))


def check(c, mostNew=0, blind=False, **what):
    """blind: the other requests' entries for pages that are wholly shared are no pages -- they must not be asked for."""
    want = c.want(**what)
    if blind:
        for g, s in enumerate(c.shared):
            live = [r for r in range(c.groups[g], c.groups[g + 1]) if c.new[r] > 0]
            for r in live[1:]:
                c.table[r, :min(s, *(c.lens[r] - c.new[r] for r in live)) // c.page] = -1
    c.upload()
    plan(c, mostNew)
    c.attend(**what)
    _synced()
    c.compare(c.result(), *want)
    c.h.Close()


SHAPES = [(14, 2, 64), (32, 8, 128), (8, 8, 64), (9, 3, 128), (71, 1, 64)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("page", [8, 32])
def test_tokens_behind_prefixes(hip, bufs, fmt, heads, kv, hd, page):
    """Prefixes that end on, before and behind a page, from one position on; a group of one, requests of no group ahead, between and behind."""
    own = [1, 2, 9, 40, 1, 3, 3, 300, 17, 64, 65, 128, 1, 5, 5, 130, 2]
    groups, shared = [1, 4, 6, 7, 13, 15], [64, 1, 90, 333, 257]
    before = [0, 64, 64, 64, 1, 1, 90] + [333] * 6 + [257] * 2 + [0, 0]
    print(f"shared tokens fmt={fmt} {heads}/{kv}/{hd} page={page}", flush=True)
    c = make(fmt, hip, bufs, heads, kv, hd, page, [1] * 17, [a + b for a, b in zip(own, before)], groups, shared, seed=page, rowsMore=3, ld=4)
    check(c, mostNew=1, blind=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd", SHAPES[:4])
@pytest.mark.parametrize("mostNew", [0, 1, 130])
def test_rows_behind_prefixes(hip, bufs, fmt, heads, kv, hd, mostNew):
    """Requests of one and of many rows in one group: wide and narrow tiles on both sides; the most rows unknown, too low, and right."""
    new, own = [1, 5, 130, 1, 33, 64, 2, 70, 1, 1], [1, 9, 130, 70, 60, 64, 2, 71, 300, 1]
    before = [200] * 4 + [515] * 4 + [0, 0]
    print(f"shared rows fmt={fmt} {heads}/{kv}/{hd} mostNew={mostNew}", flush=True)
    check(make(fmt, hip, bufs, heads, kv, hd, 16, new, [a + b for a, b in zip(own, before)], [0, 4, 8], [200, 515], seed=mostNew), mostNew, blind=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd,n,length", [(32, 8, 128, 100, 2000), (14, 2, 64, 64, 9001), (8, 8, 64, 8, 700), (4, 1, 128, 3, 20011)])
def test_one_long_prefix(hip, bufs, fmt, heads, kv, hd, n, length):
    print(f"shared long fmt={fmt} {heads}/{kv}/{hd} {n} x {length}", flush=True)
    own = [1 + 7 * r % 60 for r in range(n)]
    check(make(fmt, hip, bufs, heads, kv, hd, 64, [1] * n, [length + x for x in own], [0, n], [length], seed=n), 1, blind=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_requests_without_rows(hip, bufs, fmt):
    """The first of a group, one in between, all of one; what they have for lengths and pages does not matter."""
    new, lens = [0, 1, 0, 2, 0, 0, 1, 1, 0, 1], [0, 150, 3, 160, 5, 200, 90, 300, 0, 290]
    c = make(fmt, hip, bufs, 8, 2, 64, 8, new, lens, [0, 4, 6, 7, 10], [0, 0, 0, 0], seed=1, rowsMore=40)
    for a, r, s in ((1, 3, 148), (7, 9, 280)):          # from the first with rows
        copy_rows(c, a, r, s)
    c.shared[:] = [148, 4, 80, 280]
    for r in (0, 2, 4, 5, 8):
        c.table[r, :] = -1
    check(c, 0, blind=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("mostNew", [0, 3])
def test_shared_lengths_that_are_cut(hip, bufs, fmt, mostNew):
    """Longer than what a request has ahead of its new rows, negative, past the largest length: the tables still name the same pages where that
    is said, so the result is every request's own."""
    new, lens = [1, 3, 1, 2, 70, 1, 1, 1], [100, 67, 200, 90, 90, 300, 301, 20]
    for shared in ([64, 21, 300, -7], [65, 1 << 30, 0x7fffffff, -(1 << 31)]):          # 64, 20 and 299 are what is ahead
        c = make(fmt, hip, bufs, 8, 2, 128, 16, new, lens, [0, 3, 5, 7, 8], [64, 20, 299, 0], seed=4)
        c.shared = np.array(shared, np.int32)
        check(c, mostNew)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (6, 3, 64)])
@pytest.mark.parametrize("cap,slopes,scale", [(50.0, False, 0.0), (2.0, False, 0.3), (0.0, True, 0.0), (30.0, True, 1.0)])
@pytest.mark.parametrize("many", [False, True])
def test_changed_scores(hip, bufs, fmt, heads, kv, hd, cap, slopes, scale, many):
    """A bias by distance is from each row's own position."""
    new, own = ([1, 70, 3, 1, 130, 1], [60, 70, 64, 1, 131, 300]) if many else ([1, 3, 1, 2, 1, 1], [60, 4, 64, 1, 131, 300])
    if not many:
        own[3] = 2
    before = [150] * 3 + [777] * 3
    sl = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32) if slopes else None
    print(f"shared scores fmt={fmt} {heads}/{kv}/{hd} cap={cap} slopes={slopes} many={many}", flush=True)
    check(make(fmt, hip, bufs, heads, kv, hd, 32, new, [a + b for a, b in zip(own, before)], [0, 3, 6], [150, 777], seed=int(cap), peak=4.0), blind=True, cap=cap, slopes=sl, scale=scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 60])
def test_peaks_on_either_side(hip, bufs, fmt, new):
    """Rows whose weight is nearly all in the shared part, or nearly all in their own: the parts' references are far apart."""
    c = make(fmt, hip, bufs, 8, 2, 64, 16, [new] * 4, [400 + new + 9 * r for r in range(4)], [0, 4], [400], seed=2, peak=2.0)
    c.q *= np.exp2(c.rng.integers(-3, 4, (c.q.shape[0], 1))).astype(np.float32)
    x = np.float32(c.K).reshape(-1, c.kv * c.hd)
    for r, f in enumerate((20.0, 0.01, 30.0, 1.0)):
        x[[c.where(r, j) for j in range(400, int(c.lens[r]))]] *= f
    if fmt == 8:
        c.set_rows("K", x)
    else:
        c.K = x.astype(c.kind)
    check(c, new, blind=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 60])
def test_pages_that_are_gone(hip, bufs, fmt, new):
    """In the shared part (all of it in one group), in a request's own, both."""
    c = make(fmt, hip, bufs, 8, 2, 64, 16, [new] * 6, [320 + new + 9 * r for r in range(6)], [0, 3, 6], [160, 320], seed=2)
    c.table[:3, [0, 2, 5, 9]] = [-1, c.nPages, 0x7fffffff, -(1 << 31)]
    c.table[3:, :20] = -1
    c.table[2, 11:] = -1
    c.table[4, :] = -1                            # nothing left at all
    check(c, new)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("new", [1, 70])
def test_values_that_are_no_numbers(hip, bufs, fmt, value, new):
    """In the shared part they reach every row of the group, in a request's own part the rows that see them."""
    for where in (5, 199, 200 + new - 1):
        c = make(fmt, hip, bufs, 8, 2, 64, 8, [new] * 4, [200 + new] * 4, [0, 3, 4], [200, 0], seed=3)
        for r in range(1 if where < 200 else 2):
            c.V[c.where(r, where), 5::7] = value
        if where < 200 and where >= 200 // 8 * 8:
            share(c, c.groups, c.shared)
        check(c, new)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,size", [(1100, 3), (4096, 64), (700, 1)])
def test_many_requests_and_groups(hip, bufs, fmt, n, size):
    print(f"shared many fmt={fmt} {n} in groups of {size}", flush=True)
    rng = np.random.default_rng(n)
    groups = list(range(0, n, size)) + [n]
    shared = rng.integers(0, 70, len(groups) - 1)
    lens = [int(shared[r // size]) + int(rng.integers(1, 30)) for r in range(n)]
    check(make(fmt, hip, bufs, 2, 1, 64, 8, [1] * n, lens, groups, shared, seed=n), 1)


def test_no_groups_is_a_plan_without(hip, bufs):
    c = make(1, hip, bufs, 8, 2, 64, 16, [1, 70, 3], [100, 90, 40], [0], [], seed=1)
    c.upload()
    c.plan()
    c.attend()
    _synced()
    plain = c.result()
    c.b.put(c.d["out"], c.out0)
    _ok(c.h.PlanShared(c.d["rowStart"], c.d["lens"], 3, c.bound, 0, None, None, 0))
    c.attend()
    _synced()
    assert np.array_equal(c.result(), plain)


def test_refusals(hip, bufs):
    c = Case(hip, bufs, 8, 2, 64, 1, 16, [1, 1], [100, 90])
    c.upload()
    one = bufs.up(np.array([0, 2, 1, 1], np.int32))

    def call(n=2, rows=2, most=1, groups=one, shared=one, nGroups=1, starts=c.d["rowStart"]):
        return c.h.PlanShared(starts, c.d["lens"], n, rows, most, groups, shared, nGroups)

    assert call() == -4 and "mg_paged_share" in E.last_error()
    _ok(c.h.Share())
    _ok(c.h.Share())
    for args, why in ((dict(n=3), "nReqs"), (dict(rows=3), "rows"), (dict(most=-1), "mostNew"), (dict(nGroups=-1), "nGroups"), (dict(nGroups=3), "nGroups"), (dict(groups=None), "4 bytes"),
                      (dict(shared=one.DevicePtr() + 2), "4 bytes"), (dict(starts=None), "4 bytes")):
        assert call(**args) == -2 and why in E.last_error(), (args, E.last_error())
    assert call() == 0
    _synced()


@pytest.mark.parametrize("fmt", FORMATS)
def test_arrays_that_are_no_groups(hip, bufs, fmt):
    """Group starts that run backwards, overlap or pass the requests, row starts that do: nothing is read or written outside."""
    c = make(fmt, hip, bufs, 8, 2, 64, 16, [5, 1, 4], [60, 33, 60], [0, 2, 3], [20, 0], seed=2, rowsMore=4)
    c.upload()
    for groups in ([2, 0, 3], [-5, 2, 2], [0, 4000, -1], [0x7fffffff, -(1 << 31), 3], [0, 3, 3]):
        for starts in (c.rowStart.tolist(), [7, 2, 9, -5], [-(1 << 31), 0x7fffffff, 3, 8]):
            for lens in ([60, 33, 60], [-4, 33, 1 << 30]):
                _ok(c.h.PlanShared(c.b.up(np.array(starts, np.int32)), c.b.up(np.array(lens, np.int32)), 3, c.bound, 0, c.b.up(np.array(groups, np.int32)), c.b.up(np.array([20, 30], np.int32)), 2))
                c.attend()
                _synced()
    check_again = c.want()
    c.b.put(c.d["out"], c.out0)
    plan(c)
    c.attend()
    _synced()
    c.compare(c.result(), *check_again)


@pytest.mark.parametrize("fmt", FORMATS)
def test_the_same_call_gives_the_same_bits(hip, bufs, fmt):
    c = make(fmt, hip, bufs, 32, 8, 128, 16, [1, 1, 30, 1], [5000, 5010, 5100, 333], [0, 3], [4900], seed=9)
    c.upload()
    plan(c)
    outs = []
    for _ in range(4):
        c.b.put(c.d["out"], c.out0)
        c.attend()
        _synced()
        outs.append(c.result())
    assert all(np.array_equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("fmt", FORMATS)
def test_plans_of_both_kinds_in_turn(hip, bufs, rt, fmt):
    """A call goes by the last plan: with and without groups, captured and not; one captured behind a plan of groups does nothing on another."""
    c = make(fmt, hip, bufs, 8, 2, 64, 8, [3, 1, 90, 1], [260, 233, 400, 50], [0, 3], [200], seed=2)
    c.upload()
    want = c.want()
    stream = rt.stream()

    def got():
        _synced()
        x = c.result()
        c.b.put(c.d["out"], c.out0)
        return x

    plan(c)
    alone = rt.capture(stream, lambda: c.attend(stream=stream))
    for _ in range(3):
        plan(c)
        c.attend()
        c.compare(got(), *want)
        rt.replay(alone, stream)
        c.compare(got(), *want)
        c.plan()
        c.attend()
        c.compare(got(), *want)
        rt.replay(alone, stream)
        assert (got() == 7.25).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_captured_decode(hip, bufs, rt, fmt):
    """Plan and attention of a step captured once; requests grow, end and come, groups' lengths change between the replays, with eager work of
    the same and of another kind in between."""
    heads, kv, hd, page, n = 8, 2, 64, 8, 6
    c = make(fmt, hip, bufs, heads, kv, hd, page, [1] * n, [120 + 3 * r for r in range(n)], [0, 4, 6], [96, 60], seed=7, rowsMore=70)
    c.upload()
    c.d["groups"], c.d["shared"] = c.b.up(c.groups), c.b.up(c.shared)
    stream = rt.stream()

    def step():
        _ok(c.h.PlanShared(c.d["rowStart"], c.d["lens"], n, c.bound, 0, c.d["groups"], c.d["shared"], 2, stream))
        c.attend(stream=stream)

    graph = rt.capture(stream, step)
    for t, (new, lens, shared) in enumerate([([1] * 6, [120, 123, 126, 129, 132, 135], [96, 60]), ([1, 1, 0, 1, 1, 1], [110, 123, 9, 120, 132, 100], [40, 60]),
                                             ([1, 1, 1, 20, 1, 50], [120, 123, 126, 129, 132, 135], [90, 55]), ([0, 0, 0, 0, 1, 2], [0, 0, 0, 0, 132, 135], [96, 60]),
                                             ([1] * 6, [120, 123, 126, 129, 132, 135], [0, 60]), ([0] * 6, [0] * 6, [96, 60]), ([1] * 6, [120, 123, 126, 129, 132, 135], [96, 60])]):
        c.new, c.lens, c.shared = np.array(new, np.int32), np.array(lens, np.int32), np.array(shared, np.int32)
        c.rowStart = np.concatenate(([0], np.cumsum(c.new))).astype(np.int32)
        c.rows = int(c.rowStart[-1])
        for name, a in (("rowStart", c.rowStart), ("lens", c.lens), ("shared", c.shared), ("out", c.out0)):
            c.b.put(c.d[name], a)
        E.KSync()
        rt.replay(graph, stream)
        got = c.result()
        c.compare(got, *c.want())
        c.b.put(c.d["out"], c.out0)
        _ok(c.h.PlanShared(c.d["rowStart"], c.d["lens"], n, c.bound, 0, c.d["groups"], c.d["shared"], 2))
        c.attend()
        _synced()
        assert np.array_equal(c.result(), got), t
        if t % 2:
            c.plan()
            c.attend()
            _synced()


def test_two_handles_on_two_streams(hip, bufs, rt):
    cs = [make(1, hip, bufs, 32, 8, 128, 16, [1, 30, 1], [3000, 3100, 2999 + k], [0, 3], [2900], seed=20 + k) for k in range(2)]
    ss = [rt.stream() for _ in cs]
    for c in cs:
        c.upload()
    E.KSync()
    for _ in range(3):
        for c, s in zip(cs, ss):
            plan(c, stream=s)
            c.attend(stream=s)
    for s in ss:
        rt.call("hipStreamSynchronize", s)
    for c in cs:
        c.compare(c.result(), *c.want())

