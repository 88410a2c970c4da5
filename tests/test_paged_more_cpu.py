"""What the 8-bit paged cache and the plans of shared prefixes accept, and what the rules say of them, on the host (paged_rules.h)."""
import ctypes

import numpy as np
import pytest

from mongoose_amd import engine as E
from mongoose_amd.lib import lib
from tests import paged_q8_model as Q
from tests.test_paged_cpu import GOOD, _run


def test_formats(tmp_path):
    out = _run(tmp_path, r"""
int main() {
    PagedGeo g{};
    for (int f : {0, 1, 8}) { const bool no = paged_geo(g, 14, 2, 64, 16, 100, f, 4, 64, 1000) != nullptr; std::printf("%d %zu\n", no, paged_pool_bytes(g)); }
    for (int f : {-1, 2, 3, 4, 7, 9, 16}) std::printf("%d", paged_geo(g, 14, 2, 64, 16, 100, f, 4, 64, 1000) != nullptr);
    const bool no = paged_geo(g, 8, 8, 128, 4096, 524287, 8, 4, 64, 1000) != nullptr;
    std::printf("\n%d %zu\n", no, paged_pool_bytes(g));
}
""").splitlines()
    assert out == [f"0 {1600 * 128 * 4}", f"0 {1600 * 128 * 2}", f"0 {1600 * (128 + 8)}", "1111111", f"0 {4096 * 524287 * (1024 + 32)}"]


@pytest.mark.parametrize("fmt", [2, 7, 9])
def test_create_names_the_formats(fmt):
    assert lib.mg_paged_create(*{**GOOD, "kvFormat": fmt}.values()) is None
    assert "8 (Q8)" in E.last_error()


def test_calls_without_a_handle():
    assert lib.mg_paged_pool_bytes(None) == 0
    assert lib.mg_paged_load(None, None, None, None, None, None, 0, 0, None, 0, None, 0, None) == -1
    assert lib.mg_paged_share(None) == -1
    assert lib.mg_paged_plan_shared(None, None, None, 0, 0, 0, None, None, 0, None) == -1


def test_arguments_that_are_refused(tmp_path):
    lines = _run(tmp_path, r"""
static char mem[4096] __attribute__((aligned(16)));
static void is(const char* what, const char* why) { std::printf("%s|%s\n", what, why ? why : "-"); }
int main() {
    PagedGeo g{};
    if (paged_geo(g, 14, 2, 64, 16, 100, 8, 4, 64, 1000)) return 1;
    char *a = mem, *b = mem + 64, *odd = mem + 2, *four = mem + 4;
    auto L = [&](const void* K, const void* t, int n, int rows, const void* k, int ldk, int ldv) { return paged_load_refusal(g, K, a, t, a, a, n, rows, k, ldk, b, ldv); };
    is("-", L(a, four, 4, 1 << 30, a, 128, 132)); is("-", L(nullptr, nullptr, 0, 5, nullptr, 0, 0)); is("-", L(nullptr, nullptr, 4, 0, nullptr, 0, 0));
    is("nReqs", L(a, a, 5, 1, a, 128, 128)); is("nReqs", L(a, a, -1, 1, a, 128, 128)); is("rows", L(a, a, 4, -1, a, 128, 128)); is("16 bytes", L(four, a, 4, 1, a, 128, 128));
    is("16 bytes", L(a, a, 4, 1, nullptr, 128, 128)); is("4 bytes", L(a, odd, 4, 1, a, 128, 128)); is("smaller", L(a, a, 4, 1, a, 124, 128)); is("multiple of 4", L(a, a, 4, 1, a, 128, 129));
    auto P = [&](const void* s, int n, int rows, int most, const void* gs, const void* sl, int ng) { return paged_plan_shared_refusal(g, s, a, n, rows, most, gs, sl, ng); };
    is("-", P(a, 4, 64, 0, a, b, 4)); is("-", P(a, 4, 64, 1 << 30, nullptr, nullptr, 0)); is("nReqs", P(a, 5, 64, 0, a, b, 1)); is("rows", P(a, 4, 65, 0, a, b, 1));
    is("mostNew", P(a, 4, 64, -1, a, b, 1)); is("nGroups", P(a, 4, 64, 0, a, b, -1)); is("nGroups", P(a, 4, 64, 0, a, b, 5)); is("pointer", P(nullptr, 4, 64, 0, a, b, 1));
    is("pointer", P(a, 4, 64, 0, odd, b, 1)); is("pointer", P(a, 4, 64, 0, a, nullptr, 1));
}
""").splitlines()
    assert len(lines) == 21
    for line in lines:
        want, got = line.split("|")
        assert (want in got) if want != "-" else got == "-", line


def test_what_load_writes_overlaps_nothing_that_it_reads(tmp_path):
    out = _run(tmp_path, r"""
static float mem[100000] __attribute__((aligned(16)));
int main() {
    PagedGeo g{};
    if (paged_geo(g, 14, 2, 64, 16, 10, 8, 4, 64, 100)) return 1;       // pools of 160 x (128 + 8) bytes: 5,440 floats; 7 entries a request's row of the table
    auto L = [&](int K, int V, int table, int starts, int lens, int n, int rows, int k, int ldk, int v, int ldv) {
        return paged_load_overlap(g, mem + K, mem + V, mem + table, mem + starts, mem + lens, n, rows, mem + k, ldk, mem + v, ldv); };
    auto is = [](const char* want, const char* got) { std::printf("%s|%s\n", want, got ? got : "-"); };
    const int K = 50000, V = 55440, T = 70000, S = 70028, N = 70033;
    is("-", L(K, V, T, S, N, 4, 8, 0, 128, 1024, 128));
    is("-", L(K, V, T, S, N, 4, 8, 0, 256, 128, 256));              // columns of one array
    is("-", L(K, K, T, S, N, 4, 8, 0, 128, 1024, 128));             // (K may be V)
    is("-", L(K, V, T, S, N, 4, 8, 60880, 128, 48976, 128));        // next to the pools
    is("kOut", L(K, V, T, S, N, 4, 8, 0, 256, 124, 256));
    is("kOut", L(K, V, T, S, N, 4, 8, 0, 128, 1020, 128));
    is("is read", L(K, V, T, S, N, 4, 8, 60876, 128, 0, 128));
    is("is read", L(K, V, T, S, N, 4, 8, 0, 128, 48980, 128));
    is("is read", L(K, V, T, S, N, 4, 8, T - 1020, 128, 0, 128));
    is("is read", L(K, V, T, S, N, 4, 8, 0, 128, S + 4, 128));
    is("is read", L(K, V, T, S, N, 4, 8, N + 3, 128, 0, 128));
    is("-", L(K, V, T, S, N, 4, 8, N + 4, 128, 0, 128));
    is("-", L(K, V, T, S, N, 0, 8, K, 128, K, 128));
    is("-", L(K, V, T, S, N, 4, 0, K, 128, K, 128));
}
""").splitlines()
    assert len(out) == 14
    for line in out:
        want, got = line.split("|")
        assert (want in got) if want != "-" else got == "-", line


def test_the_positions_of_a_request_behind_a_shared_prefix(tmp_path):
    """What its tiles' units cover: everything from the shared length on that its rows see; the group's tile of the shared length: all of it."""
    out = _run(tmp_path, r"""
int main() {
    for (int keys : {32, 64, 128}) for (int rows : {1, 3, 40}) for (int own : {rows, rows + 1, rows + 200}) for (int from : {0, 1, 63, 64, 65, 500}) for (int tileRows : {16, 128}) {
        const int len = from + own;
        for (int first = 0; first < rows * 3; first += tileRows) {
            PagedTile t{};
            t.rows = rows; t.len = len; t.first = first; t.tileRows = tileRows; t.unitKeys = keys; t.from = from;
            paged_units(t, 0, 3);
            const PagedSpan s = paged_span(rows, len, 0, 0, 3, first, tileRows, from);
            if (s.begin != from || s.end > len || t.units < 1) { std::printf("span %d..%d\n", s.begin, s.end); return 0; }
            for (int q = first; q < std::min(first + tileRows, rows * 3); q++) for (int j = from; j <= len - rows + q / 3; j++)
                if (j < s.begin || j >= s.end || j / keys < t.unit0 || j / keys >= t.unit0 + t.units) { std::printf("position %d\n", j); return 0; }
            if (from > 0) {                     // the rows as a group's, whose prefix is all of the length
                PagedTile g{};
                g.rows = rows; g.len = from; g.prefix = from; g.first = first; g.tileRows = tileRows; g.unitKeys = keys;
                paged_units(g, 0, 3);
                const PagedSpan a = paged_span(rows, from, from, 0, 3, first, tileRows);
                if (a.begin != 0 || a.end != from || g.unit0 != 0 || g.units != (from + keys - 1) / keys) { std::printf("group\n"); return 0; }
                for (int q = 0; q < rows; q++) for (int j = 0; j < from + 3; j++) if (paged_sees(from - rows + q, j, from, 0, from) != (j < from)) { std::printf("sees\n"); return 0; }
            }
        }
    }
    std::printf("ok\n");
}
""")
    assert out == "ok\n", out


def test_the_model_of_a_quantized_row():
    """By hand: a scale of 1, halves away from zero, the greatest at 127; zeros; a row with an infinity."""
    q, s = Q.held(np.array([[127, 0.5, -0.5, 1.49, -126.5, 2.5], [0, 0, 0, 0, 0, 0], [1, np.inf, 0, 0, 0, 0]], np.float32))
    assert q.tolist() == [[127, 1, -1, 1, -127, 3], [0] * 6, [0] * 6] and s[0] == 1 and s[1] == 0 and np.isnan(s[2])
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    q, s = Q.held(x)
    assert (np.abs(Q.values(q, s) - x) <= s[:, None] * (0.5 + 1e-6)).all() and (np.abs(q).max(1) == 127).all()
    kv = np.stack((q[:32], q[32:][:18].repeat(2, 0)[:32]), 1), np.stack((s[:32], s[32:][:18].repeat(2)[:32]), 1)
    back = Q.from_pool(Q.pool(*kv, 8), 32, 2, 64, 8)
    assert np.array_equal(back[0], kv[0]) and np.array_equal(back[1], kv[1])


def test_a_released_tensor_is_no_missing_argument():
    gone, live, h = E.Tensor(None, None, 64, [16]), E.Tensor(None, 64, 64, [16]), E.HIPPaged(None)
    assert h.PlanShared(live, live, 1, 1, 0, live, live, 1) == -1 and "NULL handle" in E.last_error()
    for call in (lambda: h.PlanShared(live, live, 1, 1, 0, gone, live, 1), lambda: h.PlanShared(live, live, 1, 1, 0, live, gone, 1),
                 lambda: h.Load(live, live, live, live, live, 1, 1, live, 64, gone, 64)):
        with pytest.raises(ctypes.ArgumentError, match="released"):
            call()
