"""What the calls on a paged KV cache refuse, and the positions that a token sees, on the host (paged_rules.h)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from mongoose_amd import engine as E
from mongoose_amd.lib import lib
from tests import paged_model as P

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mongoose_amd", "csrc")


def _run(tmp_path, source):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include "paged_rules.h"\n#include <algorithm>\n#include <cstdio>\n#include <vector>\nusing namespace mg;\n' + source)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout


GOOD = dict(nHeads=14, nKVHeads=2, headDim=64, pageSize=16, nPages=100, kvFormat=0, maxReqs=4, maxRows=64, maxLen=1000)


@pytest.mark.parametrize("change,why", [
    (dict(headDim=80), "headDim"), (dict(nHeads=15), "multiple"), (dict(nKVHeads=0), "multiple"), (dict(nHeads=-14), "multiple"),
    (dict(nHeads=129, nKVHeads=1), "128 query heads"), (dict(pageSize=0), "power of two"), (dict(pageSize=24), "power of two"),
    (dict(pageSize=8192), "power of two"), (dict(pageSize=4), "power of two"), (dict(nPages=0), "nPages"), (dict(nPages=1 << 27), "2^31"), (dict(kvFormat=2), "kvFormat"),
    (dict(maxReqs=0), "maxReqs"), (dict(maxReqs=4097), "maxReqs"), (dict(maxRows=0), "maxRows"), (dict(maxRows=(1 << 20) + 1), "maxRows"),
    (dict(maxLen=0), "maxLen"), (dict(maxLen=(1 << 24) + 1), "maxLen"),
    (dict(maxRows=1 << 20, maxLen=1 << 18), "2^40"),
    (dict(maxReqs=4096, maxLen=1 << 23), "2^34")])
def test_create_refuses(change, why):
    assert lib.mg_paged_create(*{**GOOD, **change}.values()) is None
    assert why in E.last_error(), E.last_error()


def test_calls_without_a_handle():
    assert lib.mg_paged_table_width(None) == 0
    lib.mg_paged_destroy(None)
    assert lib.mg_paged_plan(None, None, None, 0, 0, 0, None, None) == -1
    assert lib.mg_paged_tables(None, None, 0, None, None, None, None, None, None, 0, None, None, None, None, None) == -1
    assert lib.mg_paged_store(None, None, None, None, 0, 0, 0, None, 0, None, None, None, None, 0, None, None, 0, None) == -1
    assert lib.mg_paged_attention(None, None, 0, None, None, None, None, 0, 0.0, 0.0, None, None) == -1


def test_arguments_that_are_refused(tmp_path):
    out = _run(tmp_path, r"""
static char mem[4096] __attribute__((aligned(16)));
static void is(const char* what, const char* why) { std::printf("%s|%s\n", what, why ? why : "-"); }
int main() {
    PagedGeo g{};
    if (paged_geo(g, 14, 2, 64, 16, 100, 0, 4, 64, 1000)) return 1;
    std::printf("%d %d %d %d\n", g.group, g.kvDim, g.pageShift, g.width);
    char *a = mem, *b = mem + 64, *odd = mem + 2, *four = mem + 4;
    auto T = [&](const void* nl, int n, const void* l, const void* lo, const void* ring, int rows, const void* slots) {
        return paged_tables_refusal(g, nl, n, l, lo, a, ring, a, a, rows, a, slots, a, a); };
    is("-", T(a, 4, b, b, a, 64, a)); is("-", T(nullptr, 0, nullptr, nullptr, a, 0, nullptr)); is("nReqs", T(a, 5, b, b, a, 64, a));
    is("nReqs", T(a, -1, b, b, a, 64, a)); is("rows", T(a, 4, b, b, a, 65, a)); is("rows", T(a, 4, b, b, a, -1, a)); is("pointer", T(nullptr, 1, b, b, a, 1, a));
    is("pointer", T(a, 1, odd, b, a, 1, a)); is("pointer", T(a, 1, b, b, nullptr, 1, a)); is("pointer", T(a, 1, b, b, a, 1, nullptr)); is("same array", T(a, 1, b, a, a, 1, a));
    auto S = [&](const void* q, int ldq, int ldk, int ldv, int ldo, const void* K, const void* V, const void* slots, int rows, int tab) {
        return paged_store_refusal(g, q, a, a, ldq, ldk, ldv, a, ldo, K, V, slots, a, rows, a, a, tab); };
    is("-", S(a, 896, 128, 128, 896, a, b, four, 64, 1)); is("-", S(nullptr, 0, 0, 0, 0, nullptr, nullptr, nullptr, 0, 0)); is("16 bytes", S(four, 896, 128, 128, 896, a, b, a, 1, 1));
    is("16 bytes", S(a, 896, 128, 128, 896, nullptr, b, a, 1, 1)); is("4 bytes", S(a, 896, 128, 128, 896, a, b, odd, 1, 1)); is("smaller", S(a, 895, 128, 128, 896, a, b, a, 1, 1));
    is("smaller", S(a, 896, 124, 128, 896, a, b, a, 1, 1)); is("smaller", S(a, 896, 128, -4, 896, a, b, a, 1, 1)); is("smaller", S(a, 896, 128, 128, 892, a, b, a, 1, 1));
    is("multiple of 4", S(a, 898, 128, 128, 896, a, b, a, 1, 1)); is("no rows", S(a, 896, 128, 128, 896, a, b, a, 1, 0)); is("same array", S(a, 896, 128, 128, 896, a, a, a, 1, 1));
    is("rows", S(a, 896, 128, 128, 896, a, b, a, 65, 1)); is("rows", S(a, 896, 128, 128, 896, a, b, a, -1, 1));
    is("-", paged_plan_refusal(g, a, b, 4, 64, 0, nullptr)); is("-", paged_plan_refusal(g, a, nullptr, 0, 0, 0, nullptr)); is("nReqs", paged_plan_refusal(g, a, b, 5, 64, 0, nullptr));
    is("rows", paged_plan_refusal(g, a, b, 4, 65, 0, nullptr)); is("window", paged_plan_refusal(g, a, b, 4, 64, -1, nullptr)); is("pointer", paged_plan_refusal(g, nullptr, b, 4, 64, 0, nullptr));
    is("pointer", paged_plan_refusal(g, a, nullptr, 1, 64, 0, nullptr)); is("prefixLens", paged_plan_refusal(g, a, b, 1, 64, 0, odd));
    auto A = [&](const void* q, int ldq, const void* K, const void* t, const void* o, int ldo, float sc, float cap, const void* sl) { return paged_attention_refusal(g, q, ldq, K, b, t, o, ldo, sc, cap, sl); };
    is("-", A(a, 896, a, four, b, 900, 0.f, 0.f, nullptr)); is("-", A(a, 896, a, a, b, 896, 0.1f, 50.f, four)); is("16 bytes", A(four, 896, a, a, b, 896, 0, 0, nullptr));
    is("16 bytes", A(a, 896, a, a, nullptr, 896, 0, 0, nullptr)); is("4 bytes", A(a, 896, a, odd, b, 896, 0, 0, nullptr)); is("4 bytes", A(a, 896, a, a, b, 896, 0, 0, odd));
    is("smaller", A(a, 892, a, a, b, 896, 0, 0, nullptr)); is("smaller", A(a, 896, a, a, b, 0, 0, 0, nullptr)); is("multiple of 4", A(a, 897, a, a, b, 896, 0, 0, nullptr));
    is("scale", A(a, 896, a, a, b, 896, -1.f, 0, nullptr)); is("scale", A(a, 896, a, a, b, 896, __builtin_nanf(""), 0, nullptr)); is("scale", A(a, 896, a, a, b, 896, __builtin_inff(), 0, nullptr));
    is("softcap", A(a, 896, a, a, b, 896, 0, -1.f, nullptr)); is("softcap", A(a, 896, a, a, b, 896, 0, __builtin_nanf(""), nullptr)); is("same array", A(a, 896, a, a, a, 896, 0, 0, nullptr));
}
""")
    lines = out.splitlines()
    assert lines[0] == "7 128 4 63"
    for line in lines[1:]:
        want, got = line.split("|")
        assert (want in got) if want != "-" else got == "-", line
    assert len(lines) == 49


def test_what_a_token_sees(tmp_path):
    out = _run(tmp_path, r"""
int main() {
    for (int len : {1, 7}) for (int w : {0, 1, 3, 100}) for (int pre : {0, 1, 4, 7}) for (int i = -1; i < len; i++) for (int j = 0; j < 9; j++) std::printf("%d", paged_sees(i, j, len, w, pre));
    std::printf("\n%u %u\n", sat_add(0x7fffffffu, 0x7fffffffu), sat_add(3, 4));
    std::printf("%d %d %d %d\n", paged_pages(0, 4), paged_pages(1, 4), paged_pages(16, 4), paged_pages(0x7fffffff, 0));
}
""").splitlines()
    want = "".join(str(int(P.sees(i, np.int64(j), n, w, pre))) for n in (1, 7) for w in (0, 1, 3, 100) for pre in (0, 1, 4, 7) for i in range(-1, n) for j in range(9))
    assert out[0] == want
    assert out[1:] == ["2147483647 7", "0 1 1 2147483647"]


def test_the_model_of_a_step():
    """The block tables' plain form itself, on a step worked out by hand: pages of 4, a request that grows into a new page, one
    that ends and one that is new."""
    table = np.array([[5, 9], [2, 7], [9, 9]], np.int32)
    ring = P.Ring([0, 1, 3, 4, 6, 8, -7, -7, -7, -7], 4, 2)          # free: 6, 8
    got = P.tables(np.array([2, -1, 1], np.int32), np.array([3, 5, 0], np.int32), table, ring, 4, 8, 4)
    assert got["table"].tolist() == [[5, 6], [2, 7], [8, 9]]
    assert got["slots"].tolist() == [23, 24, 32, -1] and got["positions"].tolist() == [3, 4, 0, -1]
    assert got["rowStart"].tolist() == [0, 2, 2, 3] and got["lensOut"].tolist() == [5, 0, 1]
    assert got["ring"].tolist() == [0, 1, 3, 4, 6, 8, 2, 7, -7, -7] and got["ringState"].tolist() == [6, 2]
    assert got["counts"].tolist() == [3, 2, 2, 0]


@pytest.mark.parametrize("few", [0, 1])
@pytest.mark.parametrize("tileRows,unitKeys,least", [(16, 128, 1), (16, 64, 2), (128, 64, 2), (128, 32, 3)])
def test_the_plan_gives_every_unit_to_one_worker(tmp_path, tileRows, unitKeys, least, few):
    """Random batches: every position that a token sees is in its tile's units, every unit in exactly one worker's share, the workers of
    a tile are all of worker0 .. worker1, no two partial results share a place, and a tile without units has one worker."""
    out = _run(tmp_path, r"""
#include <random>
#include <set>
int main() {
    std::mt19937 rng(7);
    auto rnd = [&](int a, int b) { return a + (int)(rng() %% (unsigned)(b - a + 1)); };
    long long split = 0, empty = 0;
    for (int it = 0; it < 400; it++) {
        const int group = rnd(1, 9), n = rnd(1, 12), window = rnd(0, 2) ? 0 : rnd(1, 300), most = rnd(1, 3) == 1 ? rnd(1, 3) : rnd(1, 200);
        std::vector<PagedTile> tiles;
        long long cost = 0;
        for (int r = 0; r < n; r++) {
            const int rows = rnd(0, 2) ? rnd(0, 3) : rnd(0, 60), len = rnd(0, 20) ? rnd(0, 40) + rnd(0, 1) * rnd(0, 3000) : 0, prefix = rnd(0, 3) ? 0 : rnd(0, len);
            for (int f = 0; f < rows * group; f += %(tileRows)d) {
                PagedTile t{};
                t.req = r; t.rows = rows; t.len = len; t.prefix = prefix; t.first = f; t.index = (int)tiles.size();
                t.tileRows = %(tileRows)d; t.unitKeys = %(unitKeys)d;
                paged_units(t, window, group);
                t.cost0 = (int)cost;
                cost += paged_cost(t);
                for (int q = f; q < std::min(f + t.tileRows, rows * group); q++)
                    for (int j = 0; j < len; j++)
                        if (paged_sees(len - rows + q / group, j, len, window, prefix) && (j / t.unitKeys < t.unit0 || j / t.unitKeys >= t.unit0 + t.units)) { std::printf("position %%d\n", j); return 0; }
                const PagedSpan s = paged_span(rows, len, prefix, window, group, f, t.tileRows);
                if (s.begin < 0 || s.end > len || s.pos1 >= len) { std::printf("span\n"); return 0; }
                tiles.push_back(t);
            }
        }
        if (tiles.empty()) continue;
        const int C = (int)cost, T = (int)tiles.size(), given = %(few)d ? 2 * T + most : most;
        if (paged_few(T, given) != %(few)d) continue;
        int workers = std::max(1, std::min(given, C));
        std::set<int> places;
        std::vector<int> seen(T, 0), zero(T, 0), done(T, 0), owner;
        if (%(few)d) {
            workers = 0;
            for (auto& t : tiles) {
                const int n = paged_workers_for(t, C, T, given, %(least)d);
                if (n < 1 || (n > 1 && t.units / n < %(least)d)) { std::printf("count\n"); return 0; }
                t.worker0 = workers; t.worker1 = workers + n - 1;
                workers += n;
                owner.insert(owner.end(), n, t.index);
            }
            if (workers > given) { std::printf("too many\n"); return 0; }
        } else for (auto& t : tiles) if (t.units) { t.worker0 = paged_worker_of(C, workers, t.cost0 + PAGED_TILE_COST); t.worker1 = paged_worker_of(C, workers, t.cost0 + PAGED_TILE_COST + t.units - 1); }
        for (int w = 0; w < workers; w++) {
            int a = paged_share(C, workers, w), b = paged_share(C, workers, w + 1);
            if (%(few)d) {
                const PagedTile& t = tiles[owner[w]];
                const int n = t.worker1 - t.worker0 + 1, k = w - t.worker0;
                a = paged_part(t, n, k);
                b = k + 1 < n ? paged_part(t, n, k + 1) : t.cost0 + paged_cost(t);
            }
            size_t i = tiles.size() - 1;
            while (tiles[i].cost0 > a) i--;
            for (; i < tiles.size() && tiles[i].cost0 < b; i++) {
                const PagedTile& t = tiles[i];
                const int u0 = paged_unit_at(t, a), u1 = paged_unit_at(t, b);
                if (t.units == 0) { zero[i] += a <= t.cost0; continue; }
                if (u0 > u1 || (u0 < u1 && u0 != seen[i])) { std::printf("order\n"); return 0; }
                if ((u0 < u1) != (w >= t.worker0 && w <= t.worker1)) { std::printf("workers %%d %%d..%%d\n", w, t.worker0, t.worker1); return 0; }
                if (u0 < u1) { seen[i] = u1; done[i]++; }
                if (u0 < u1 && t.worker0 != t.worker1) { split++; if (!places.insert(w * 2 + (w == t.worker0)).second) { std::printf("place\n"); return 0; } }
            }
        }
        for (size_t i = 0; i < tiles.size(); i++) {
            if (tiles[i].units == 0 ? zero[i] != 1 : seen[i] != tiles[i].units || done[i] != tiles[i].worker1 - tiles[i].worker0 + 1) { std::printf("left out\n"); return 0; }
            empty += tiles[i].units == 0;
        }
    }
    std::printf(split > 300 && empty > 10 ? "ok\n" : "too few %%lld %%lld\n", split, empty);
}
""" % dict(tileRows=tileRows, unitKeys=unitKeys, least=least, few=few))
    assert out == "ok\n", out


def test_scales_and_caps_without_a_reciprocal_are_refused(tmp_path):
    out = _run(tmp_path, r"""
static char mem[256] __attribute__((aligned(16)));
int main() {
    PagedGeo g{};
    if (paged_geo(g, 8, 2, 64, 16, 100, 1, 4, 64, 1000)) return 1;
    for (float x : {1e-30f, 1e30f, 1e-31f, 1e-40f, 1e31f}) {
        const char* a = paged_attention_refusal(g, mem, 512, mem, mem, mem, mem + 64, 512, x, 0.f, nullptr);
        const char* b = paged_attention_refusal(g, mem, 512, mem, mem, mem, mem + 64, 512, 0.f, x, nullptr);
        std::printf("%d%d ", a != nullptr, b != nullptr);
    }
}
""")
    assert out == "00 00 11 11 11 "


def test_what_store_writes_overlaps_nothing_that_it_reads(tmp_path):
    out = _run(tmp_path, r"""
static float mem[400000] __attribute__((aligned(16)));
int main() {
    // strided rows against every float of them
    for (int it = 0; it < 60000; it++) {
        unsigned x = it * 2654435761u;
        auto rnd = [&](int n) { x = x * 1664525u + 1013904223u; return (int)((x >> 8) % (unsigned)n); };
        const int wa = 1 + rnd(5), wb = 1 + rnd(5), lda = wa + rnd(7), ldb = rnd(2) && lda >= wb ? lda : wb + rnd(7), rows = rnd(5), at = rnd(80);
        bool meet = false, extent = false;
        for (int i = 0; i < rows; i++) for (int j = 0; j < rows; j++) for (int s = 0; s < wa; s++) for (int t = 0; t < wb; t++) meet |= 40 + i * lda + s == at + j * ldb + t;
        extent = rows > 0 && 40 < at + (rows - 1) * ldb + wb && at < 40 + (rows - 1) * lda + wa;
        if (paged_rows_meet(mem + 40, lda, wa, mem + at, ldb, wb, rows) != (lda == ldb ? meet : extent)) { std::printf("%d %d %d %d rows %d at %d\n", lda, wa, ldb, wb, rows, at); return 0; }
    }
    PagedGeo g{};
    if (paged_geo(g, 14, 2, 64, 16, 10, 1, 4, 64, 100)) return 1;       // rows of 896, 128 and 128; pools of 10,240 floats' bytes
    auto S = [&](int q, int k, int v, int ld, int o, int ldo, int K, int V, int rows) { return paged_store_overlap(g, mem + q, mem + k, mem + v, ld, ld, ld, mem + o, ldo, mem + K, mem + V, rows); };
    auto is = [](const char* want, const char* got) { std::printf("%s|%s\n", want, got ? got : "-"); };
    const int K = 200000, V = K + 10240;
    is("-", S(0, 896, 1024, 1152, 0, 1152, K, V, 8));              // in place
    is("-", S(0, 896, 1024, 1152, 100000, 896, K, V, 8));
    is("-", S(0, 896, 1024, 2048, 1152, 2048, K, V, 8));           // columns behind
    is("-", S(0, 896, 1024, 1152, 0, 896, K, V, 1));               // one row has no stride
    is("-", S(0, 896, 1024, 1152, 0, 896, K, K, 0));
    is("same stride", S(0, 896, 1024, 1152, 0, 896, K, V, 8));
    is("same stride", S(0, 896, 1024, 1152, 4, 1152, K, V, 8));
    is("same stride", S(0, 896, 1024, 1152, 1152, 1152, K, V, 8));       // the next row
    is("-", S(0, 896, 1024, 1152, 1152 * 8, 1152, K, V, 8));
    is("k or v", S(0, 896, 1024, 2048, 1148, 2048, K, V, 8));
    is("k or v", S(100000, 100896, 1024, 1152, 512, 1152, K, V, 1));
    is("K and V", S(0, 896, 1024, 1152, 0, 1152, K, K + 10236, 8));
    is("the rows", S(0, 896, 1024, 1152, 0, 1152, 1152 * 7 + 1148, V, 8));
    is("the rows", S(0, 896, 1024, 1152, 100000, 896, K, 100000 + 7 * 896, 8));
}
""").splitlines()
    assert len(out) == 14, out
    for line in out:
        want, got = line.split("|")
        assert (want in got) if want != "-" else got == "-", line


def test_what_attention_writes_overlaps_nothing_that_it_reads(tmp_path):
    out = _run(tmp_path, r"""
static float mem[400000] __attribute__((aligned(16)));
int main() {
    PagedGeo g{};
    if (paged_geo(g, 14, 2, 64, 16, 10, 0, 4, 64, 100)) return 1;       // rows of 896; pools of 20,480 floats
    auto A = [&](int q, int ldq, int K, int V, int o, int ldo, int rows) { return paged_attention_overlap(g, mem + q, ldq, mem + K, mem + V, mem + o, ldo, rows); };
    auto is = [](const char* want, const char* got) { std::printf("%s|%s\n", want, got ? got : "-"); };
    is("-", A(0, 1792, 200000, 220480, 896, 1792, 64));        // other columns
    is("-", A(0, 896, 200000, 200000, 57344, 896, 64));        // one behind the other; K may be V
    is("overlaps q", A(0, 896, 200000, 220480, 57340, 896, 64));
    is("overlaps q", A(0, 1792, 200000, 220480, 892, 1792, 64));
    is("overlaps q", A(0, 1152, 200000, 220480, 1152, 1152, 2));
    is("overlaps q", A(4, 1152, 200000, 220480, 0, 1152, 1));
    is("-", A(0, 1152, 200000, 220480, 1152, 1152, 1));
    is("K or V", A(0, 896, 200000, 220480, 240956, 896, 3));
    is("K or V", A(0, 896, 200000, 220480, 199108, 896, 2));
    is("-", A(0, 896, 200000, 220480, 240960, 896, 3));
}
""").splitlines()
    assert len(out) == 10, out
    for line in out:
        want, got = line.split("|")
        assert (want in got) if want != "-" else got == "-", line


def test_arrays_of_the_tables_that_overlap(tmp_path):
    """Eleven arrays one behind the other; each in turn moved onto the last entry of each other one."""
    out = _run(tmp_path, r"""
static int mem[4000];
int main() {
    PagedGeo g{};
    if (paged_geo(g, 14, 2, 64, 16, 100, 0, 4, 64, 1000)) return 1;
    const int n = 3, rows = 7, size[11] = {n, n, n, n * 63, 100, 2, 2, n + 1, rows, rows, 4};      // in the order of the arguments
    auto call = [&](const int* at, int n, int rows) {
        const int* p[11];
        for (int i = 0; i < 11; i++) p[i] = mem + at[i];
        return paged_tables_overlap(g, p[0], n, p[1], p[2], p[3], p[4], p[5], p[6], rows, p[7], p[8], p[9], p[10]) != nullptr;
    };
    int at[11], end = 0;
    for (int i = 0; i < 11; i++) { at[i] = end; end += size[i]; }
    std::printf("%d", call(at, n, rows));
    for (int i = 0; i < 11; i++) for (int j = 0; j < 11; j++) if (i != j) {
        int moved[11];
        std::copy(at, at + 11, moved);
        moved[i] = at[j] + size[j] - 1;
        moved[i] = std::max(moved[i], 0);
        int other = 1000;                               // (nothing else is in the way)
        for (int k = 0; k < 11; k++) if (k != i && k != j) { moved[k] = other; other += size[k]; }
        const bool reads = (i == 0 || i == 1 || i == 5) && (j == 0 || j == 1 || j == 5);        // newLens, lens, ringState are only read
        if (call(moved, n, rows) == reads) { std::printf(" %d onto %d", i, j); return 0; }
    }
    at[2] = at[1]; at[6] = at[5];
    std::printf("%d", call(at, n, rows));               // in place
    int none[11] = {};
    none[4] = 100; none[5] = none[6] = 300; none[7] = 310; none[10] = 320;
    std::printf("%d\n", call(none, 0, 0));               // no requests, no rows: those arrays are nothing
}
""")
    assert out == "000\n", out


@pytest.mark.parametrize("window", [1, 3, 1 << 24, (1 << 31) - 2, (1 << 31) - 1])
def test_windows_up_to_the_largest(tmp_path, window):
    """Requests with more rows than positions among them: their first rows are at negative positions."""
    out = _run(tmp_path, r"""
int main() {
    const int w = paged_window(%d, 1000);
    for (int rows : {1, 5, 40}) for (int len : {0, 1, 3, 40, 1000}) for (int prefix : {0, 2}) for (int first = 0; first < rows * 3; first += 16) {
        if (prefix > len) continue;
        const PagedSpan s = paged_span(rows, len, prefix, w, 3, first, 16);
        for (int q = first; q < std::min(first + 16, rows * 3); q++) for (int j = 0; j < len; j++) {
            const int i = len - rows + q / 3;
            const bool sees = (j <= i && (long long)j > (long long)i - %dll) || j < prefix;
            if (sees != paged_sees(i, j, len, w, prefix) || (sees && (j < s.begin || j >= s.end))) { std::printf("%%d of %%d at %%d: %%d\n", rows, len, i, j); return 0; }
        }
    }
    std::printf("ok\n");
}
""" % (window, window))
    assert out == "ok\n", out


def test_a_released_tensor_is_no_missing_argument():
    """None for slopes or prefixLens asks for another formula; a tensor that is gone must not."""
    gone, live, h = E.Tensor(None, None, 64, [16]), E.Tensor(None, 64, 64, [16]), E.HIPPaged(None)
    assert h.Plan(live, live, 1, 1, 0, live) == -1 and "NULL handle" in E.last_error()
    for call in (lambda: h.Plan(live, live, 1, 1, 0, gone), lambda: h.Attention(live, 64, live, live, live, live, 64, slopes=gone),
                 lambda: h.Store(live, live, live, 64, 64, 64, gone, 64, live, live, live, live, 1, live, live, 1),
                 lambda: h.Tables(live, 1, live, live, live, live, live, live, 1, live, live, live, gone)):
        with pytest.raises(ctypes.ArgumentError, match="released"):
            call()
