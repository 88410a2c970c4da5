"""Where the workers of a plan of groups leave their shares, and how many there may be, and which plans an attention call takes for its own, on the
host (paged_rules.h)."""
from tests.test_paged_cpu import _run

# The workers of every tile as the plan has them: `units` of each tile, `workers` a KV head
PLAN = r"""
struct Pair { int tile, worker; };
static std::vector<Pair> pairs_of(const std::vector<int>& units, int most, int least) {
    std::vector<PagedTile> tiles(units.size());
    int cost = 0;
    for (size_t i = 0; i < units.size(); i++) { tiles[i].units = units[i]; tiles[i].cost0 = cost; cost += paged_cost(tiles[i]); }
    std::vector<Pair> out;
    const int n = (int)units.size(), workers = std::max(1, std::min(most, cost));
    for (int i = 0, next = 0; i < n; i++) {
        int w0, w1;
        if (paged_few(n, most)) {
            w0 = next;
            next += paged_workers_for(tiles[i], cost, n, most, least);
            w1 = next - 1;
        } else {
            const int x = tiles[i].cost0 + PAGED_TILE_COST;
            w0 = paged_worker_of(cost, workers, x);
            w1 = paged_worker_of(cost, workers, x + tiles[i].units - 1);
        }
        for (int w = w0; w <= w1; w++) out.push_back({i, w});
    }
    return out;
}
// Pairs that have another's place, and 1 where one is out of `places`
template <typename F> static int meet(const std::vector<Pair>& pairs, int places, bool& out, F place) {
    std::vector<int> at(places, 0);
    int n = 0;
    for (auto& p : pairs) {
        const int x = place(p);
        if (x < 0 || x >= places) { out = true; continue; }
        n += at[x]++ > 0;
    }
    return n;
}
"""


def test_no_two_shares_have_one_place(tmp_path):
    """Tiles from one to many times the workers, of equal and of very different lengths.  Two places a worker -- one for a tile that goes on
    from the worker before, one for a tile of its own start -- would not do for tiles of one worker."""
    out = _run(tmp_path, PLAN + r"""
int main() {
    unsigned seed = 1;
    auto next = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); };
    long long plans = 0, before = 0;
    for (int workers : {1, 2, 7, 32, 64, 128, 512}) for (int n : {1, 2, 3, 15, 16, 17, 31, 32, 33, 40, 63, 64, 65, 80, 100, 128, 129, 366, 1000, 2100}) for (int kind = 0; kind < 6; kind++) for (int least : {1, 3}) {
        std::vector<int> units(n);
        for (int i = 0; i < n; i++)
            units[i] = kind == 0 ? 1 : kind == 1 ? 32 : kind == 2 ? 1 + next(100) : kind == 3 ? (i == n / 2 ? 5000 : 1) : kind == 4 ? (next(4) ? 1 + next(3) : 300 + next(900)) : i % 2 ? 1 : 63;
        const auto pairs = pairs_of(units, workers, least);
        bool out = false;
        if (meet(pairs, n + workers, out, [](Pair p) { return paged_place(p.tile, p.worker); }) || out) { std::printf("%d tiles, %d workers, kind %d\n", n, workers, kind); return 0; }
        std::vector<int> first(n, -1);
        for (auto& p : pairs) if (first[p.tile] < 0) first[p.tile] = p.worker;
        before += meet(pairs, 2 * workers, out, [&](Pair p) { return p.worker * 2 + (p.worker == first[p.tile]); }) > 0;
        plans++;
    }
    std::printf("%lld %d\n", plans, before > 200);
}
""")
    assert out == "1680 1\n", out


def test_groups_have_no_more_tiles_than_there_is_room_for(tmp_path):
    """Any cut of the rows into groups of two requests and more."""
    out = _run(tmp_path, r"""
int main() {
    unsigned seed = 5;
    auto next = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); };
    for (int group : {1, 3, 4, 7, 128}) for (int maxReqs : {1, 2, 3, 64, 4096}) for (int maxRows : {1, 2, 5, 17, 64, 256, 257, 4096}) {
        PagedGeo g{};
        if (paged_geo(g, group, 1, 64, 16, 100, 1, maxReqs, maxRows, 1000)) return 1;
        const int most = paged_group_tiles(g);
        for (int turn = 0; turn < 200; turn++) {
            int left = 1 + next(maxRows), reqs = maxReqs, tiles = 0;
            const int tileRows = left * group <= 256 ? PAGED_NARROW : PAGED_WIDE;
            while (left >= 2 && reqs >= 2) {
                const int rows = turn == 0 ? 2 : std::min(left, 2 + next(turn % 3 ? 40 : left));
                tiles += (rows * group + tileRows - 1) / tileRows;
                left -= rows;
                reqs -= 2;
            }
            if (tiles > most) { std::printf("group %d, %d requests, %d rows: %d > %d\n", group, maxReqs, maxRows, tiles, most); return 0; }
        }
    }
    std::printf("ok\n");
}
""")
    assert out == "ok\n", out


def test_plans_of_other_kinds_of_tiles_are_other_plans(tmp_path):
    """Two plans are one where all that their tiles follow from is: also what mostNew says of the requests, where their tiles go by it."""
    out = _run(tmp_path, r"""
int main() {
    const PagedPlanFor a{4, 75, 0, 1, 256};
    for (PagedPlanFor b : {PagedPlanFor{5, 75, 0, 1, 256}, {4, 76, 0, 1, 256}, {4, 75, 9, 1, 256}, {4, 75, 0, 2, 256}, {4, 75, 0, 1, 1 << 27}}) std::printf("%d%d ", a.is(b), b.is(a));
    std::printf("%d\n", a.is(a));
    for (int format : {0, 1, 8}) {
        PagedGeo g{};
        if (paged_geo(g, 8, 2, 64, 8, 100, format, 4, 5000, 1000)) return 1;
        auto made = [&](int rows, int most) { return PagedPlanFor{4, rows, 0, 1, paged_narrow_rows_shared(g, rows, most, false)}; };
        std::printf("%d %d %d %d %d\n", made(75, 0).is(made(75, 1)), made(75, 0).is(made(75, 70)), made(75, 1).is(made(75, 64)), made(64, 0).is(made(64, 1)), made(5000, 5).is(made(5000, 0)));
        // two plans that are one agree on which requests have narrow tiles
        for (int rows : {1, 64, 65, 1024, 1025, 5000}) for (int x : {0, 1, 4, 5, 8, 9, 64, 65, 5000}) for (int y : {0, 1, 4, 5, 8, 9, 64, 65, 5000})
            if (made(rows, x).is(made(rows, y)) != (paged_narrow_rows_shared(g, rows, x, false) == paged_narrow_rows_shared(g, rows, y, false))) std::printf("%d %d %d\n", rows, x, y);
    }
}
""").splitlines()
    # (75 rows: 300 of a KV head; up to 256 all are narrow; 5,000: 5 tokens are 20, past the line of 16 and not that of 32)
    assert out == ["00 00 00 00 00 1", "0 1 1 1 1", "0 1 1 1 1", "0 1 1 1 0"], out
