"""Which stretches of positions no row of a tile sees, on the host (paged_rules.h)."""
from tests.test_paged_cpu import _run


def test_a_stretch_that_is_passed_over_is_seen_by_no_row(tmp_path):
    """Any rows, windows and prefixes; and without a prefix no stretch is gone through that none sees, but for what lies behind the length."""
    out = _run(tmp_path, r"""
int main() {
    long long passed = 0;
    for (int len : {1, 40, 200}) for (int first : {0, 7, 39, 150, 199}) for (int rows : {1, 2, 33}) for (int window : {0, 1, 5, 32, 64, 1000}) for (int prefix : {0, 1, 20, 64, 180})
        for (int begin = 0; begin < len; begin++) for (int size : {1, 16, 64}) {
            const int last = first + rows - 1, end = begin + size;
            if (last >= len || prefix > len) continue;
            bool sees = false;
            for (int i = first; i <= last; i++) for (int j = begin; j < end && j < len; j++) sees |= paged_sees(i, j, len, window, prefix);
            const bool some = paged_some_see(first, last, begin, end, window, prefix);
            if (sees && !some) { std::printf("%d..%d see %d..%d\n", first, last, begin, end); return 0; }
            if (some && !sees && prefix == 0) { std::printf("%d..%d do not see %d..%d\n", first, last, begin, end); return 0; }
            passed += !some;
        }
    std::printf("%d\n", passed > 1000);
}
""")
    assert out == "1\n", out
