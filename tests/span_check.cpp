// Spans of rows (air.rs_amd/csrc/host/span.hpp, as the entry points include it): which meet.
#include <cstdio>

#include "host/span.hpp"

int main() {
    using airkv::Span;
    auto at = [](uintptr_t x) { return (const void *)x; };
    int bad = 0;
    auto check = [&](bool got, bool want, const char *what) {
        if (got != want) std::printf("%s: %d\n", what, (int)got), ++bad;
    };
    const Span a(at(4096), 3, 64, 32, 4);              // 4096 .. 4096 + (2 * 64 + 32) * 4 = 4736
    check(a.end == 4736, true, "end");
    check(a.meets(Span(at(4736), 1, 32, 32, 4)), false, "behind");
    check(a.meets(Span(at(4732), 1, 32, 32, 4)), true, "its last element");
    check(a.meets(Span(at(4096 - 128), 1, 32, 32, 4)), false, "before");
    check(a.meets(Span(at(4096 - 124), 1, 32, 32, 4)), true, "its first element");
    check(Span(at(4096 - 128), 1, 32, 32, 4).meets(a), false, "before, the other way");
    check(a.meets(a), true, "itself");
    // the largest arguments that are taken: the sizes pass 63 and 64 bits
    const int64_t n = INT32_MAX, stride = (int64_t)1 << 31;
    const Span big(at(1 << 20), n, stride, stride, 4);
    check(big.end > big.at, true, "2^64 bytes");
    check(big.meets(Span(at((uintptr_t)1 << 40), 1, 32, 32, 4)), true, "inside 2^64 bytes");
    check(Span(at((uintptr_t)1 << 40), 1, 32, 32, 4).meets(big), true, "inside, the other way");
    check(big.meets(Span(at(4096), 1, 32, 32, 4)), false, "before 2^64 bytes");
    std::printf("%d differ\n", bad);
    return bad != 0;
}
