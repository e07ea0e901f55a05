// Checks diff_prefill_plan.hpp: the closed sums against counting, and that the
// slices of a launch hold every (block, tile) once, with piece slots of their own
// that the joining finds.  Prints "<cases> cases, <n> wrong".
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "kernels/diff_prefill_plan.hpp"

using namespace airkv;

static long cases = 0, wrong = 0;
static void check(bool ok, const char *what, long long a = 0, long long b = 0, long long c = 0) {
    if (!ok && wrong++ < 20) std::printf("wrong: %s (%lld, %lld, %lld)\n", what, a, b, c);
}

static void sums(DiffBlocks s) {
    ++cases;
    const int64_t n = s.blocks();
    int64_t at = 0;
    for (int64_t k = 0; k < n; ++k) {
        check(s.before(k) == at, "units before a block", s.q, s.prefix, k);
        // the keys its last row sees, counted row by row
        const int64_t last = std::min((k + 1) * s.rows, s.q * s.g) - 1;
        check(s.keys(k) == s.prefix + last / s.g + 1, "keys of a block", s.q, s.prefix, k);
        at += s.extra + (s.keys(k) + kDiffKeys - 1) / kDiffKeys;
    }
    check(s.units() == at, "units of a sequence", s.q, s.prefix, s.g);
}

static void walk(const std::vector<DiffBlocks> &seqs, int64_t slices, int64_t least) {
    ++cases;
    std::vector<int64_t> pre{0};
    for (const auto &s : seqs) pre.push_back(pre.back() + s.units());
    const int64_t units = pre.back(), chunk = diff_prefill_chunk(units, slices, least);
    check(chunk * slices >= units, "the slices hold every unit", units, slices, chunk);
    std::set<int64_t> used;                            // piece slots
    std::map<std::pair<int, int64_t>, int64_t> done;   // tiles of each block
    std::map<std::pair<int, int64_t>, std::vector<int64_t>> pieces, joined;
    for (int64_t w = 0; w < slices; ++w) {
        int64_t u = w * chunk;
        const int64_t end = std::min(u + chunk, units);
        while (u < end) {
            int b = 0;
            while (pre[b + 1] <= u) ++b;
            const DiffBlocks &s = seqs[b];
            int64_t k = 0;
            while (k + 1 < s.blocks() && s.before(k + 1) <= u - pre[b]) ++k;
            const int64_t from = u - pre[b] - s.before(k), nt = s.tiles(k), mine = std::min(end - u, s.extra + nt - from);
            check(from >= 0 && mine > 0, "a block's units", b, k, from);
            const int64_t t0 = diff_tile_of(from, s.extra), t1 = diff_tile_of(from + mine, s.extra);
            check(t0 <= t1 && t1 <= nt && (done[{b, k}]) == t0, "a block's tiles in order", b, k, t0);
            done[{b, k}] = t1;
            u += mine;
            if (t0 == t1) continue;
            if (!(t0 == 0 && t1 == nt)) {
                const int64_t slot = 2 * w + (t0 == 0 ? 1 : 0);
                check(used.insert(slot).second && slot < 2 * slices, "a piece slot of its own", slot, w, t0);
                pieces[{b, k}].push_back(slot);
                if (t0 == 0) {
                    const int64_t n = (u - t1 + nt - 1) / chunk - w + 1;
                    for (int64_t i = 0; i < n; ++i) joined[{b, k}].push_back(2 * (w + i) + (i == 0 ? 1 : 0));
                }
            }
        }
    }
    for (size_t b = 0; b < seqs.size(); ++b)
        for (int64_t k = 0; k < seqs[b].blocks(); ++k)
            check((done[{(int)b, k}]) == seqs[b].tiles(k), "every block is finished", (long long)b, k);
    check(pieces == joined, "the joining finds every piece, in order", units, slices, chunk);
}

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return (int)std::uniform_int_distribution<int>(lo, hi)(rng); };
    for (int i = 0; i < 3000; ++i) {
        const uint64_t n = pick(0, 300), m = pick(1, 500), a = pick(0, 900), b = pick(0, 900);
        uint64_t want = 0;
        for (uint64_t j = 0; j < n; ++j) want += (a * j + b) / m;
        check(floor_sum(n, m, a, b) == want, "floor_sum", n, m, a);
        ++cases;
    }
    for (int i = 0; i < 1500; ++i)
        sums({pick(0, 900), i % 3 ? pick(0, 5000) : 0, pick(1, i % 5 ? 16 : 300), i % 2 ? 64 : 128, i % 8});
    sums({131072, 1 << 20, 8, 64, 7});                   // sums of long sequences stay exact
    for (int i = 0; i < 600; ++i) {
        std::vector<DiffBlocks> seqs;
        const int g = pick(1, 20), rows = i % 2 ? 64 : 128, extra = pick(0, 9);
        for (int n = pick(1, 12); n > 0; --n) seqs.push_back({pick(0, 3) ? pick(1, 200) : 0, pick(0, 2) ? pick(0, 2000) : 0, g, rows, extra});
        for (auto &s : seqs)
            if (!s.q) s.prefix = 0;
        walk(seqs, pick(1, 140), pick(1, 32));
    }
    std::printf("%ld cases, %ld wrong\n", cases, wrong);
    return wrong != 0;
}
