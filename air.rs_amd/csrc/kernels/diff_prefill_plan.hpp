// Arithmetic of the differential prefill's work division, in host and device
// code, so that it can be checked on the CPU (tests/diff_prefill_plan_check.cpp).
//
// A sequence's rows are its (new token, query pair of the K/V pair) combinations,
// token after token: row f is token f / g, pair f % g.  A block is `rows`
// consecutive ones; it needs the keys its last token sees, in tiles of kDiffKeys.
// A block counts as `extra` units (what beginning and ending it costs, in tiles'
// time) and one for each of its tiles; a K/V pair's units, sequence after
// sequence, block after block, are cut into equal slices, one workgroup each.  The
// slice that holds a block's first tile begins it.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define AIRKV_DP_HD __host__ __device__
#else
#define AIRKV_DP_HD
#endif

namespace airkv {

constexpr int kDiffKeys = 32;

// sum of floor((a * i + b) / m) over i = 0 .. n - 1, by the Euclidean descent on
// (m, a): lattice points under a line, exchanging the axes at each step.
AIRKV_DP_HD inline uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
    uint64_t sum = 0;
    while (n) {
        if (a >= m) {
            sum += n * (n - 1) / 2 * (a / m);
            a %= m;
        }
        if (b >= m) {
            sum += n * (b / m);
            b %= m;
        }
        const uint64_t top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top % m;
        const uint64_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// One sequence: q new tokens behind `prefix` cached ones, g query pairs.
struct DiffBlocks {
    int64_t q, prefix;
    int g, rows, extra;
    AIRKV_DP_HD int64_t blocks() const { return (q * g + rows - 1) / rows; }
    // keys and key tiles of block k: up to the last token it holds
    AIRKV_DP_HD int64_t keys(int64_t k) const {
        const int64_t last = (k + 1) * rows < q * g ? ((k + 1) * rows - 1) / g : q - 1;
        return prefix + last + 1;
    }
    AIRKV_DP_HD int64_t tiles(int64_t k) const { return (keys(k) + kDiffKeys - 1) / kDiffKeys; }
    // units of block k, and of the blocks before it (k < blocks(): all of them full)
    AIRKV_DP_HD int64_t cost(int64_t k) const { return extra + tiles(k); }
    AIRKV_DP_HD int64_t before(int64_t k) const {
        return extra * k + (int64_t)floor_sum((uint64_t)k, (uint64_t)kDiffKeys * g, (uint64_t)rows,
                                  (uint64_t)(prefix + kDiffKeys) * g + rows - 1);
    }
    AIRKV_DP_HD int64_t units() const {
        const int64_t n = blocks();
        return n ? before(n - 1) + cost(n - 1) : 0;
    }
};

// The tiles [t0, t1) of a block that its units [from, to) hold.
AIRKV_DP_HD inline int64_t diff_tile_of(int64_t unit, int extra) { return unit > extra ? unit - extra : 0; }

// Units per slice: an equal share, but at least `least`, so that small launches
// are not cut into pieces whose joining costs more than their work.
AIRKV_DP_HD inline int64_t diff_prefill_chunk(int64_t units, int64_t slices, int64_t least) {
    const int64_t c = (units + slices - 1) / slices;
    return c > least ? c : least;
}

}  // namespace airkv
