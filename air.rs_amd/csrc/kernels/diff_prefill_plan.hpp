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

// The sum of floor((a i + b) / m) over i = 0 .. n - 1, for small a.  What a has of whole m's
// leaves the floor (nothing else is left of it where the pairs divide rows / 32).  The rest, by
// Hermite's identity floor(a x) = sum of floor(x + s / a) over s = 0 .. a - 1 with
// x = (a i + b) / (a m):
//   floor((a i + b) / m) = sum over s of floor((i + c_s) / m),  c_s = floor((b + s m) / a),
// and over i each s runs through the numerators from c_s to c_s + n.  The sum of
// floor(y / m) over y < N, w = floor(N / m), is w N - m w (w + 1) / 2; the c_s lie within m
// of the first, so that its w serves all of them, plus what N has past m (w + 1).
AIRKV_DP_HD inline uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
    if (n == 0) return 0;
    auto half = [](uint64_t w) { return w & 1 ? (w + 1) / 2 * w : w / 2 * (w + 1); };      // w (w + 1) / 2
    uint64_t sum = 0;
    if (a >= m) {
        sum = a / m * half(n - 1);
        a %= m;
    }
    if (a == 0) return sum + n * (b / m);
    const uint64_t step = m / a, step_rest = m - step * a;
    uint64_t c = b / a, c_rest = b - c * a;
    const uint64_t w0 = c / m, w1 = (c + n) / m, top0 = w0 * m + m, top1 = w1 * m + m;
    uint64_t all = 0, past = 0;                        // of the c_s; past the tops
    for (uint64_t s = 0; s < a; ++s) {
        all += c;
        past += (c + n > top1 ? c + n - top1 : 0) - (c > top0 ? c - top0 : 0);
        c += step;
        c_rest += step_rest;
        if (c_rest >= a) {
            c_rest -= a;
            ++c;
        }
    }
    return sum + w1 * (all + a * n) - w0 * all - a * m * (half(w1) - half(w0)) + past;
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
    // (rows and kDiffKeys are multiples of 32: the tiles of a full block are
    // floor((rows k + c) / (kDiffKeys g)), and 32 goes out of both)
    AIRKV_DP_HD int64_t before(int64_t k) const {
        const uint64_t c = (uint64_t)(prefix + kDiffKeys) * g + rows - 1;
        return extra * k + (int64_t)floor_sum((uint64_t)k, (uint64_t)(kDiffKeys / 32) * g, (uint64_t)rows / 32, c / 32);
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
