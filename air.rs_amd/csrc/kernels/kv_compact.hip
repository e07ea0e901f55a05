// Compaction of cached sequences inside their own pages: token keep[i] of a
// sequence moves to position i, for ascending kept positions, K, V and scales bit
// for bit (the device half of dropping tokens from the middle of a sequence; the
// manager's truncate then frees the blocks past the kept ones).
//
// keep[i] >= i, so walking the kept tokens in ascending order never reads a row
// that was already written.  One workgroup is a chain: it walks one column part of
// one (sequence, head, K or V) stripe, kStep rows at a time, with the next step's
// loads issued before the present step's stores.  A step's sources lie at or behind
// its first destination, so its stores wait until every wave holds its rows (one
// barrier a step); the next step's sources lie behind all of them.  Nothing orders
// two chains: they touch different bytes.
//
// Bound by memory: each moved row is read once and written once.  64 sequences of
// 512 to 4096 tokens, half kept: 666 MB in 141 us, 4.7 TB/s; 4 of 32K to 64K moved
// behind their first tokens, 128 chains: 1.37 GB in 326 us, 4.2 TB/s, what half of
// the CUs carry (a chain's steps are in order; more chains would split lines).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../pool.hpp"

namespace airkv {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWindow = 1024;              // kept tokens whose rows are resolved at a time
constexpr int kUnroll = 8;                 // pieces of a step per thread (4: 143 and 332 us)

// Threads of a chain: the wide ones where sequences fill half a step of theirs (64 that
// keep 256 to 2048 of 8 heads' bf16 rows: 141 against 151 us), the narrow ones where
// they do not (100 that keep 10 to 100: 20 against 40 us).
constexpr int kWide = 1024, kNarrow = 256;

struct CompactArgs {
    const int32_t *tables, *lens, *keep, *cu;
    int32_t max_blocks, total_keep, heads, bs;
    int64_t num_blocks;
    uint8_t *pages[2], *scales[2];
    int32_t row_bytes, scale_row_bytes;    // one token's row of one head
    int32_t parts, part_pieces;            // a page row as column parts of 16-byte pieces
    unsigned long long *errors;
};

// One chain over n kept tokens.  T: the piece a thread moves.
template <class T, int THREADS>
__device__ __forceinline__ void walk(const CompactArgs &a, uint8_t *base, int64_t row_bytes, int64_t head_row, int piece0,
                                     int pieces, int b, int c0, int n, int64_t len, bool counts, int64_t (*s_src)[kWindow],
                                     int64_t (*s_dst)[kWindow]) {
    const int tid = threadIdx.x;
    const int per = THREADS / pieces;                  // rows of a pass
    const int my = tid / pieces, piece = piece0 + tid % pieces;
    const int step = per * kUnroll;
    const int32_t *table = a.tables + (int64_t)b * a.max_blocks;
    for (int w0 = 0; w0 < n; w0 += kWindow) {
        const int wn = n - w0 < kWindow ? n - w0 : kWindow;
        // rows of the window's tokens, without the head's offset; -1: nothing moves
        for (int i = tid; i < wn; i += THREADS) {
            const int to = w0 + i;
            const int64_t from = a.keep[c0 + to];
            const int64_t before = to > 0 ? a.keep[c0 + to - 1] : -1;
            bool ok = from > before && from >= to && from < len;
            int64_t src = -1, dst = -1;
            if (ok && from != to) {
                const int32_t sb = table[from / a.bs], db = table[to / a.bs];
                ok = sb >= 0 && sb < a.num_blocks && db >= 0 && db < a.num_blocks;
                if (ok) {
                    src = (int64_t)sb * a.heads * a.bs + from % a.bs;
                    dst = (int64_t)db * a.heads * a.bs + to % a.bs;
                }
            }
            if (!ok && counts) atomicAdd(a.errors, 1ull);
            (*s_src)[i] = src;
            (*s_dst)[i] = dst;
        }
        __syncthreads();
        auto load = [&](int at, T (&x)[kUnroll]) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = at + u * per + my;
                if (my < per && i < wn && (*s_src)[i] >= 0)
                    x[u] = __builtin_nontemporal_load(
                        reinterpret_cast<const T *>(base + ((*s_src)[i] + head_row) * row_bytes) + piece);
            }
        };
        auto store = [&](int at, const T (&x)[kUnroll]) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = at + u * per + my;
                if (my < per && i < wn && (*s_src)[i] >= 0)
                    __builtin_nontemporal_store(x[u], reinterpret_cast<T *>(base + ((*s_dst)[i] + head_row) * row_bytes) + piece);
            }
        };
        // the rows are in registers (not on their way) when the barrier is passed
        auto hold = [&](T (&x)[kUnroll]) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) asm volatile("" : "+v"(x[u])::"memory");
            __syncthreads();
        };
        T x[kUnroll] = {}, y[kUnroll] = {};
        load(0, x);
        for (int at = 0; at < wn; at += 2 * step) {
            load(at + step, y);
            hold(x);
            store(at, x);
            if (at + step >= wn) break;
            load(at + 2 * step, x);
            hold(y);
            store(at + step, y);
        }
        __syncthreads();                               // the window's rows are overwritten next
    }
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_compact_kernel(CompactArgs a) {
    __shared__ int64_t s_src[kWindow], s_dst[kWindow];
    const int b = blockIdx.x;
    const int64_t max_len = (int64_t)a.max_blocks * a.bs;
    const int32_t n_tok = a.lens[b];
    const int64_t len = n_tok < 0 ? 0 : n_tok > max_len ? max_len : n_tok;
    const int c0 = a.cu[b], c1 = a.cu[b + 1];
    const bool first = blockIdx.y == 0;
    if (first && threadIdx.x == 0 && n_tok != len) atomicAdd(a.errors, 1ull);
    if (c0 < 0 || c1 > a.total_keep || c1 < c0) {
        if (first && threadIdx.x == 0) atomicAdd(a.errors, 1ull);
        return;
    }
    if (c1 == c0) return;
    int y = blockIdx.y;
    const int chains = 2 * a.heads * a.parts;
    if (y < chains) {
        const int part = y % a.parts, th = y / a.parts, h = th % a.heads, t = th / a.heads;
        const int all = a.row_bytes / 16, p0 = part * a.part_pieces;
        const int pieces = all - p0 < a.part_pieces ? all - p0 : a.part_pieces;
        walk<u32x4, THREADS>(a, a.pages[t], a.row_bytes, (int64_t)h * a.bs, p0, pieces, b, c0, c1 - c0, len, first, &s_src, &s_dst);
    } else {
        y -= chains;
        const int h = y % a.heads, t = y / a.heads;
        walk<uint32_t, THREADS>(a, a.scales[t], a.scale_row_bytes, (int64_t)h * a.bs, 0, a.scale_row_bytes / 4, b, c0, c1 - c0, len, false,
                                &s_src, &s_dst);
    }
}

}  // namespace

hipError_t launch_compact(const air_kv_pool &p, hipStream_t s, const int32_t *tables, const int32_t *lens, int32_t batch,
                          int32_t max_blocks, const int32_t *keep, const int32_t *cu, int32_t total_keep) {
    CompactArgs a;
    a.tables = tables; a.lens = lens; a.keep = keep; a.cu = cu;
    a.max_blocks = max_blocks; a.total_keep = total_keep;
    a.heads = p.desc.n_kv_heads; a.bs = p.desc.block_size;
    a.num_blocks = p.desc.num_blocks;
    a.pages[0] = (uint8_t *)p.k_pages; a.pages[1] = (uint8_t *)p.v_pages;
    a.scales[0] = (uint8_t *)p.k_scales; a.scales[1] = (uint8_t *)p.v_scales;
    const bool quant = dtype_quantized(p.desc.dtype);
    a.row_bytes = (int32_t)(p.desc.head_dim * p.elem_bytes);
    a.scale_row_bytes = quant ? p.desc.head_dim / p.desc.scale_group * 4 : 0;
    a.errors = p.errors;
    // few chains: rows of two lines or more are walked in column parts of a line
    // (half lines: 553 us where lines take 331); loads and stores go past the L2 (345 us
    // with stores, 353 with loads that stay in it)
    const int64_t stripes = (int64_t)batch * 2 * a.heads;
    a.part_pieces = a.row_bytes / 16;
    a.parts = 1;
    if (stripes < 2 * p.cus && a.row_bytes >= 256) {
        a.part_pieces = 8;
        a.parts = (a.row_bytes / 16 + 7) / 8;
    }
    const dim3 grid((unsigned)batch, (unsigned)(2 * a.heads * a.parts + (quant ? 2 * a.heads : 0)));
    const int64_t half_step = (int64_t)kUnroll * (kWide / 2) / a.part_pieces;      // rows
    if (total_keep >= half_step * batch || stripes * a.parts < 4 * p.cus) hipLaunchKernelGGL((kv_compact_kernel<kWide>), grid, dim3(kWide), 0, s, a);
    else hipLaunchKernelGGL((kv_compact_kernel<kNarrow>), grid, dim3(kNarrow), 0, s, a);
    return hipGetLastError();
}

}  // namespace airkv
