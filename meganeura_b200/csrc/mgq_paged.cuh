// What the kernels over a paged cache share: limits, element types, and how attention's work is cut.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "mgq_launch.cuh"
#include "mgq_tcgen05.cuh"

namespace mgq {

inline uint32_t page_shift(uint32_t page_size)
{
    uint32_t s = 0;
    while ((1u << s) < page_size) s++;
    return s;
}
inline uint32_t element_bytes(int dtype) { return dtype == MGQ_FMT_F32 ? 4 : 2; }

// Round to nearest, as a cast does: values beyond f16's range become infinite, NaN stays.
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---------------------------------------------------------------- how attention's work is cut
// A unit is a block of tokens of one sequence by the query heads of one key / value head (at most ROWS of these pairs) against
// all keys that any of its tokens sees, in blocks of KEYS.  The lengths are known on the device only, and they differ: the units' key
// blocks, in the order sequence, head, tokens, form one long list that is cut into equal pieces, one per CTA.  A unit that a piece's border cuts leaves
// unnormalised sums of both parts in the workspace, and merge_kernel joins them.
struct AttendArgs {
    const void *q, *k, *v;
    void *out;
    const uint32_t *starts, *lengths, *table;
    uint32_t sequences, rows, kv_heads, group, d, page_shift, pages, table_width, window, q_pitch, out_pitch;
    uint32_t rows_from, rows_to;         // sequences with this many pairs of token and head of a key / value head are this kernel's
    float scale_log2;                    // scale * log2(e): scores are exponents of 2
    struct PartHead *heads;              // [CTAs][2]
    float *parts;                        // [CTAs][2]: sums [ROWS][d], then maximum and weight of each row [ROWS][2]
};

enum PartState : uint32_t { kNoPart = 0, kOpens = 1, kGoesOn = 2, kCloses = 3 };
struct PartHead {
    uint32_t state, row0, tokens, head0, heads, pad[3];
};

struct Segment {
    uint32_t row0, tokens, head0, heads, kv;        // rows [row0, +tokens) by heads [head0, +heads)
    int pos0, len;                                  // position of the first token, tokens of the sequence that exist
    const uint32_t *table;
    uint32_t begin, end;                            // key blocks
    bool first, last;                               // of its unit
};

template <int ROWS, int KEYS, int EXTRA>
struct Walk {
    uint32_t slice, slices, per_tile;               // heads of a unit, units per key / value head, tokens of a unit
    uint32_t s, head, tile, off;                    // the next segment: sequence, head block, token block, key blocks behind
    uint32_t r0, n, tiles;
    int len;
    unsigned long long left;

    __device__ __forceinline__ void open(const AttendArgs &a, uint32_t seq)
    {
        s = seq;
        r0 = min(a.starts[s], a.rows);
        n = max(min(a.starts[s + 1], a.rows), r0) - r0;
        len = (int)min(a.lengths[s], a.table_width << a.page_shift);
        const unsigned long long pairs = (unsigned long long)n * a.group;
        tiles = pairs >= a.rows_from && pairs <= a.rows_to ? (n + per_tile - 1) / per_tile : 0;
    }
    __device__ __forceinline__ void keys(const AttendArgs &a, uint32_t t, uint32_t &lo, uint32_t &hi) const
    {
        const int first = len - (int)n + (int)(t * per_tile), last = min(len - 1, first + (int)per_tile - 1);
        hi = last < 0 ? 0u : (uint32_t)last / KEYS + 1;
        lo = a.window && first >= (int)a.window ? min((uint32_t)(first - (int)a.window + 1) / KEYS, hi) : 0u;
    }
    // Key blocks of a unit; one without any still costs a block, because its rows have to be written.
    __device__ __forceinline__ uint32_t cost(const AttendArgs &a, uint32_t t) const
    {
        uint32_t lo, hi;
        keys(a, t, lo, hi);
        return EXTRA + max(1u, hi - lo);
    }
    __device__ __forceinline__ unsigned long long head_cost(const AttendArgs &a) const
    {
        unsigned long long c = 0;
        for (uint32_t t = 0; t < tiles; t++) c += cost(a, t);
        return c;
    }

    // Every thread of the block: this CTA's piece.  `scratch`: 40 words of shared memory, free again when the call returns.
    __device__ __forceinline__ void begin(const AttendArgs &a, uint32_t cta, uint32_t ctas, unsigned long long *scratch)
    {
        slice = min(a.group, (uint32_t)ROWS);
        slices = (a.group + slice - 1) / slice;
        per_tile = ROWS / slice;
        s = head = tile = off = 0;
        const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, warps = blockDim.x >> 5, each = (a.sequences + blockDim.x - 1) / blockDim.x;
        const uint32_t s0 = min(t * each, a.sequences), s1 = min(s0 + each, a.sequences), heads = a.kv_heads * slices;
        unsigned long long mine = 0;
        for (uint32_t i = s0; i < s1; i++) {
            open(a, i);
            mine += head_cost(a) * heads;
        }
        unsigned long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long below = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += below;
        }
        if (lane == 31) scratch[warp] = upto;
        __syncthreads();
        unsigned long long base = upto - mine, total = 0;
        for (uint32_t w = 0; w < warps; w++) {
            if (w < warp) base += scratch[w];
            total += scratch[w];
        }
        const unsigned long long pieces = min((unsigned long long)ctas, max(total, 1ull));
        const unsigned long long w0 = cta < pieces ? total * cta / pieces : total, w1 = cta < pieces ? total * (cta + 1) / pieces : total;
        if (w0 >= base && w0 < base + mine) {            // one thread at most
            unsigned long long rest = w0 - base, c = 0;
            for (uint32_t i = s0; i < s1; i++) {
                open(a, i);
                c = head_cost(a);
                if (rest < c * heads) break;
                rest -= c * heads;
            }
            head = (uint32_t)(rest / c);
            rest %= c;
            tile = 0;
            while (rest >= cost(a, tile)) rest -= cost(a, tile++);
            scratch[32] = s;
            scratch[33] = head;
            scratch[34] = tile;
            scratch[35] = rest;
        }
        __syncthreads();
        left = w1 - w0;
        if (left) {
            const uint32_t at = (uint32_t)scratch[32];
            head = (uint32_t)scratch[33];
            tile = (uint32_t)scratch[34];
            off = (uint32_t)scratch[35];
            open(a, at);
        }
        __syncthreads();
    }

    __device__ __forceinline__ bool next(const AttendArgs &a, Segment &g)
    {
        while (left) {
            while (tile == tiles) {                      // behind the last unit of a head, or a sequence without any
                tile = 0;
                if (tiles && ++head < a.kv_heads * slices) break;
                head = 0;
                open(a, s + 1);                          // `left` says that there is one
            }
            uint32_t lo, hi;
            keys(a, tile, lo, hi);
            const uint32_t all = EXTRA + max(1u, hi - lo), take = (uint32_t)min((unsigned long long)(all - off), left);
            const uint32_t from = max(off, (uint32_t)EXTRA) - EXTRA, to = max(off + take, (uint32_t)EXTRA) - EXTRA;       // its own blocks
            g.row0 = r0 + tile * per_tile;
            g.tokens = min(per_tile, n - tile * per_tile);
            g.kv = head / slices;
            const uint32_t sub = head - g.kv * slices;
            g.head0 = g.kv * a.group + sub * slice;
            g.heads = min(slice, a.group - sub * slice);
            g.pos0 = len - (int)n + (int)(tile * per_tile);
            g.len = len;
            g.table = a.table + (size_t)s * a.table_width;
            g.begin = lo + from;
            g.end = min(lo + to, hi);                    // none where no row sees a key
            g.first = from == 0;
            off += take;
            left -= take;
            g.last = off == all;
            if (g.last) {
                off = 0;
                tile++;
            }
            if (to > from) return true;                  // else the piece ends in front of the unit's first block
        }
        return false;
    }
};

__device__ __forceinline__ uint32_t part_index(uint32_t cta, const Segment &g) { return 2 * cta + (g.first ? 1u : 0u); }
// One thread per CTA: no parts yet, and what a part holds.
__device__ __forceinline__ void clear_parts(const AttendArgs &a, uint32_t cta)
{
    a.heads[2 * cta].state = kNoPart;
    a.heads[2 * cta + 1].state = kNoPart;
}
__device__ __forceinline__ void name_part(const AttendArgs &a, uint32_t cta, const Segment &g)
{
    PartHead &h = a.heads[part_index(cta, g)];
    h.row0 = g.row0;
    h.tokens = g.tokens;
    h.head0 = g.head0;
    h.heads = g.heads;
    h.state = g.first ? kOpens : g.last ? kCloses : kGoesOn;
}

// Joins the parts of the unit that CTA blockIdx.x of an attention kernel began and did not end: with M the largest of the parts' maxima
// o = sum 2^(m - M) o_part / sum 2^(m - M) l_part.  The parts are those of the CTAs that follow, up to the one that ends the
// unit, added in this order.  Grid: (CTAs, anything): the rows are shared out over y, a warp takes a row.  Round trips to L2 bound it: a warp finds the
// unit's end with one, then takes eight parts with each, maxima, weights and sums together.
constexpr int kMergeThreads = 128, kMergeWarps = kMergeThreads / 32;
template <typename T, int ROWS, int COLS, int BATCH, bool WIDE>      // COLS: columns of a lane; four side by side (WIDE) or one in 32
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const AttendArgs a, uint32_t ctas)
{
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, c0 = blockIdx.x;
    auto column = [&](int i) { return WIDE ? 4 * lane + 128 * (i / 4) + i % 4 : lane + 32 * i; };
    pdl_launch_dependents();
    pdl_wait();
    const PartHead h = a.heads[2 * c0 + 1];
    if (h.state != kOpens) return;
    uint32_t parts = 1;
    for (;; parts += 32) {
        const uint32_t c = c0 + parts + lane, last = __ballot_sync(0xffffffffu, c + 1 >= ctas || a.heads[2 * c].state == kCloses);
        if (last) {
            parts += __ffs(last);
            break;
        }
    }
    const uint32_t d = a.d;
    const size_t size = (size_t)ROWS * (d + 2);
    for (uint32_t r = blockIdx.y * kMergeWarps + warp; r < h.tokens * h.heads; r += gridDim.y * kMergeWarps) {
        float top = -INFINITY, l = 0.f, o[COLS];
#pragma unroll
        for (int i = 0; i < COLS; i++) o[i] = 0.f;
        for (uint32_t p0 = 0; p0 < parts; p0 += BATCH) {
            float2 ml[BATCH];
            float v[BATCH][COLS];
#pragma unroll
            for (int b = 0; b < BATCH; b++) {
                const uint32_t p = p0 + b;
                const float *part = a.parts + (2 * (size_t)(c0 + p) + (p == 0 ? 1 : 0)) * size;
                const bool live = p < parts;
                ml[b] = live ? *reinterpret_cast<const float2 *>(part + ROWS * d + 2 * r) : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int i = 0; i < COLS; i += WIDE ? 4 : 1) {
                    const bool in = live && column(i) < d;
                    if constexpr (WIDE) {
                        const float4 q = in ? *reinterpret_cast<const float4 *>(part + r * d + column(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        v[b][i] = q.x; v[b][i + 1] = q.y; v[b][i + 2] = q.z; v[b][i + 3] = q.w;
                    } else {
                        v[b][i] = in ? part[r * d + column(i)] : 0.f;
                    }
                }
            }
            const float before = top;
#pragma unroll
            for (int b = 0; b < BATCH; b++) top = fmaxf(top, ml[b].x);
            const float keep = before > -INFINITY ? exp2f(before - top) : 1.f;
            l *= keep;
#pragma unroll
            for (int i = 0; i < COLS; i++) o[i] *= keep;
#pragma unroll
            for (int b = 0; b < BATCH; b++) {
                const float w = ml[b].y != 0.f ? exp2f(ml[b].x - top) : 0.f;         // a NaN is a weight; a part without weight may hold anything
                l += w * ml[b].y;
#pragma unroll
                for (int i = 0; i < COLS; i++) o[i] += w != 0.f ? w * v[b][i] : 0.f;
            }
        }
        const float scale = l == 0.f ? 0.f : 1.f / l;
        const uint32_t token = r / h.heads, head = r - token * h.heads;
        T *out = static_cast<T *>(a.out) + (size_t)(h.row0 + token) * a.out_pitch + (size_t)(h.head0 + head) * d;
#pragma unroll
        for (int i = 0; i < COLS; i++)
            if (column(i) < d) out[column(i)] = rounded<T>(o[i] * scale);
    }
}
// pairs: a bound of the rows of a unit that has parts.  Units of few rows may have many parts: eight at a time; of 256 rows a handful, and registers for
// more warps count.
template <typename T, int ROWS>
int launch_merge(const AttendArgs &a, uint32_t ctas, uint32_t pairs, cudaStream_t stream)
{
    constexpr int kBatch = ROWS > 64 ? 2 : 8;
    const dim3 grid(ctas, (min(pairs, (uint32_t)ROWS) + kMergeWarps - 1) / kMergeWarps);
    auto *kernel = a.d % 4 == 0 ? (a.d <= 128 ? merge_kernel<T, ROWS, 4, kBatch, true> : merge_kernel<T, ROWS, 8, kBatch / 2, true>)
                                : (a.d <= 128 ? merge_kernel<T, ROWS, 4, kBatch, false> : merge_kernel<T, ROWS, 8, kBatch / 2, false>);
    return launch(kernel, grid, dim3(kMergeThreads), 0, stream, a, ctas);
}

// 16-bit types with heads of a multiple of 8 elements on 16-byte boundaries: few new tokens (mgq_paged_decode.cu).
bool decode_takes(const AttendArgs &a, int dtype);
uint32_t decode_ctas(uint32_t head_dim);
constexpr int kDecodeRows = 16, kDecodePairs = 32;         // of a unit; of a sequence that is not yet many tokens'
int launch_decode(const AttendArgs &a, int dtype, uint32_t pairs, cudaStream_t stream);      // pairs: a bound of a sequence's tokens * heads per key / value head

// The same types with heads of up to 128, everything on 16-byte boundaries: many new tokens (mgq_paged_prefill.cu).
bool prefill_takes(const AttendArgs &a, int dtype);
constexpr uint32_t kPrefillCtas = 148, kPrefillRows = 256;
int launch_prefill(const AttendArgs &a, int dtype, cudaStream_t stream);

// f32 with heads of up to 128, a multiple of 4, on 16-byte boundaries: up to 24 pairs of a sequence per key / value head (mgq_paged_few.cu); from 25 on the
// tiles of 64 rows.  16 sequences of four heads of 128: 16 pairs 199 and 310 us, 24 pairs 290 and 310, 28 pairs 364 and 310; of one head of 80: 16
// pairs 292 and 378, 24 pairs 431 and 391.
bool few_takes(const AttendArgs &a, int dtype);
constexpr uint32_t kFewPairs = 24;
uint32_t few_ctas(uint32_t rows);                          // rows of a unit: 1, 4 or 8
size_t few_part_floats(uint32_t rows, uint32_t d);
int launch_few(const AttendArgs &a, uint32_t rows, cudaStream_t stream);

// {head_dim, kv_heads, pages * page_size} of a cache, for boxes of 64 elements by `tokens` tokens of one head in the 128-byte swizzle.  What
// lies outside the cache reads as zero.
struct CacheMaps {
    CUtensorMap k, v;
};
int encode_caches(CacheMaps &maps, int dtype, const AttendArgs &a, uint32_t tokens);         // mgq_paged_decode.cu

}  // namespace mgq
