// What the kernels over a paged cache share: limits, element types, and how attention's work is cut.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "mgq_launch.cuh"

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
    float *parts;                        // [CTAs][2][ROWS][d + 2]: sums, maximum, weight
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

template <int ROWS, int KEYS>
struct Walk {
    const AttendArgs &a;
    uint32_t slice, slices, per_tile;               // heads of a unit, units per key / value head, tokens of a unit
    uint32_t s = 0, head = 0, tile = 0, off = 0;    // the next segment: sequence, head block, token block, key blocks behind
    uint32_t r0 = 0, n = 0, tiles = 0;
    int len = 0;
    unsigned long long left = 0;

    __device__ __forceinline__ explicit Walk(const AttendArgs &args) : a(args)
    {
        slice = min(a.group, (uint32_t)ROWS);
        slices = (a.group + slice - 1) / slice;
        per_tile = ROWS / slice;
    }
    __device__ __forceinline__ void open(uint32_t seq)
    {
        s = seq;
        r0 = min(a.starts[s], a.rows);
        n = max(min(a.starts[s + 1], a.rows), r0) - r0;
        len = (int)min(a.lengths[s], a.table_width << a.page_shift);
        const unsigned long long pairs = (unsigned long long)n * a.group;
        tiles = pairs >= a.rows_from && pairs <= a.rows_to ? (n + per_tile - 1) / per_tile : 0;
    }
    __device__ __forceinline__ void keys(uint32_t t, uint32_t &lo, uint32_t &hi) const
    {
        const int first = len - (int)n + (int)(t * per_tile), last = min(len - 1, first + (int)per_tile - 1);
        hi = last < 0 ? 0u : (uint32_t)last / KEYS + 1;
        lo = a.window && first >= (int)a.window ? min((uint32_t)(first - (int)a.window + 1) / KEYS, hi) : 0u;
    }
    // Key blocks of a unit; one without any still costs a block, because its rows have to be written.
    __device__ __forceinline__ uint32_t cost(uint32_t t) const
    {
        uint32_t lo, hi;
        keys(t, lo, hi);
        return max(1u, hi - lo);
    }
    __device__ __forceinline__ unsigned long long head_cost() const
    {
        unsigned long long c = 0;
        for (uint32_t t = 0; t < tiles; t++) c += cost(t);
        return c;
    }

    // Every thread of the block: this CTA's piece.  `scratch`: 40 words of shared memory, free again when the call returns.  Pieces have
    // at least `least` key blocks where there are that many.
    __device__ __forceinline__ void begin(uint32_t cta, uint32_t ctas, uint32_t least, unsigned long long *scratch)
    {
        const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, warps = blockDim.x >> 5, each = (a.sequences + blockDim.x - 1) / blockDim.x;
        const uint32_t s0 = min(t * each, a.sequences), s1 = min(s0 + each, a.sequences), heads = a.kv_heads * slices;
        unsigned long long mine = 0;
        for (uint32_t i = s0; i < s1; i++) {
            open(i);
            mine += head_cost() * heads;
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
        const unsigned long long pieces = min((unsigned long long)ctas, max(total / least, 1ull));
        const unsigned long long w0 = cta < pieces ? total * cta / pieces : total, w1 = cta < pieces ? total * (cta + 1) / pieces : total;
        if (w0 >= base && w0 < base + mine) {            // one thread at most
            unsigned long long rest = w0 - base, c = 0;
            for (uint32_t i = s0; i < s1; i++) {
                open(i);
                c = head_cost();
                if (rest < c * heads) break;
                rest -= c * heads;
            }
            head = (uint32_t)(rest / c);
            rest %= c;
            tile = 0;
            while (rest >= cost(tile)) rest -= cost(tile++);
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
            open(at);
        }
        __syncthreads();
    }

    __device__ __forceinline__ bool next(Segment &g)
    {
        if (!left) return false;
        while (tile == tiles) {                          // behind the last unit of a head, or a sequence without any
            tile = 0;
            if (tiles && ++head < a.kv_heads * slices) break;
            head = 0;
            open(s + 1);                                 // `left` says that there is one
        }
        uint32_t lo, hi;
        keys(tile, lo, hi);
        const uint32_t all = max(1u, hi - lo), take = (uint32_t)min((unsigned long long)(all - off), left);
        g.row0 = r0 + tile * per_tile;
        g.tokens = min(per_tile, n - tile * per_tile);
        g.kv = head / slices;
        const uint32_t sub = head - g.kv * slices;
        g.head0 = g.kv * a.group + sub * slice;
        g.heads = min(slice, a.group - sub * slice);
        g.pos0 = len - (int)n + (int)(tile * per_tile);
        g.len = len;
        g.table = a.table + (size_t)s * a.table_width;
        g.begin = lo + off;
        g.end = min(lo + off + take, hi);                // none where no row sees a key
        g.first = off == 0;
        off += take;
        left -= take;
        g.last = off == all;
        if (g.last) {
            off = 0;
            tile++;
        }
        return true;
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

}  // namespace mgq
