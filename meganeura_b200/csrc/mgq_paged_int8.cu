// New keys and values into a paged cache of 8-bit codes with a scale for each block of tokens and head.
#include "mgq_paged_int8.cuh"

namespace mgq {
namespace {

// A block's scale is that of its largest value, so its rows belong together.  Those of a step that fall into one block, a run, mostly stand one behind another.  A CTA
// takes the runs that begin in a window of rows, for a number of jobs (a head of the keys or of the values each): a run of more than kShort rows by all its threads, shorter ones
// by a warp each.  Where other rows of the step fall into a run's block as well, which a look at all slots shows, the CTA of the first of them gathers them all, so that no block
// is written from two places.  new = max(old, that of the largest), where old is 0 if the block's first slot is among the rows: the block starts anew.  Codes that the block holds
// already become rint(code * old / new) where the scale grew.  Rotated values stay with their threads between the pass for the largest and the one for the codes, kHold
// steps of 16 values a thread (32 rows of 128 for a CTA; 12 to 44 bytes a thread in local memory, at 64 registers); what lies behind is computed again.
// Loads that wait for one another bound it (slots, then scale and rows, then what is held), so CTAs per SM count more than registers: 4096 rows of the Qwen3-8B shape
// took 52, 45, 39 us with two, three, four; and windows are as wide as leaves eight CTAs per SM, of one job.  As every CTA looks at all slots, it takes as many jobs as leave six of
// them: with one 41 us for 4096 rows and 189 for 16384, so 35 and 125 (before the look, with one, 36 and 138; 64 single tokens 10.2 then, now 11.2; 131072 rows of two
// heads of 64 160 and 266).  Rows in mixed order are gathered value by value: 4096 take 0.6 ms.
constexpr int kThreads = 256, kWarps = kThreads / 32, kHold = 1, kCtas = 4;
constexpr uint32_t kMostBlock = 1024, kMostWindow = 32, kShort = 4;

struct Append8Args {
    const void *q, *k, *v;
    const uint32_t *positions, *slots;
    void *q_out;
    int8_t *k_cache, *v_cache;
    float *k_scales, *v_scales;
    uint32_t rows, q_heads, kv_heads, d, q_pitch, k_pitch, v_pitch, slots_end, block_shift, window, jobs, cache_ctas;      // jobs of a CTA: heads of keys or values
    double log2_theta;
    bool rotate;
};

// (cos, sin) of position * theta^(-2i/d), the product and its reduction to one turn in 64 bits.
__device__ __forceinline__ float2 turn_of(uint32_t position, double frequency)
{
    const double angle = (double)position * frequency, turn = 6.283185307179586476925286766559;
    float2 w;
    sincosf((float)fma(-rint(angle * (1.0 / turn)), turn, angle), &w.y, &w.x);
    return w;
}
__device__ __forceinline__ void rotate_pair(float &lo, float &hi, float2 w)
{
    const float x = lo * w.x - hi * w.y;
    hi = lo * w.y + hi * w.x;
    lo = x;
}
template <typename T>
__device__ __forceinline__ void read8(const T *p, float (&f)[8], bool wide)
{
    T v[8];
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = to_f32(v[i]);
}

// Rows [r0, r0 + n) into their block, by THREADS threads (a warp or the CTA).
template <typename S, int THREADS, typename Slot>
__device__ __forceinline__ void store_run(const Append8Args &a, const double *frequency, uint32_t *written, uint32_t *tops, uint32_t r0, uint32_t n, uint32_t head, bool values,
                                          bool wide, Slot slot_of)
{
    auto meet = [] {
        if constexpr (THREADS == 32) __syncwarp();
        else                         __syncthreads();
    };
    const uint32_t t = threadIdx.x % THREADS, half = a.d / 2, steps = half / 8, block = 1u << a.block_shift, pitch = values ? a.v_pitch : a.k_pitch;
    const bool rotate = a.rotate && !values;
    const S *src = static_cast<const S *>(values ? a.v : a.k) + (size_t)head * a.d;
    int8_t *cache = (values ? a.v_cache : a.k_cache) + (size_t)head * a.d;
    const size_t row_bytes = (size_t)a.kv_heads * a.d;
    const uint32_t id = slot_of(r0) >> a.block_shift;
    float *scale_at = (values ? a.v_scales : a.k_scales) + (size_t)id * a.kv_heads + head;
    const float was = *scale_at;
    const uint32_t items = n * steps;                    // eight pairs of a row each
    auto fetch = [&](uint32_t i, float (&lo)[8], float (&hi)[8]) {
        const uint32_t r = i / steps, p = (i - r * steps) * 8;
        const S *row = src + (size_t)(r0 + r) * pitch + p;
        read8(row, lo, wide);
        read8(row + half, hi, wide);
    };
    auto turn = [&](uint32_t i, float (&lo)[8], float (&hi)[8]) {
        if (!rotate) return;
        const uint32_t r = i / steps, p = (i - r * steps) * 8, position = a.positions[r0 + r];
#pragma unroll
        for (int e = 0; e < 8; e++) rotate_pair(lo[e], hi[e], turn_of(position, frequency[p + e]));
    };
    // the rows' loads are on their way while their slots are noted
    float lo[kHold][8], hi[kHold][8];
#pragma unroll
    for (int b = 0; b < kHold; b++)
        if (b * THREADS + t < items) fetch(b * THREADS + t, lo[b], hi[b]);
    for (uint32_t w = t; w < (block + 31) / 32; w += THREADS) written[w] = 0;
    meet();
    for (uint32_t r = t; r < n; r += THREADS) {
        const uint32_t at = slot_of(r0 + r) & (block - 1);
        atomicOr(&written[at / 32], 1u << (at & 31u));
    }
    uint32_t top = 0;
    auto larger = [&](const float (&f)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
    };
#pragma unroll
    for (int b = 0; b < kHold; b++)
        if (b * THREADS + t < items) {
            turn(b * THREADS + t, lo[b], hi[b]);
            larger(lo[b]);
            larger(hi[b]);
        }
    for (uint32_t i = kHold * THREADS + t; i < items; i += THREADS) {
        float x[8], y[8];
        fetch(i, x, y);
        turn(i, x, y);
        larger(x);
        larger(y);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (THREADS > 32) {
        if (t % 32 == 0) tops[t / 32] = top;
        meet();
        for (uint32_t w = 0; w < THREADS / 32; w++) top = max(top, tops[w]);
    } else {
        meet();
    }
    const bool anew = written[0] & 1u;
    const float old = anew ? 0.f : was;
    // both are not negative or NaN: as bit patterns NaN is the largest
    const uint32_t old_bits = __float_as_uint(old) & 0x7FFFFFFFu;
    const float scale = __uint_as_float(max(old_bits, __float_as_uint(scale_of(top)))), inverse = inverse_of(scale);
    auto put = [&](uint32_t i, const float (&x)[8], const float (&y)[8]) {
        const uint32_t r = i / steps, p = (i - r * steps) * 8;
        int8_t *dst = cache + (size_t)slot_of(r0 + r) * row_bytes + p;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(codes_of(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse),
                                                     codes_of(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse));
        *reinterpret_cast<uint2 *>(dst + half) = make_uint2(codes_of(y[0] * inverse, y[1] * inverse, y[2] * inverse, y[3] * inverse),
                                                            codes_of(y[4] * inverse, y[5] * inverse, y[6] * inverse, y[7] * inverse));
    };
#pragma unroll
    for (int b = 0; b < kHold; b++)
        if (b * THREADS + t < items) put(b * THREADS + t, lo[b], hi[b]);
    for (uint32_t i = kHold * THREADS + t; i < items; i += THREADS) {
        float x[8], y[8];
        fetch(i, x, y);
        turn(i, x, y);
        put(i, x, y);
    }
    if (!anew && old_bits != __float_as_uint(scale)) {
        const float ratio = inverse != 0.f ? old / scale : 0.f;
        const uint32_t pieces = a.d / 16;
        for (uint32_t i = t; i < block * pieces; i += THREADS) {
            const uint32_t at = i / pieces;
            if (written[at / 32] >> (at & 31u) & 1u) continue;
            uint4 *p = reinterpret_cast<uint4 *>(cache + (((size_t)id << a.block_shift) + at) * row_bytes) + (i - at * pieces);
            uint4 v = *p;
            uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int8_t *c = reinterpret_cast<const int8_t *>(&w[e]);
                w[e] = codes_of(c[0] * ratio, c[1] * ratio, c[2] * ratio, c[3] * ratio);
            }
            *p = v;
        }
    }
    meet();                                              // the notes and the old scale have been read by all
    if (t == 0) *scale_at = scale;
}

template <typename S, typename T, bool MANY>             // source, rotated queries; several jobs
__global__ void __launch_bounds__(kThreads, kCtas) append8_kernel(const Append8Args a, bool wide)
{
    __shared__ double s_frequency[MGQ_PAGED_MAX_HEAD / 2];
    __shared__ float2 s_turn[kThreads];
    __shared__ uint32_t s_written[kWarps][kMostBlock / 32], s_top[kWarps];
    const uint32_t t = threadIdx.x, half = a.d / 2, steps = half / 8;
    if (a.rotate && t < half) s_frequency[t] = exp2(-a.log2_theta * (double)t / (double)half);
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();
    if (blockIdx.x >= a.cache_ctas) {                    // queries: as many rows at a time as have an angle for every thread
        const uint32_t at_once = kThreads / half, row_items = a.q_heads * steps;
        for (uint32_t r0 = (blockIdx.x - a.cache_ctas) * at_once; r0 < a.rows; r0 += (gridDim.x - a.cache_ctas) * at_once) {
            const uint32_t rows = min(at_once, a.rows - r0);
            float x[8], y[8];
            auto fetch = [&](uint32_t i) {
                const uint32_t r = i / row_items, in_row = i - r * row_items, head = in_row / steps;
                const S *src = static_cast<const S *>(a.q) + (size_t)(r0 + r) * a.q_pitch + head * a.d + (in_row - head * steps) * 8;
                read8(src, x, wide);
                read8(src + half, y, wide);
            };
            if (t < rows * row_items) fetch(t);          // on its way while the angles are found
            if (a.rotate) {
                if (t < rows * half) s_turn[t] = turn_of(a.positions[r0 + t / half], s_frequency[t % half]);
                __syncthreads();
            }
            for (uint32_t i = t; i < rows * row_items; i += kThreads) {
                if (i != t) fetch(i);
                const uint32_t r = i / row_items, in_row = i - r * row_items, head = in_row / steps, p = (in_row - head * steps) * 8;
                T lo[8], hi[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float2 w = a.rotate ? s_turn[r * half + p + e] : make_float2(1.f, 0.f);
                    lo[e] = rounded<T>(x[e] * w.x - y[e] * w.y);
                    hi[e] = rounded<T>(x[e] * w.y + y[e] * w.x);
                }
                T *to = static_cast<T *>(a.q_out) + ((size_t)(r0 + r) * a.q_heads + head) * a.d + p;
                if (wide) {
                    *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(lo);
                    *reinterpret_cast<uint4 *>(to + half) = *reinterpret_cast<const uint4 *>(hi);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        to[e] = lo[e];
                        to[half + e] = hi[e];
                    }
                }
            }
            if (a.rotate) __syncthreads();
        }
        return;
    }
    // the window's slots, the one in front and 256 behind
    __shared__ uint32_t s_slots[1 + kMostWindow + kThreads], s_earlier, s_later, s_filter[kThreads], s_rows[kMostBlock], s_count;
    const uint32_t jobs = MANY ? a.jobs : 1u, groups = 2 * a.kv_heads / jobs, job0 = blockIdx.x % groups * jobs, from = blockIdx.x / groups * a.window;
    // all rows' slots are looked at below: the first 256 and 4096 more are on their way while the window's are fetched
    auto four_slots = [&](uint32_t r) {
        if (r + 3 < a.rows && reinterpret_cast<uintptr_t>(a.slots) % 16 == 0) return *reinterpret_cast<const uint4 *>(a.slots + r);
        auto slot = [&](uint32_t r) { return r < a.rows ? a.slots[r] : 0xFFFFFFFFu; };
        return make_uint4(slot(r), slot(r + 1), slot(r + 2), slot(r + 3));
    };
    constexpr int kLooks = 4;
    const uint32_t first = t < a.rows ? a.slots[t] : 0xFFFFFFFFu;
    uint4 more[kLooks];
    if (a.rows > kThreads)
#pragma unroll
        for (int i = 0; i < kLooks; i++)
            if (kThreads + 4 * i * kThreads < a.rows) more[i] = four_slots(kThreads + 4 * (i * kThreads + t));
    for (uint32_t i = t; i < 1 + kMostWindow + kThreads; i += kThreads) {
        const uint32_t r = from + i - 1;                 // row -1 is none
        s_slots[i] = r < a.rows ? a.slots[r] : 0xFFFFFFFFu;
    }
    s_filter[t] = 0;
    if (t == 0) s_earlier = s_later = 0;
    __syncthreads();
    const uint32_t lane = t & 31u, warp = t >> 5, before = s_slots[lane], slot = s_slots[lane + 1], mine = slot >> a.block_shift;
    const bool begins = lane < a.window && slot < a.slots_end && !(before < a.slots_end && before >> a.block_shift == mine);
    const uint32_t runs = __ballot_sync(0xffffffffu, begins);
    if (!runs) return;
    auto slot_of = [&](uint32_t r) { return r - from + 1 < 1 + kMostWindow + kThreads ? s_slots[r - from + 1] : r < a.rows ? a.slots[r] : 0xFFFFFFFFu; };
    auto rows_of = [&](uint32_t r0) {                    // whole warps
        const uint32_t id = slot_of(r0) >> a.block_shift;
        for (uint32_t n = 0;; n += 32) {
            const uint32_t slot = slot_of(r0 + n + lane), rest = __ballot_sync(0xffffffffu, !(slot < a.slots_end && slot >> a.block_shift == id));
            if (rest) return n + __ffs(rest) - 1;
        }
    };
    // s_earlier, s_later: runs whose block has rows in front of and behind them, too.  Every warp looks at a part of the rows, for bits of the runs' blocks in s_filter (which all
    // warps set alike), where a row's block is not that of the row in front (or the row is a lane's first).
    {
        const uint32_t last = from + 31 - __clz(runs), end = max(from + a.window, last + rows_of(last));
        if (begins) atomicOr(&s_filter[mine >> 5 & (kThreads - 1)], 1u << (mine & 31u));
        uint32_t i = 0;
        for (uint32_t left = runs; left & left - 1; left &= left - 1, i++) {          // against those behind it in the window
            if (i % kWarps != warp) continue;
            const uint32_t one = left & -left, same = __ballot_sync(0xffffffffu, begins && mine == s_slots[__ffs(left)] >> a.block_shift) & ~(one | one - 1);
            if (same && lane == 0) {
                atomicOr(&s_later, one);
                atomicOr(&s_earlier, same);
            }
        }
        __syncwarp();
        auto meets = [&](uint32_t id) { return s_filter[id >> 5 & (kThreads - 1)] >> (id & 31u) & 1u; };
        auto look = [&](uint32_t r, uint32_t slot) {
            if (slot >= a.slots_end || (r >= from && r < end)) return;
            for (uint32_t left = runs; left; left &= left - 1)
                if (s_slots[__ffs(left)] >> a.block_shift == slot >> a.block_shift) atomicOr(r < from ? &s_earlier : &s_later, left & -left);
        };
        auto look_at_four = [&](uint32_t r, uint4 v) {
            const uint32_t x = v.x >> a.block_shift, y = v.y >> a.block_shift, z = v.z >> a.block_shift, w = v.w >> a.block_shift;
            uint32_t hits = meets(x);
            if (y != x) hits |= meets(y) << 1;
            if (z != y) hits |= meets(z) << 2;
            if (w != z) hits |= meets(w) << 3;
#pragma unroll 1
            for (; hits; hits &= hits - 1) look(r + __ffs(hits) - 1, hits & 1u ? v.x : hits & 2u ? v.y : hits & 4u ? v.z : v.w);
        };
        if (meets(first >> a.block_shift)) look(t, first);
        if (a.rows > kThreads) {
#pragma unroll 1
            for (uint32_t r = kThreads + 4 * t;;) {
#pragma unroll
                for (int i = 0; i < kLooks; i++)
                    if (r - 4 * t + 4 * i * kThreads < a.rows) look_at_four(r + 4 * i * kThreads, more[i]);
                r += 4 * kLooks * kThreads;
                if (r - 4 * t >= a.rows) break;
#pragma unroll
                for (int i = 0; i < kLooks; i++) more[i] = four_slots(r + 4 * i * kThreads);
            }
        }
        __syncthreads();
    }
    // Blocks whose rows stand apart, first rows of theirs: value by value, as what counts is that little of this stands beside the rest.
    const uint32_t mixed = s_earlier | s_later;
#pragma unroll 1
    for (uint32_t left = s_later & ~s_earlier; left; left &= left - 1) {
        const uint32_t r0 = from + __ffs(left) - 1, id = slot_of(r0) >> a.block_shift, block = 1u << a.block_shift;
        __syncthreads();
        if (t == 0) s_count = 0;
        for (uint32_t w = t; w < (block + 31) / 32; w += kThreads) s_written[0][w] = 0;
        __syncthreads();
        for (uint32_t r = r0 + t; r < a.rows; r += kThreads) {
            const uint32_t slot = a.slots[r], at = slot & (block - 1);
            if (slot >= a.slots_end || slot >> a.block_shift != id) continue;
            const uint32_t i = atomicAdd(&s_count, 1u);
            if (i < kMostBlock) s_rows[i] = r;           // always, as slots differ
            atomicOr(&s_written[0][at / 32], 1u << (at & 31u));
        }
        __syncthreads();
        const uint32_t n = min(s_count, kMostBlock);
#pragma unroll 1
        for (uint32_t job = job0; job < job0 + jobs; job++) {
            const uint32_t head = job >> 1;
            const bool values = job & 1u, rotate = a.rotate && !values;
            const size_t row_bytes = (size_t)a.kv_heads * a.d;
            int8_t *cache = (values ? a.v_cache : a.k_cache) + (size_t)head * a.d;
            float *scale_at = (values ? a.v_scales : a.k_scales) + (size_t)id * a.kv_heads + head, scale = 0.f;
            uint32_t top = 0;
#pragma unroll 1
            for (int pass = 0; pass < 2; pass++) {
                const float inverse = inverse_of(scale);
#pragma unroll 1
                for (uint32_t i = t; i < n * half; i += kThreads) {
                    const uint32_t r = s_rows[i / half], p = i % half;
                    const S *row = static_cast<const S *>(values ? a.v : a.k) + (size_t)r * (values ? a.v_pitch : a.k_pitch) + (size_t)head * a.d + p;
                    float x = to_f32(row[0]), y = to_f32(row[half]);
                    if (rotate) rotate_pair(x, y, turn_of(a.positions[r], s_frequency[p]));
                    if (pass) {
                        int8_t *to = cache + (size_t)a.slots[r] * row_bytes + p;
                        to[0] = (int8_t)__float2int_rn(x * inverse);
                        to[half] = (int8_t)__float2int_rn(y * inverse);
                    } else {
                        top = max(top, max(__float_as_uint(x) & 0x7FFFFFFFu, __float_as_uint(y) & 0x7FFFFFFFu));
                    }
                }
                if (pass) break;
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) s_top[warp] = top;
                __syncthreads();
                for (uint32_t w = 0; w < kWarps; w++) top = max(top, s_top[w]);
                const bool anew = s_written[0][0] & 1u;
                const float old = anew ? 0.f : fabsf(*scale_at);
                scale = __uint_as_float(max(__float_as_uint(old), __float_as_uint(scale_of(top))));
                if (!anew && __float_as_uint(old) != __float_as_uint(scale)) {
                    const float ratio = inverse_of(scale) != 0.f ? old / scale : 0.f;
                    for (uint32_t i = t; i < block * a.d; i += kThreads) {
                        const uint32_t at = i / a.d;
                        int8_t *c = cache + ((size_t)id * block + at) * row_bytes + (i - at * a.d);
                        if (!(s_written[0][at / 32] >> (at & 31u) & 1u)) *c = (int8_t)max(min(__float2int_rn(*c * ratio), 127), -128);
                    }
                }
            }
            __syncthreads();                             // the old scale and the warps' largest have been read
            if (t == 0) *scale_at = scale;
        }
    }
    uint32_t shorter = 0;
    for (uint32_t left = runs & ~mixed; left; left &= left - 1) {
        const uint32_t r0 = from + __ffs(left) - 1, n = rows_of(r0);
        if (n > kShort)
            for (uint32_t job = job0; job < job0 + jobs; job++) store_run<S, kThreads>(a, s_frequency, s_written[0], s_top, r0, n, job >> 1, job & 1u, wide, slot_of);
        else
            shorter |= left & -left;
    }
    for (uint32_t i = 0; shorter; shorter &= shorter - 1) {
        const uint32_t r0 = from + __ffs(shorter) - 1;
        for (uint32_t job = job0; job < job0 + jobs; job++, i++)
            if (i % kWarps == warp) store_run<S, 32>(a, s_frequency, s_written[warp], s_top, r0, rows_of(r0), job >> 1, job & 1u, wide, slot_of);
    }
}

template <typename S, typename T>
int launch_typed(Append8Args &a, bool wide, cudaStream_t stream)
{
    a.window = min(max((uint32_t)((unsigned long long)a.rows * 2 * a.kv_heads / (148 * 8)), 1u), kMostWindow);
    const uint32_t windows = (a.rows + a.window - 1) / a.window, all = 2 * a.kv_heads;
    a.jobs = (uint32_t)min(max((unsigned long long)windows * all / (148 * 6), 1ull), (unsigned long long)all);
    while (all % a.jobs) a.jobs--;
    a.cache_ctas = windows * (all / a.jobs);
    const uint32_t at_once = 2 * kThreads / a.d;         // rows of queries
    const dim3 grid(a.cache_ctas + (a.q ? min((a.rows + at_once - 1) / at_once, 148u * 4u) : 0u));
    return launch(a.jobs > 1 ? append8_kernel<S, T, true> : append8_kernel<S, T, false>, grid, dim3(kThreads), 0, stream, a, wide);
}

}  // namespace

int launch_paged_append_int8(const void *q, const void *k, const void *v, int src_dtype, const uint32_t *positions, const uint32_t *slots, void *q_out, int q_dtype,
                             int8_t *k_cache, int8_t *v_cache, float *k_scales, float *v_scales, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
                             uint32_t q_pitch, uint32_t k_pitch, uint32_t v_pitch, uint32_t page_size, uint32_t pages, uint32_t block, float theta, void *stream)
{
    Append8Args a{q, k, v, positions, slots, q_out, k_cache, v_cache, k_scales, v_scales, rows, q ? q_heads : 0u, kv_heads, head_dim, q_pitch, k_pitch, v_pitch,
                  pages * page_size, page_shift(block), 1, 1, 0, theta > 0.f ? log2((double)theta) : 0.0, theta > 0.f};
    auto fits = [](const void *p, uint32_t pitch, int dtype) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % (16 / element_bytes(dtype)) == 0); };
    const bool wide = fits(q, q_pitch, src_dtype) && fits(k, k_pitch, src_dtype) && fits(v, v_pitch, src_dtype) && fits(q_out, 0, q_dtype);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (src_dtype == MGQ_FMT_F32) return q_dtype == MGQ_FMT_F16 ? launch_typed<float, __half>(a, wide, s) : launch_typed<float, __nv_bfloat16>(a, wide, s);
    return src_dtype == MGQ_FMT_F16 ? launch_typed<__half, __half>(a, wide, s) : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, wide, s);
}

}  // namespace mgq
