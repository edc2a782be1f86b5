// New keys and values into a paged cache of 8-bit codes with a scale for each block of tokens and head.
#include "mgq_paged_int8.cuh"

namespace mgq {
namespace {

// A block's scale is that of its largest value, so its rows belong together: those of a step that fall into one block, a run, stand one behind another.  A CTA
// takes the runs that begin in a window of rows, for one head of the keys or of the values: a run of more than kShort rows by all its threads, shorter ones by a
// warp each.  new = max(old, largest / 127), where old is 0 if the block's first slot is among the rows: the block starts anew.  Codes that the block holds already
// become rint(code * old / new) where the scale grew.  Rotated values stay in registers between the pass for the largest and the one for the codes, kHold
// steps of 16 values a thread (32 rows of 128 for a CTA); what lies behind is computed again.
// Loads that wait for one another bound it (slots, then scale and rows, then what is held), so CTAs per SM count more than registers: 4096 rows of the Qwen3-8B shape
// took 52, 45, 39 us with two, three, four; and windows are as wide as leaves eight CTAs per SM.
constexpr int kThreads = 256, kWarps = kThreads / 32, kHold = 1, kCtas = 4;
constexpr uint32_t kMostBlock = 1024, kMostWindow = 32, kShort = 4;

struct Append8Args {
    const void *q, *k, *v;
    const uint32_t *positions, *slots;
    void *q_out;
    int8_t *k_cache, *v_cache;
    float *k_scales, *v_scales;
    uint32_t rows, q_heads, kv_heads, d, q_pitch, k_pitch, v_pitch, slots_end, block_shift, window, cache_ctas;
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
        for (int e = 0; e < 8; e++) {
            const float2 w = turn_of(position, frequency[p + e]);
            const float x = lo[e] * w.x - hi[e] * w.y;
            hi[e] = lo[e] * w.y + hi[e] * w.x;
            lo[e] = x;
        }
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

template <typename S, typename T>                        // source, rotated queries
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
    __shared__ uint32_t s_slots[1 + kMostWindow + kThreads], s_runs;
    const uint32_t job = blockIdx.x % (2 * a.kv_heads), head = job >> 1, from = blockIdx.x / (2 * a.kv_heads) * a.window;
    const bool values = job & 1u;
    for (uint32_t i = t; i < 1 + kMostWindow + kThreads; i += kThreads) {
        const uint32_t r = from + i - 1;                 // row -1 is none
        s_slots[i] = r < a.rows ? a.slots[r] : 0xFFFFFFFFu;
    }
    __syncthreads();
    if (t < 32) {
        const uint32_t before = s_slots[t], slot = s_slots[t + 1];
        const bool begins = t < a.window && slot < a.slots_end && !(before < a.slots_end && before >> a.block_shift == slot >> a.block_shift);
        const uint32_t runs = __ballot_sync(0xffffffffu, begins);
        if (t == 0) s_runs = runs;
    }
    __syncthreads();
    const uint32_t lane = t & 31u, warp = t >> 5, runs = s_runs;
    auto slot_of = [&](uint32_t r) { return r - from + 1 < 1 + kMostWindow + kThreads ? s_slots[r - from + 1] : r < a.rows ? a.slots[r] : 0xFFFFFFFFu; };
    auto rows_of = [&](uint32_t r0) {                    // whole warps
        const uint32_t id = slot_of(r0) >> a.block_shift;
        for (uint32_t n = 0;; n += 32) {
            const uint32_t slot = slot_of(r0 + n + lane), rest = __ballot_sync(0xffffffffu, !(slot < a.slots_end && slot >> a.block_shift == id));
            if (rest) return n + __ffs(rest) - 1;
        }
    };
    uint32_t shorter = 0;
    for (uint32_t left = runs; left; left &= left - 1) {
        const uint32_t r0 = from + __ffs(left) - 1, n = rows_of(r0);
        if (n > kShort) store_run<S, kThreads>(a, s_frequency, s_written[0], s_top, r0, n, head, values, wide, slot_of);
        else            shorter |= left & -left;
    }
    for (uint32_t i = 0; shorter; shorter &= shorter - 1, i++) {
        const uint32_t r0 = from + __ffs(shorter) - 1;
        if (i % kWarps == warp) store_run<S, 32>(a, s_frequency, s_written[warp], s_top, r0, rows_of(r0), head, values, wide, slot_of);
    }
}

template <typename S, typename T>
int launch_typed(Append8Args &a, bool wide, cudaStream_t stream)
{
    a.window = min(max((uint32_t)((unsigned long long)a.rows * 2 * a.kv_heads / (148 * 8)), 1u), kMostWindow);
    a.cache_ctas = (a.rows + a.window - 1) / a.window * 2 * a.kv_heads;
    const uint32_t at_once = 2 * kThreads / a.d;         // rows of queries
    return launch(append8_kernel<S, T>, dim3(a.cache_ctas + (a.q ? min((a.rows + at_once - 1) / at_once, 148u * 4u) : 0u)), dim3(kThreads), 0, stream, a, wide);
}

}  // namespace

int launch_paged_append_int8(const void *q, const void *k, const void *v, int src_dtype, const uint32_t *positions, const uint32_t *slots, void *q_out, int q_dtype,
                             int8_t *k_cache, int8_t *v_cache, float *k_scales, float *v_scales, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
                             uint32_t q_pitch, uint32_t k_pitch, uint32_t v_pitch, uint32_t page_size, uint32_t pages, uint32_t block, float theta, void *stream)
{
    Append8Args a{q, k, v, positions, slots, q_out, k_cache, v_cache, k_scales, v_scales, rows, q ? q_heads : 0u, kv_heads, head_dim, q_pitch, k_pitch, v_pitch,
                  pages * page_size, page_shift(block), 1, 0, theta > 0.f ? log2((double)theta) : 0.0, theta > 0.f};
    auto fits = [](const void *p, uint32_t pitch, int dtype) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % (16 / element_bytes(dtype)) == 0); };
    const bool wide = fits(q, q_pitch, src_dtype) && fits(k, k_pitch, src_dtype) && fits(v, v_pitch, src_dtype) && fits(q_out, 0, q_dtype);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (src_dtype == MGQ_FMT_F32) return q_dtype == MGQ_FMT_F16 ? launch_typed<float, __half>(a, wide, s) : launch_typed<float, __nv_bfloat16>(a, wide, s);
    return src_dtype == MGQ_FMT_F16 ? launch_typed<__half, __half>(a, wide, s) : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, wide, s);
}

}  // namespace mgq
