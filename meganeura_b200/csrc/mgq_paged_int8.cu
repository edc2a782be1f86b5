// New keys and values into a paged cache of 8-bit codes with a scale for each block of tokens and head.
#include "mgq_paged_int8.cuh"

namespace mgq {
namespace {

// A block's scale is that of its largest value, so its rows belong together: those of a step that fall into one block stand one behind another, and the CTA of
// the first of them takes all, for one head of the keys or of the values.  new = max(old, largest / 127), where old is 0 if the block's first slot is among
// them: the block starts anew.  Codes that the block holds already become rint(code * old / new) where the scale grew.
// Rotated values stay in registers between the pass for the largest and the one for the codes, kHold steps of 8 values a thread (64 rows of 128); what
// lies behind is computed again.
constexpr int kThreads = 256, kHold = 4;
constexpr uint32_t kMostBlock = 1024;

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
__device__ __forceinline__ void read4(const T *p, float (&f)[4], bool wide)
{
    if (!wide) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = to_f32(p[i]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = to_f32(e[i]);
    }
}

template <typename S, typename T>                        // source, rotated queries
__global__ void __launch_bounds__(kThreads) append8_kernel(const Append8Args a, bool wide)
{
    __shared__ double s_frequency[MGQ_PAGED_MAX_HEAD / 2];
    __shared__ float2 s_turn[MGQ_PAGED_MAX_HEAD / 2];
    __shared__ uint32_t s_written[kMostBlock / 32], s_top[kThreads / 32];
    const uint32_t t = threadIdx.x, half = a.d / 2, steps = half / 4;
    if (a.rotate && t < half) s_frequency[t] = exp2(-a.log2_theta * (double)t / (double)half);
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();
    if (blockIdx.x >= a.cache_ctas) {                    // queries: a row at a time
        for (uint32_t r = blockIdx.x - a.cache_ctas; r < a.rows; r += gridDim.x - a.cache_ctas) {
            if (a.rotate) {
                if (t < half) s_turn[t] = turn_of(a.positions[r], s_frequency[t]);
                __syncthreads();
            }
            for (uint32_t i = t; i < a.q_heads * steps; i += kThreads) {
                const uint32_t head = i / steps, p = (i - head * steps) * 4;
                const S *src = static_cast<const S *>(a.q) + (size_t)r * a.q_pitch + head * a.d + p;
                T *dst = static_cast<T *>(a.q_out) + ((size_t)r * a.q_heads + head) * a.d + p;
                float x[4], y[4];
                read4(src, x, wide);
                read4(src + half, y, wide);
                T lo[4], hi[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 w = a.rotate ? s_turn[p + e] : make_float2(1.f, 0.f);
                    lo[e] = rounded<T>(x[e] * w.x - y[e] * w.y);
                    hi[e] = rounded<T>(x[e] * w.y + y[e] * w.x);
                    if (!wide) {
                        dst[e] = lo[e];
                        dst[half + e] = hi[e];
                    }
                }
                if (wide) {
                    *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(lo);
                    *reinterpret_cast<uint2 *>(dst + half) = *reinterpret_cast<const uint2 *>(hi);
                }
            }
            if (a.rotate) __syncthreads();
        }
        return;
    }
    const uint32_t job = blockIdx.x % (2 * a.kv_heads), head = job >> 1, block = 1u << a.block_shift;
    const bool values = job & 1u, rotate = a.rotate && !values;
    const uint32_t from = blockIdx.x / (2 * a.kv_heads) * a.window, pitch = values ? a.v_pitch : a.k_pitch;
    const S *src = static_cast<const S *>(values ? a.v : a.k) + (size_t)head * a.d;
    int8_t *cache = (values ? a.v_cache : a.k_cache) + (size_t)head * a.d;
    float *scales = values ? a.v_scales : a.k_scales;
    const size_t row_bytes = (size_t)a.kv_heads * a.d;
    for (uint32_t r0 = from; r0 < min(from + a.window, a.rows); r0++) {
        const uint32_t first = a.slots[r0], id = first >> a.block_shift;
        if (first >= a.slots_end) continue;
        if (r0 > 0) {                                    // another CTA's, or of this window's rows before
            const uint32_t before = a.slots[r0 - 1];
            if (before < a.slots_end && before >> a.block_shift == id) continue;
        }
        // the rows of this block, and its slots that they fill
        for (uint32_t w = t; w < (block + 31) / 32; w += kThreads) s_written[w] = 0;
        __syncthreads();
        uint32_t n = 0;
        for (bool more = true; more;) {
            const uint32_t r = r0 + n + t, slot = r < a.rows ? a.slots[r] : 0xFFFFFFFFu;
            const bool here = slot < a.slots_end && slot >> a.block_shift == id;
            const uint32_t rest = __ballot_sync(0xffffffffu, !here);
            if (t % 32 == 0) s_top[t / 32] = rest ? (uint32_t)__ffs(rest) - 1 : 32u;
            __syncthreads();
            uint32_t count = 0;
            for (uint32_t w = 0; w < kThreads / 32; w++) {
                count += s_top[w];
                if (s_top[w] < 32) break;
            }
            if (t < count) atomicOr(&s_written[(slot & (block - 1)) / 32], 1u << (slot & (block - 1) & 31u));
            n += count;
            more = count == kThreads;
            __syncthreads();
        }
        const float old = s_written[0] & 1u ? 0.f : scales[(size_t)id * a.kv_heads + head];
        const uint32_t items = n * steps;                // four pairs of a row each
        auto fetch = [&](uint32_t i, float (&lo)[4], float (&hi)[4]) {
            const uint32_t r = i / steps, p = (i - r * steps) * 4;
            const S *row = src + (size_t)(r0 + r) * pitch + p;
            read4(row, lo, wide);
            read4(row + half, hi, wide);
            if (!rotate) return;
            const uint32_t position = a.positions[r0 + r];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 w = turn_of(position, s_frequency[p + e]);
                const float x = lo[e] * w.x - hi[e] * w.y;
                hi[e] = lo[e] * w.y + hi[e] * w.x;
                lo[e] = x;
            }
        };
        float lo[kHold][4], hi[kHold][4];
        uint32_t top = 0;
        auto larger = [&](const float (&f)[4]) {
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
        };
#pragma unroll
        for (int b = 0; b < kHold; b++)
            if (b * kThreads + t < items) {
                fetch(b * kThreads + t, lo[b], hi[b]);
                larger(lo[b]);
                larger(hi[b]);
            }
        for (uint32_t i = kHold * kThreads + t; i < items; i += kThreads) {
            float x[4], y[4];
            fetch(i, x, y);
            larger(x);
            larger(y);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (t % 32 == 0) s_top[t / 32] = top;
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; w++) top = max(top, s_top[w]);
        // both are not negative or NaN: as bit patterns NaN is the largest
        const uint32_t old_bits = __float_as_uint(old) & 0x7FFFFFFFu;
        const float scale = __uint_as_float(max(old_bits, __float_as_uint(scale_of(top)))), inverse = inverse_of(scale);
        auto put = [&](uint32_t i, const float (&x)[4], const float (&y)[4]) {
            const uint32_t r = i / steps, p = (i - r * steps) * 4;
            int8_t *dst = cache + (size_t)a.slots[r0 + r] * row_bytes + p;
            *reinterpret_cast<uint32_t *>(dst) = codes_of(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse);
            *reinterpret_cast<uint32_t *>(dst + half) = codes_of(y[0] * inverse, y[1] * inverse, y[2] * inverse, y[3] * inverse);
        };
#pragma unroll
        for (int b = 0; b < kHold; b++)
            if (b * kThreads + t < items) put(b * kThreads + t, lo[b], hi[b]);
        for (uint32_t i = kHold * kThreads + t; i < items; i += kThreads) {
            float x[4], y[4];
            fetch(i, x, y);
            put(i, x, y);
        }
        if (!(s_written[0] & 1u) && old_bits != __float_as_uint(scale)) {
            const float ratio = inverse != 0.f ? old / scale : 0.f;
            const uint32_t words = a.d / 4;
            for (uint32_t i = t; i < block * words; i += kThreads) {
                const uint32_t at = i / words;
                if (s_written[at / 32] >> (at & 31u) & 1u) continue;
                uint32_t *p = reinterpret_cast<uint32_t *>(cache + (((size_t)id << a.block_shift) + at) * row_bytes) + (i - at * words);
                const uint32_t w = *p;
                const int8_t *c = reinterpret_cast<const int8_t *>(&w);
                *p = codes_of(c[0] * ratio, c[1] * ratio, c[2] * ratio, c[3] * ratio);
            }
        }
        __syncthreads();                                 // the old scale has been read by all
        if (t == 0) scales[(size_t)id * a.kv_heads + head] = scale;
    }
}

template <typename S, typename T>
int launch_typed(Append8Args &a, bool wide, cudaStream_t stream)
{
    a.window = a.rows <= 1024 ? 1 : 4;
    a.cache_ctas = (a.rows + a.window - 1) / a.window * 2 * a.kv_heads;
    return launch(append8_kernel<S, T>, dim3(a.cache_ctas + (a.q ? min(a.rows, 148u * 4u) : 0u)), dim3(kThreads), 0, stream, a, wide);
}

}  // namespace

int launch_paged_append_int8(const void *q, const void *k, const void *v, int src_dtype, const uint32_t *positions, const uint32_t *slots, void *q_out, int q_dtype,
                             int8_t *k_cache, int8_t *v_cache, float *k_scales, float *v_scales, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
                             uint32_t q_pitch, uint32_t k_pitch, uint32_t v_pitch, uint32_t page_size, uint32_t pages, uint32_t block, float theta, void *stream)
{
    Append8Args a{q, k, v, positions, slots, q_out, k_cache, v_cache, k_scales, v_scales, rows, q ? q_heads : 0u, kv_heads, head_dim, q_pitch, k_pitch, v_pitch,
                  pages * page_size, page_shift(block), 1, 0, theta > 0.f ? log2((double)theta) : 0.0, theta > 0.f};
    auto fits = [](const void *p, uint32_t pitch, int dtype) { return !p || (reinterpret_cast<uintptr_t>(p) % (4 * element_bytes(dtype)) == 0 && pitch % 4 == 0); };
    const bool wide = fits(q, q_pitch, src_dtype) && fits(k, k_pitch, src_dtype) && fits(v, v_pitch, src_dtype) && fits(q_out, 0, q_dtype);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (src_dtype == MGQ_FMT_F32) return q_dtype == MGQ_FMT_F16 ? launch_typed<float, __half>(a, wide, s) : launch_typed<float, __nv_bfloat16>(a, wide, s);
    return src_dtype == MGQ_FMT_F16 ? launch_typed<__half, __half>(a, wide, s) : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, wide, s);
}

}  // namespace mgq
