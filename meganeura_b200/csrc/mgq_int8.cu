// Rows quantized to 8-bit integers with a scale each, and products of such rows: the quantizer, the kernel for few rows, and which kernel serves a product.
#include "mgq_int8.cuh"

namespace mgq {
namespace {

// ---------------------------------------------------------------- rows of codes
// scale = max |x| / 127, code = rint(x / scale).  One pass over HBM: a CTA takes a row and keeps it in registers as it was read, 8 values a thread and step, up to
// kHold steps (16384 values at 512 threads); what lies behind is read again, from L2.  The largest magnitude is found among the bit patterns without their
// sign, whose order is that of the magnitudes with NaN above infinity, so that one that is not finite makes the scale so.
// 2048 x 12288 in bf16: 13.8 us from HBM, 5.5 TB/s, 11.2 where L2 holds the rows; 8 x 4096: 1.9 us in a graph, a launch.
constexpr int kHold = 4;
constexpr uint32_t kMostThreads = 512;

template <typename T, int N> struct Piece {              // N values as they lie in memory
    T v[N];
};
template <typename T>
__device__ __forceinline__ void fetch(Piece<T, 8> &p, const T *src)
{
    uint4 *dst = reinterpret_cast<uint4 *>(p.v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) dst[i] = reinterpret_cast<const uint4 *>(src)[i];
}
template <typename T>
__device__ __forceinline__ void fetch(Piece<T, 1> &p, const T *src) { p.v[0] = *src; }
template <typename T, int N>
__device__ __forceinline__ uint32_t largest(const Piece<T, N> &p, uint32_t top)
{
#pragma unroll
    for (int e = 0; e < N; e++) top = max(top, __float_as_uint(to_f32(p.v[e])) & 0x7FFFFFFFu);
    return top;
}
template <typename T, int N>
__device__ __forceinline__ void store(const Piece<T, N> &p, float inverse, int8_t *dst)
{
    if constexpr (N == 8) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = to_f32(p.v[e]) * inverse;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(codes_of(f[0], f[1], f[2], f[3]), codes_of(f[4], f[5], f[6], f[7]));
    } else {
        *dst = (int8_t)__float2int_rn(to_f32(p.v[0]) * inverse);
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(kMostThreads) quantize_rows_kernel(const T *x, uint32_t pitch, int8_t *codes, float *scales, uint32_t k)
{
    __shared__ uint32_t s_top[kMostThreads / 32];
    const uint32_t t = threadIdx.x, step = blockDim.x * N;
    const T *row = x + (size_t)blockIdx.x * pitch;
    int8_t *out = codes + (size_t)blockIdx.x * k;
    pdl_launch_dependents();
    pdl_wait();
    Piece<T, N> held[kHold];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kHold; i++)
        if (t * N + i * step < k) fetch(held[i], row + t * N + i * step);
#pragma unroll
    for (int i = 0; i < kHold; i++)
        if (t * N + i * step < k) top = largest(held[i], top);
    for (uint32_t at = t * N + kHold * step; at < k; at += step) {
        Piece<T, N> p;
        fetch(p, row + at);
        top = largest(p, top);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (t % 32 == 0) s_top[t / 32] = top;
    __syncthreads();
    for (uint32_t w = 0; w < blockDim.x / 32; w++) top = max(top, s_top[w]);
    const float scale = scale_of(top), inverse = inverse_of(scale);
    if (t == 0) scales[blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < kHold; i++)
        if (t * N + i * step < k) store(held[i], inverse, out + t * N + i * step);
    for (uint32_t at = t * N + kHold * step; at < k; at += step) {
        Piece<T, N> p;
        fetch(p, row + at);
        store(p, inverse, out + at);
    }
}

template <typename T>
int launch_quantize(const void *x, uint32_t pitch, int8_t *codes, float *scales, uint32_t rows, uint32_t k, cudaStream_t stream)
{
    const T *src = static_cast<const T *>(x);
    const bool wide = k % 8 == 0 && pitch % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
    // a step per thread where there are few rows; where there are more than four CTAs of the most threads per SM as many as a thread holds: 4096 rows of 4096 took 18.6 us
    // with a step each
    const uint32_t steps = ((wide ? k / 8 : k) + (rows > 148 * 4 ? kHold : 1) - 1) / (rows > 148 * 4 ? kHold : 1), threads = min((steps + 31) / 32 * 32, kMostThreads);
    return launch(wide ? quantize_rows_kernel<T, 8> : quantize_rows_kernel<T, 1>, dim3(rows), dim3(threads), 0, stream, src, pitch, codes, scales, k);
}

// ---------------------------------------------------------------- few rows
// HBM bound: the weights are read once.  m16n8k32 products of 16 weight rows (left) by up to 8 activation rows; the order of k inside a product is free as long
// as both operands have the same, so a lane loads 16 consecutive bytes of a row for two products, straight from global memory to registers.  The warps of a
// CTA share out k and meet in shared memory; sums are whole numbers, so their order is free.  The first weights are brought into L2 before the wait for the
// kernels in front, which may write activations and weights: a load before it could see old ones.
constexpr int kAhead = 4;                                // steps of 64 k that a warp has under way

__device__ __forceinline__ uint4 load_stream(const int8_t *p)
{
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) few_rows_kernel(const ProductArgs a)
{
    __shared__ int s_sum[WARPS][16][kFewRows + 1];
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, row = lane >> 2, quad = lane & 3u;
    const uint32_t n0 = blockIdx.x * 16, k = a.k;
    const uint32_t steps = (k + 63) / 64, from = steps * warp / WARPS, to = steps * (warp + 1) / WARPS;
    const int8_t *w0 = a.w + (size_t)min(n0 + row, a.n - 1) * k, *w1 = a.w + (size_t)min(n0 + row + 8, a.n - 1) * k;       // rows behind the last are not stored
    const int8_t *x = a.a + (size_t)min(row, a.m - 1) * k;
    int c[4] = {};
    uint4 w[kAhead][2], b[kAhead];
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    auto fetch = [&](uint32_t s, int slot) {
        const uint32_t at = s * 64 + quad * 16;
        const bool in = s < to && at < k;
        w[slot][0] = in ? load_stream(w0 + at) : none;
        w[slot][1] = in ? load_stream(w1 + at) : none;
        b[slot] = in ? *reinterpret_cast<const uint4 *>(x + at) : none;
    };
    if (quad == 0)
        for (uint32_t s = from & ~1u; s < min(from + kAhead, to); s += 2) {               // 128 bytes
            asm volatile("prefetch.global.L2 [%0];" ::"l"(w0 + s * 64));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(w1 + s * 64));
        }
    pdl_launch_dependents();
    pdl_wait();
#pragma unroll
    for (int i = 0; i < kAhead; i++) fetch(from + i, i);
    for (uint32_t s0 = from; s0 < to; s0 += kAhead)
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            mma_s8(c, w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, b[i].x, b[i].y);
            mma_s8(c, w[i][0].z, w[i][1].z, w[i][0].w, w[i][1].w, b[i].z, b[i].w);
            fetch(s0 + kAhead + i, i);
        }
#pragma unroll
    for (int e = 0; e < 4; e++) s_sum[warp][row + e / 2 * 8][2 * quad + e % 2] = c[e];
    __syncthreads();
    for (uint32_t i = t; i < 16 * a.m; i += WARPS * 32) {
        const uint32_t n = i % 16, m = i / 16;
        if (n0 + n >= a.n) continue;
        int sum = 0;
#pragma unroll
        for (int v = 0; v < WARPS; v++) sum += s_sum[v][n][m];
        finish<T>(a, m, n0 + n, sum, a.a_scales[m], a.w_scales[n0 + n]);
    }
}

// As many warps share a tile of 16 columns as let all tiles run at once: one CTA of sixteen on an SM, three of eight, seven or so of four.  8 rows of 4096 by 1536, 2304, 4096,
// 5900, 8192, 24576 columns take 2.9, 3.1, 5.7, 8.7, 11.1, 27.0 us with sixteen, 4.2, 4.6, 4.8, 5.5, 8.7, 16.9 with eight, 5.0, 5.5, 6.8, 7.7, 7.6, 17.4 with four.  Of k up to
// 1024 four bring all with their first loads: 1024 by 1536 columns 2.1, 2.3, 1.9.
template <typename T>
int launch_few(const ProductArgs &a, cudaStream_t stream)
{
    const uint32_t tiles = (a.n + 15) / 16;
    if (tiles > 3 * 148 || (tiles <= 148 && a.k <= 4 * kAhead * 64)) return launch(few_rows_kernel<T, 4>, dim3(tiles), dim3(128), 0, stream, a);
    return tiles > 148 ? launch(few_rows_kernel<T, 8>, dim3(tiles), dim3(256), 0, stream, a) : launch(few_rows_kernel<T, 16>, dim3(tiles), dim3(512), 0, stream, a);
}

}  // namespace

int launch_quantize_rows(const void *x, int dtype, uint32_t pitch, int8_t *codes, float *scales, uint32_t rows, uint32_t k, void *stream)
{
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case MGQ_FMT_F32: return launch_quantize<float>(x, pitch, codes, scales, rows, k, s);
        case MGQ_FMT_F16: return launch_quantize<__half>(x, pitch, codes, scales, rows, k, s);
        default: return launch_quantize<__nv_bfloat16>(x, pitch, codes, scales, rows, k, s);
    }
}

int launch_matmul_int8(const int8_t *x, const float *x_scales, const int8_t *w, const float *w_scales, const void *addend, void *out, int dtype, uint32_t m, uint32_t k,
                       uint32_t n, uint32_t addend_pitch, uint32_t out_pitch, void *stream)
{
    const ProductArgs a{x, w, x_scales, w_scales, addend, out, m, k, n, addend_pitch, out_pitch};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (m > kFewRows) return launch_product_tc(a, dtype, stream);
    switch (dtype) {
        case MGQ_FMT_F32: return launch_few<float>(a, s);
        case MGQ_FMT_F16: return launch_few<__half>(a, s);
        default: return launch_few<__nv_bfloat16>(a, s);
    }
}

}  // namespace mgq
