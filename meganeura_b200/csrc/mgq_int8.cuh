// What the kernels of 8-bit integers share: how a value becomes a code and a scale, and a product's arguments and end.
#pragma once
#include <cstdint>

#include "mgq_launch.cuh"

namespace mgq {

// Rows and blocks whose largest magnitude is below are zeros: their scale's inverse would leave f32's range.
constexpr float kLeast = 0x1p-100f;
// From the largest magnitude's bit pattern.  A 127th is a product with 1/127 as f32 rounds it, which is how torch divides a tensor by a number on the GPU (a true quotient is another
// in 4 % of the rows, by 2^-24, which some codes near a tie show); the inverse is rounded to nearest.  So scale and codes are the same as those of the same formulas there.
__device__ __forceinline__ float scale_of(uint32_t top) { return __uint_as_float(top) < kLeast ? 0.f : __uint_as_float(top) * (1.f / 127.f); }
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.f && scale < INFINITY ? 1.f / scale : 0.f; }
// Four values, in units of their scale, to the nearest whole numbers; NaN is 0.  At most 127 * (1 + 4 * 2^-24) comes in, so nothing is cut off.
__device__ __forceinline__ uint32_t codes_of(float x, float y, float z, float w)
{
    uint32_t v;
    asm("{\n\t.reg .b32 h;\n\t"
        "cvt.pack.sat.s8.s32.b32 h, %4, %3, 0;\n\t"
        "cvt.pack.sat.s8.s32.b32 %0, %2, %1, h;\n\t}"
        : "=r"(v) : "r"(__float2int_rn(x)), "r"(__float2int_rn(y)), "r"(__float2int_rn(z)), "r"(__float2int_rn(w)));
    return v;
}

// out[m, n] = (sum over k of a[m, k] w[n, k]) a_scales[m] w_scales[n] (+ addend[m, n])
struct ProductArgs {
    const int8_t *a, *w;
    const float *a_scales, *w_scales;
    const void *addend;
    void *out;
    uint32_t m, k, n, addend_pitch, out_pitch;
};
template <typename T> __device__ __forceinline__ T to_type(float y);
template <> __device__ __forceinline__ float to_type<float>(float y) { return y; }
template <> __device__ __forceinline__ __half to_type<__half>(float y) { return __float2half_rn(y); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type<__nv_bfloat16>(float y) { return __float2bfloat16_rn(y); }
template <typename T>
__device__ __forceinline__ void finish(const ProductArgs &a, uint32_t m, uint32_t n, int sum, float a_scale, float w_scale)
{
    float y = (float)sum * a_scale * w_scale;
    if (a.addend) y += to_f32(static_cast<const T *>(a.addend)[(size_t)m * a.addend_pitch + n]);
    static_cast<T *>(a.out)[(size_t)m * a.out_pitch + n] = to_type<T>(y);
}

// Activation rows up to which mma.sync (mgq_int8.cu) takes a product, with tcgen05 (mgq_int8_tc.cu) beyond.  8 rows of 4096 by 4096 and 24576 columns take 4.8 and 17.4 us
// there; 9 to 16, two blocks of columns for mma.sync, took 10.4 and 24.5, on tcgen05 6.2 and 19.1.
constexpr uint32_t kFewRows = 8;
int launch_product_tc(const ProductArgs &a, int dtype, void *stream);

}  // namespace mgq
