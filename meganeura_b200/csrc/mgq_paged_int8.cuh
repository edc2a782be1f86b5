// What the kernels over a paged cache of 8-bit codes share.
#pragma once
#include "mgq_int8.cuh"
#include "mgq_paged.cuh"

namespace mgq {

// A cache's codes are [pages, page_size, kv_heads, d], its scales [pages, page_size / block, kv_heads]: slot s of the cache belongs to block s / block.
struct Attend8Args : AttendArgs {
    const float *k_scales, *v_scales;
    uint32_t block_shift;
};

// Few new tokens per sequence (mgq_paged_int8_decode.cu).
uint32_t decode8_ctas(uint32_t head_dim);
constexpr uint32_t kDecode8Rows = 32;                      // of a unit, at most
// Pairs of a sequence that is not yet many tokens': 32 sequences of the Qwen3-8B shape with 32 pairs take 90 us with the kernel for few tokens and 97 with the other,
// with 48 pairs 131 and 98.
constexpr uint32_t kDecode8Pairs = 32;
int launch_decode8(const Attend8Args &a, int dtype, uint32_t pairs, cudaStream_t stream);    // pairs: a bound of a sequence's tokens * heads per key / value head

// Many new tokens: heads of up to 128, queries and results on 16 bytes (mgq_paged_int8_prefill.cu).
bool prefill8_takes(const Attend8Args &a);
int launch_prefill8(const Attend8Args &a, int dtype, cudaStream_t stream);

}  // namespace mgq
