// What the attention kernels of many new tokens share: tiles, pairs of f32, a row of scores in TMEM, results turned for whole lines.
#pragma once
#include "mgq_paged.cuh"

namespace mgq {

constexpr uint32_t kKeys = 128, kTile = 128;             // keys of a block, rows of a tile
constexpr uint32_t kHalf = kKeys * 128;                  // 128 rows of 64 elements

template <typename T> __device__ __forceinline__ uint32_t pack(float x, float y);
template <> __device__ __forceinline__ uint32_t pack<__half>(float x, float y)
{
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float x, float y)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// The largest; NaN if one is NaN.
__device__ __forceinline__ float max3(float x, float y, float z)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// Two f32 side by side, for instructions that take two.
using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pair_of(float x, float y)
{
    pair_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ void parts_of(pair_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ pair_t pair_fma(pair_t x, pair_t y, pair_t z)
{
    pair_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
    return v;
}
__device__ __forceinline__ pair_t pair_add(pair_t x, pair_t y)
{
    pair_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
// 64 columns of this lane's row; wait_row before they are used.
__device__ __forceinline__ void tmem_ld_row(uint32_t addr, float (&y)[64])
{
#pragma unroll
    for (int c = 0; c < 64; c += 32)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                     "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                     "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                     : "=f"(y[c + 0]), "=f"(y[c + 1]), "=f"(y[c + 2]), "=f"(y[c + 3]), "=f"(y[c + 4]), "=f"(y[c + 5]), "=f"(y[c + 6]), "=f"(y[c + 7]),
                       "=f"(y[c + 8]), "=f"(y[c + 9]), "=f"(y[c + 10]), "=f"(y[c + 11]), "=f"(y[c + 12]), "=f"(y[c + 13]), "=f"(y[c + 14]), "=f"(y[c + 15]),
                       "=f"(y[c + 16]), "=f"(y[c + 17]), "=f"(y[c + 18]), "=f"(y[c + 19]), "=f"(y[c + 20]), "=f"(y[c + 21]), "=f"(y[c + 22]), "=f"(y[c + 23]),
                       "=f"(y[c + 24]), "=f"(y[c + 25]), "=f"(y[c + 26]), "=f"(y[c + 27]), "=f"(y[c + 28]), "=f"(y[c + 29]), "=f"(y[c + 30]), "=f"(y[c + 31])
                     : "r"(addr + c) : "memory");
}
__device__ __forceinline__ void wait_row(float (&y)[64])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 64; c++) asm volatile("" : "+f"(y[c]));      // nothing that uses them moves in front of the wait
}
__device__ __forceinline__ float row_max(const float (&y)[64])
{
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; i++) t[i] = max3(y[i], y[4 + i], y[8 + i]);
#pragma unroll
    for (int e = 12; e < 60; e += 8)
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = max3(t[i], y[e + i], y[e + 4 + i]);
    return max3(max3(t[0], t[1], y[60]), max3(t[2], t[3], y[61]), max3(y[62], y[63], y[63]));
}
// Every eight lanes transpose their eight pieces of 16 bytes: afterwards lane i of them holds piece i of all eight lanes.
__device__ __forceinline__ void transpose8(uint32_t (&v)[8][4])
{
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (int s = 4; s > 0; s >>= 1) {
        const bool upper = lane & s;
#pragma unroll
        for (int a = 0; a < 8; a++) {
            if (a & s) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? v[a][i] : v[a + s][i], s);
                if (upper) v[a][i] = got;
                else       v[a + s][i] = got;
            }
        }
    }
}
// All 128 threads of a tile's warps: whether any of them says so.
__device__ __forceinline__ bool any_of_tile(uint32_t tile, bool mine)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)mine), "r"(tile + 1) : "memory");
    return any != 0;
}
// Bits lo .. hi - 1 of the 32 that begin at `base`.
__device__ __forceinline__ uint32_t bits(int lo, int hi, int base)
{
    lo = max(lo - base, 0);
    hi = min(hi - base, 32);
    return hi <= lo ? 0u : (0xFFFFFFFFu >> (32 - hi + lo)) << lo;
}

// Key blocks of one tile of a segment: [g.begin, what is returned).  last_token: that of the tile's last row, were all tokens there.
__device__ __forceinline__ uint32_t tile_end(const Segment &g, uint32_t tile, uint32_t last_token)
{
    if (tile * kTile >= g.tokens * g.heads) return g.begin;
    const int last = min(g.pos0 + (int)min(last_token, g.tokens - 1), g.len - 1);
    return last < 0 ? g.begin : max(g.begin, min(g.end, (uint32_t)last / kKeys + 1));
}

}  // namespace mgq
