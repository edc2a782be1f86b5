// Attention of few new tokens per sequence (single tokens, drafted ones) over a paged cache of f16 or bf16: reads every key and value
// once, so HBM bounds it, and all that matters is that loads never pause.
//
// A unit's pairs of token and head (16 or 32: heads of one key / value head share its keys) are the rows of m16n8k16 products.  The
// four warps of a CTA split the keys: each takes 16 of a block of 64, has a ring of its own for their keys and values, filled with
// 16-byte cp.async that run across the borders of units, and an online softmax of its own; nothing in the loop waits for another warp.  At a unit's end the
// four sums are joined in shared memory.  Scores, maxima and sums are f32; a weight enters its product as the sum of two 16-bit values (the tensor
// cores have time for both), so only the result is rounded.
// Rows in shared memory are padded by 16 bytes, which keeps ldmatrix free of bank conflicts for every head size.
#include <cstdint>

#include "mgq_paged.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 128, kWarps = 4, kBlock = 64, kStep = 16;      // keys of a block, of a warp's step
constexpr int kChunk = 16, kPitch = kChunk + 2;                         // columns joined at a time

template <int D> __host__ __device__ constexpr int ctas_per_sm() { return D == 64 ? 3 : D == 128 ? 2 : 1; }
template <int D> __host__ __device__ constexpr int row_bytes() { return D * 2 + 16; }
constexpr int kStages = 3;
template <int D, int MT> constexpr size_t smem_bytes() { return (size_t)kWarps * kStages * 2 * kStep * row_bytes<D>() + (size_t)kWarps * 16 * MT * kPitch * 4; }

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool real)
{
    const uint32_t bytes = real ? 16 : 0;                // the rest is zero-filled
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (sizeof(T) == sizeof(__half) && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (x, y) rounded to T, and what that leaves over.
template <typename T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t &high, uint32_t &low)
{
    const T hx = rounded<T>(x), hy = rounded<T>(y);
    const T lx = rounded<T>(x - to_f32(hx)), ly = rounded<T>(y - to_f32(hy));
    high = (uint32_t)*reinterpret_cast<const uint16_t *>(&hx) | (uint32_t)*reinterpret_cast<const uint16_t *>(&hy) << 16;
    low = (uint32_t)*reinterpret_cast<const uint16_t *>(&lx) | (uint32_t)*reinterpret_cast<const uint16_t *>(&ly) << 16;
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Whether one of 8 values of T is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite8(const uint4 &v)
{
    constexpr uint32_t mask = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; i++) bad |= (w[i] & mask) == mask || (w[i] >> 16 & mask) == mask;
    return bad;
}

template <typename T, int D, int MT>                     // D: head size rounded up to 64, 128 or 256; MT: blocks of 16 rows
__global__ void __launch_bounds__(kThreads, ctas_per_sm<D>()) decode_kernel(const AttendArgs a)
{
    constexpr int ROWS = 16 * MT, RB = row_bytes<D>(), NT = D / 8, KT = D / 16, CH = D / 8;     // CH: 16-byte pieces of a row
    using Way = Walk<ROWS, kBlock>;
    extern __shared__ __align__(16) uint8_t s_mem[];
    __shared__ unsigned long long s_walk[40];
    __shared__ Way s_way[kWarps];
    __shared__ Segment s_seg[kWarps][8];
    __shared__ uint32_t s_there[kWarps][kStages];
    __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, d = a.d;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_mem) + warp * (kStages * 2 * kStep * RB);
    float *s_join = reinterpret_cast<float *>(s_mem + (size_t)kWarps * kStages * 2 * kStep * RB);
    pdl_launch_dependents();
    pdl_wait();
    {
        Way way;
        way.begin(a, blockIdx.x, gridDim.x, 1, s_walk);
        if (lane == 0) s_way[warp] = way;
    }
    if (t == 0) clear_parts(a, blockIdx.x);
    __syncwarp();

    // ---- the producer's side of a warp: one step of 16 keys at a time, a segment without keys is a step without loads
    uint32_t p_seg = 0, p_block = 0, p_end = 0, p_slot = 0, p_steps = 0;      // segments begun, its next and last block, ring slot, steps issued
    bool p_live = true;
    const uint32_t *p_table = nullptr;
    int p_len = 0;
    const uint8_t *p_k = nullptr, *p_v = nullptr;
    const size_t row_stride = (size_t)a.kv_heads * d * sizeof(T);
    auto produce = [&]() {
        if (p_live && p_block >= p_end) {                // the next segment
            if (lane == 0) {
                Segment g;
                const bool more = s_way[warp].next(a, g);
                g.table = more ? g.table : nullptr;
                s_seg[warp][p_seg & 7u] = g;
            }
            __syncwarp();
            const Segment &g = s_seg[warp][p_seg & 7u];
            p_live = g.table != nullptr;
            if (p_live) {
                p_seg++;
                p_table = g.table;
                p_len = g.len;
                p_block = g.begin;
                p_end = max(g.end, g.begin + 1);
                const size_t head = ((size_t)g.kv * d + (lane % CH) * 8) * sizeof(T);
                p_k = static_cast<const uint8_t *>(a.k) + head;
                p_v = static_cast<const uint8_t *>(a.v) + head;
                if (g.end <= g.begin) p_len = 0;
            }
        }
        if (p_live) {
            const uint32_t key0 = p_block * kBlock + warp * kStep, slot = p_slot;
            uint32_t page[2];
            bool real[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {                // pages have at least 8 tokens
                const uint32_t key = key0 + 8 * h;
                page[h] = (int)key < p_len ? p_table[key >> a.page_shift] : 0xFFFFFFFFu;
                real[h] = page[h] < a.pages;
            }
            const uint32_t within = (1u << a.page_shift) - 1, dst = ring + slot * (2 * kStep * RB) + (lane % CH) * 16;
            const bool column = (lane % CH) * 8 < d;
#pragma unroll
            for (int i = 0; i < kStep * CH / 32; i++) {
                const uint32_t r = i * (32 / CH) + lane / CH, h = r / 8;
                const uint32_t pg = h ? page[1] : page[0];
                const bool ok = (h ? real[1] : real[0]) && (int)(key0 + r) < p_len && column;
                const size_t at = ok ? (((size_t)pg << a.page_shift) + ((key0 + r) & within)) * row_stride : 0;
                copy16(dst + r * RB, p_k + at, ok);
                copy16(dst + (kStep + r) * RB, p_v + at, ok);
            }
            if (lane == 0) {
                uint32_t there = (real[0] ? 0xFFu : 0u) | (real[1] ? 0xFF00u : 0u);
                const int upto = p_len - (int)key0;
                if (upto < kStep) there &= upto > 0 ? (1u << upto) - 1 : 0u;
                s_there[warp][slot] = there;
            }
            p_block++;
            p_steps++;
        }
        p_slot = p_slot == kStages - 1 ? 0 : p_slot + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) produce();

    // ---- the consumer's side
    uint32_t c_seg = 0, slot = 0;
    const uint32_t row = lane >> 2, quad = lane & 3u;
    while (c_seg < p_seg) {
        const Segment g = s_seg[warp][c_seg & 7u];
        c_seg++;
        const uint32_t pairs = g.tokens * g.heads;
        uint32_t q[MT][KT][4];
        int pos[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t r = mt * 16 + half * 8 + row, token = r / g.heads, head = r - token * g.heads;
                const bool live = r < pairs;
                pos[mt][half] = live ? g.pos0 + (int)token : -1;
                const T *src = static_cast<const T *>(a.q) + (size_t)(g.row0 + (live ? token : 0)) * a.q_pitch + (size_t)(g.head0 + head) * d + 2 * quad;
#pragma unroll
                for (int k = 0; k < KT; k++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        q[mt][k][half + 2 * j] = live && k * 16 + j * 8 + 2 * quad < d ? *reinterpret_cast<const uint32_t *>(src + k * 16 + j * 8) : 0u;
            }
        float o[MT][NT][4], m[MT][2], l[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
#pragma unroll
            for (int n = 0; n < NT; n++) o[mt][n][0] = o[mt][n][1] = o[mt][n][2] = o[mt][n][3] = 0.f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
        }
        const uint32_t blocks = max(g.end, g.begin + 1) - g.begin;
        const int last_pos = g.pos0 + (int)g.tokens - 1;
        for (uint32_t b = 0; b < blocks; b++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            const uint32_t there = s_there[warp][slot];
            const uint32_t kbase = ring + slot * (2 * kStep * RB), vbase = kbase + kStep * RB;
            slot = slot == kStages - 1 ? 0 : slot + 1;
            produce();
            if (!there) continue;
            const int key0 = (int)((g.begin + b) * kBlock + warp * kStep);
            float s[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++) s[mt][n][0] = s[mt][n][1] = s[mt][n][2] = s[mt][n][3] = 0.f;
            const uint32_t kaddr = kbase + ((lane & 7u) + (lane >> 4) * 8) * RB + ((lane >> 3) & 1u) * 16;
#pragma unroll
            for (int k = 0; k < KT; k++) {
                uint32_t kf[4];
                ldmatrix4(kf, kaddr + k * 32);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    mma<T>(s[mt][0], q[mt][k], kf[0], kf[1]);
                    mma<T>(s[mt][1], q[mt][k], kf[2], kf[3]);
                }
            }
            const bool whole = there == 0xFFFFu && key0 + kStep - 1 <= g.pos0 && (!a.window || key0 > last_pos - (int)a.window);
            bool hidden = false;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    float top = m[mt][half];
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x = s[mt][n][2 * half + e] * a.scale_log2;
                            if (!whole) {
                                const int key = key0 + n * 8 + 2 * (int)quad + e, p = pos[mt][half];
                                const bool seen = key <= p && (there >> (n * 8 + 2 * quad + e) & 1u) && (!a.window || key > p - (int)a.window);
                                hidden |= !seen && (there >> (n * 8 + 2 * quad + e) & 1u);
                                x = seen ? x : -INFINITY;
                            }
                            s[mt][n][2 * half + e] = x;
                            top = fmaxf(top, x);
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float base = top == -INFINITY ? 0.f : top;
                    if (__any_sync(0xffffffffu, top > m[mt][half])) {
                        const float keep = exp2_fast(m[mt][half] - base);
                        l[mt][half] *= keep;
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            o[mt][n][2 * half] *= keep;
                            o[mt][n][2 * half + 1] *= keep;
                        }
                        m[mt][half] = top;
                    }
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float p = exp2_fast(s[mt][n][2 * half + e] - base);
                            s[mt][n][2 * half + e] = p;
                            l[mt][half] += p;
                        }
                }
            // where some row does not see a value that is infinite or NaN, its product with a weight of 0 must not be formed
            if (!whole && __any_sync(0xffffffffu, hidden)) {
                bool bad = false;
#pragma unroll
                for (int i = 0; i < kStep * CH / 32; i++) {
                    uint4 v;
                    const uint32_t at = vbase + (i * (32 / CH) + lane / CH) * RB + (lane % CH) * 16;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
                    bad |= not_finite8<T>(v);
                }
                if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
                    for (uint32_t j = 0; j < kStep; j++) {
                        float p[MT][2];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int half = 0; half < 2; half++) {
                                const float even = j < 8 ? s[mt][0][2 * half] : s[mt][1][2 * half], oddv = j < 8 ? s[mt][0][2 * half + 1] : s[mt][1][2 * half + 1];
                                p[mt][half] = __shfl_sync(0xffffffffu, j & 1u ? oddv : even, (lane & ~3u) | (j & 7u) >> 1);
                            }
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            uint32_t w;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vbase + j * RB + n * 16 + quad * 4) : "memory");
                            const T *v = reinterpret_cast<const T *>(&w);
#pragma unroll
                            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                                for (int half = 0; half < 2; half++)
#pragma unroll
                                    for (int e = 0; e < 2; e++)
                                        o[mt][n][2 * half + e] += p[mt][half] != 0.f ? p[mt][half] * to_f32(v[e]) : 0.f;
                        }
                    }
                    continue;
                }
            }
            uint32_t high[MT][4], low[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++) split_pair<T>(s[mt][i >> 1][2 * (i & 1)], s[mt][i >> 1][2 * (i & 1) + 1], high[mt][i], low[mt][i]);
            const uint32_t vaddr = vbase + (lane & 15u) * RB + (lane >> 4) * 16;
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t vf[4];
                ldmatrix4_t(vf, vaddr + n * 16);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    mma<T>(o[mt][n], high[mt], vf[0], vf[1]);
                    mma<T>(o[mt][n + 1], high[mt], vf[2], vf[3]);
                    mma<T>(o[mt][n], low[mt], vf[0], vf[1]);
                    mma<T>(o[mt][n + 1], low[mt], vf[2], vf[3]);
                }
            }
        }

        // ---- the four warps' sums
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float sum = l[mt][half];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (quad == 0) {
                    s_m[warp][mt * 16 + half * 8 + row] = m[mt][half];
                    s_l[warp][mt * 16 + half * 8 + row] = sum;
                }
            }
        __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t r = mt * 16 + half * 8 + row;
                const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
                const float mine = s_l[warp][r] != 0.f ? exp2_fast(m[mt][half] - top) : 0.f;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) o[mt][n][2 * half + e] = mine != 0.f ? o[mt][n][2 * half + e] * mine : 0.f;
            }
        const bool alone = g.first && g.last;
        float *part = a.parts + (size_t)part_index(blockIdx.x, g) * ROWS * (d + 2);
        // the sums of a row's weights, needed where it is finished or stored
        auto total = [&](uint32_t r, float &top) {
            top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) sum += s_l[w][r] != 0.f ? s_l[w][r] * exp2_fast(s_m[w][r] - top) : 0.f;
            return sum;
        };
#pragma unroll
        for (int c = 0; c < D / kChunk; c++) {
            if (c * kChunk >= (int)d) break;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int half = 0; half < 2; half++)
                        *reinterpret_cast<float2 *>(s_join + (warp * ROWS + mt * 16 + half * 8 + row) * kPitch + n * 8 + 2 * quad) =
                            make_float2(o[mt][2 * c + n][2 * half], o[mt][2 * c + n][2 * half + 1]);
            __syncthreads();
            for (uint32_t i = t; i < pairs * (kChunk / 2); i += kThreads) {
                const uint32_t r = i / (kChunk / 2), col = i % (kChunk / 2) * 2;
                if (c * kChunk + col >= d) continue;
                float x = 0.f, y = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    const float2 v = *reinterpret_cast<const float2 *>(s_join + (w * ROWS + r) * kPitch + col);
                    x += v.x;
                    y += v.y;
                }
                if (alone) {
                    float top;
                    const float sum = total(r, top), scale = sum == 0.f ? 0.f : 1.f / sum;
                    const uint32_t token = r / g.heads, head = r - token * g.heads;
                    const T pair[2] = {rounded<T>(x * scale), rounded<T>(y * scale)};
                    *reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + (size_t)(g.row0 + token) * a.out_pitch + (size_t)(g.head0 + head) * d + c * kChunk + col) =
                        *reinterpret_cast<const uint32_t *>(pair);
                } else {
                    *reinterpret_cast<float2 *>(part + r * (d + 2) + c * kChunk + col) = make_float2(x, y);
                }
            }
            __syncthreads();
        }
        if (!alone) {
            if (t < pairs) {
                float top;
                const float sum = total(t, top);
                part[t * (d + 2) + d] = top;
                part[t * (d + 2) + d + 1] = sum;
            }
            if (t == 0) name_part(a, blockIdx.x, g);
            __syncthreads();                             // before the next unit's maxima
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, int D, int MT>
int launch_sized(const AttendArgs &a, cudaStream_t stream)
{
    constexpr uint32_t ctas = 148 * ctas_per_sm<D>();
    auto *kernel = decode_kernel<T, D, MT>;
    if (int rc = allow_smem(kernel, smem_bytes<D, MT>())) return rc;
    if (int rc = launch(kernel, dim3(ctas), dim3(kThreads), smem_bytes<D, MT>(), stream, a)) return rc;
    return launch(merge_kernel<T, 16 * MT>, dim3(ctas, 8), dim3(kMergeThreads), 0, stream, a, ctas);
}

template <typename T>
int launch_typed(const AttendArgs &a, uint32_t pairs, cudaStream_t stream)
{
    const bool two = pairs > 16;
    if (a.d <= 64) return two ? launch_sized<T, 64, 2>(a, stream) : launch_sized<T, 64, 1>(a, stream);
    if (a.d <= 128) return two ? launch_sized<T, 128, 2>(a, stream) : launch_sized<T, 128, 1>(a, stream);
    return launch_sized<T, 256, 1>(a, stream);
}

}  // namespace

bool decode_takes(const AttendArgs &a, int dtype)
{
    auto on = [](const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    return dtype != MGQ_FMT_F32 && a.d % 8 == 0 && on(a.k, 16) && on(a.v, 16) && on(a.q, 4) && on(a.out, 4) && a.q_pitch % 2 == 0 && a.out_pitch % 2 == 0;
}

uint32_t decode_ctas(uint32_t head_dim) { return 148 * (head_dim <= 64 ? ctas_per_sm<64>() : head_dim <= 128 ? ctas_per_sm<128>() : ctas_per_sm<256>()); }

int launch_decode(const AttendArgs &a, int dtype, uint32_t pairs, cudaStream_t stream)
{
    return dtype == MGQ_FMT_F16 ? launch_typed<__half>(a, pairs, stream) : launch_typed<__nv_bfloat16>(a, pairs, stream);
}

}  // namespace mgq
