// Attention of few new tokens per sequence (single tokens, drafted ones) over a paged cache of f16 or bf16: reads every key and value
// once, so HBM bounds it, and all that matters is that loads never pause.
//
// A unit's pairs of token and head (16: heads of one key / value head share its keys) are the rows of m16n8k16 products.  The
// four warps of a CTA split the keys: each takes 16 of a block of 64, has a ring of its own for their keys and values, filled by
// TMA boxes of 16 keys by 64 elements that run across the borders of units, and an online softmax of its own; nothing in the loop waits for another warp.  At a
// unit's end the four sums are joined in shared memory.  Scores, maxima and sums are f32; a weight enters its product as the sum of two 16-bit values (the
// tensor cores have time for both): 2^-18 of it is lost for bf16, 2^-22 for f16, whose weights are 2^15 times as large as they should be, sums too, so that
// what both parts drop is below 2^-40 of the largest weight instead of 2^-25.  So the result is what is rounded.
// More pairs than 16 are units of their own that find the keys in L2: 32 sequences of up to 20 pairs (323 MB) take 69 us, with two blocks of rows per warp
// 103 us, on tcgen05 115 us; of 32 pairs each 118 and 107 us, four sequences of 32 pairs 29 and 40 us.  From 33 pairs on they are mgq_paged_prefill.cu's.
// With 16-byte cp.async instead of boxes a step took 627 instructions and 64 single tokens of the Qwen3-8B shape 242 us.
#include <cstdint>

#include "mgq_paged.cuh"
#include "mgq_tcgen05.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 128, kWarps = 4, kBlock = 64, kStep = 16;      // keys of a block, of a warp's step
constexpr int kRows = 16;                                               // pairs of token and head
constexpr int kChunk = 16, kPitch = kChunk + 2;                         // columns joined at a time
constexpr int kStages = 3;
// Blocks of keys that starting and ending a unit take as long as: 64 single tokens of the Qwen3-8B shape took 197, 188, 181, 175, 177 us with 0, 1, 2, 4, 7, 200
// shorter ones 172, 154, 141, 127, 129.
constexpr int kExtra = 4;
constexpr uint32_t kTile = kStep * 128;                                 // 16 keys by 64 elements, as one swizzled box lies in shared memory

// Stages of 16 keys and values fill the SM's shared memory, three per warp.
template <int D> __host__ __device__ constexpr int ctas_per_sm() { return D == 64 ? 3 : D == 128 ? 2 : 1; }
template <int D> __host__ __device__ constexpr uint32_t stage_bytes() { return 2 * D / 64 * kTile; }
template <int D> constexpr size_t smem_bytes() { return 1024 + (size_t)kWarps * kStages * stage_bytes<D>() + kWarps * kRows * kPitch * 4; }

__device__ unsigned int g_decode_error;

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
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y), l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
        high = *reinterpret_cast<const uint32_t *>(&h);
        low = *reinterpret_cast<const uint32_t *>(&l);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        high = *reinterpret_cast<const uint32_t *>(&h);
        const __nv_bfloat162 l = __floats2bfloat162_rn(x - __uint_as_float(high << 16), y - __uint_as_float(high & 0xFFFF0000u));
        low = *reinterpret_cast<const uint32_t *>(&l);
    }
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

template <typename T, int D>                             // D: head size rounded up to 64, 128 or 256
__global__ void __launch_bounds__(kThreads, ctas_per_sm<D>()) decode_kernel(const __grid_constant__ CacheMaps maps, const AttendArgs a)
{
    constexpr int NT = D / 8, KT = D / 16, PARTS = D / 64;
    constexpr float kUp = std::is_same<T, __half>::value ? 32768.f : 1.f;       // weights and their sums
    constexpr uint32_t kStage = stage_bytes<D>();
    using Way = Walk<kRows, kBlock, kExtra>;
    extern __shared__ uint8_t s_raw[];
    __shared__ unsigned long long s_walk[40];
    __shared__ __align__(8) unsigned long long s_full[kWarps][kStages];
    __shared__ Way s_way[kWarps];
    __shared__ Segment s_seg[kWarps][8];
    __shared__ uint32_t s_there[kWarps][kStages];
    __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
    __shared__ volatile int s_failed;
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = __shfl_sync(0xffffffffu, t >> 5, 0), d = a.d;
    uint8_t *s_mem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t ring = smem_u32(s_mem) + warp * (kStages * kStage);
    float *s_join = reinterpret_cast<float *>(s_mem + (size_t)kWarps * kStages * kStage);
    if (t == 0) {
        for (int i = 0; i < kWarps * kStages; i++) mbar_init(&s_full[i / kStages][i % kStages], 1);
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_launch_dependents();
    pdl_wait();
    {
        Way way;
        way.begin(a, blockIdx.x, gridDim.x, s_walk);
        if (lane == 0) s_way[warp] = way;
    }
    if (t == 0) clear_parts(a, blockIdx.x);
    __syncwarp();

    // ---- the producer's side of a warp: one step of 16 keys at a time, a segment without keys is a step without loads
    uint32_t p_seg = 0, p_block = 0, p_end = 0, p_slot = 0;      // segments begun, its next and last block, ring slot
    bool p_live = true;
    const uint32_t *p_table = nullptr;
    int p_len = 0, p_kv = 0;
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
                p_len = g.end <= g.begin ? 0 : g.len;
                p_kv = (int)g.kv;
                p_block = g.begin;
                p_end = max(g.end, g.begin + 1);
            }
        }
        if (p_live) {
            if (lane == 0) {
                const uint32_t key0 = p_block * kBlock + warp * kStep, within = (1u << a.page_shift) - 1;
                uint32_t there = 0;                                             // written before the arrival that publishes it
                if ((int)key0 < p_len) {
                    const uint32_t gone = a.pages << a.page_shift;              // a slot behind the last one: the box is filled with zeros
                    uint32_t page = p_table[key0 >> a.page_shift], slot[2];
                    const bool real = page < a.pages;
                    slot[0] = real ? (page << a.page_shift) + (key0 & within) : gone;
                    there = real ? 0xFFFFu : 0u;
                    if (a.page_shift == 3) {                                    // 16 keys of two pages
                        page = (int)key0 + 8 < p_len ? p_table[(key0 >> 3) + 1] : 0xFFFFFFFFu;
                        slot[1] = page < a.pages ? page << 3 : gone;
                        there = (real ? 0xFFu : 0u) | (page < a.pages ? 0xFF00u : 0u);
                    }
                    const int upto = p_len - (int)key0;
                    if (upto < kStep) there &= (1u << upto) - 1;
                    s_there[warp][p_slot] = there;
                    unsigned long long *bar = &s_full[warp][p_slot];
                    const uint32_t dst = ring + p_slot * kStage;
                    mbar_arrive_expect_tx(bar, kStage);
#pragma unroll
                    for (int c = 0; c < PARTS; c++) {
                        tma_load_3d(dst + c * kTile, &maps.k, c * 64, p_kv, (int)slot[0], bar);
                        tma_load_3d(dst + (PARTS + c) * kTile, &maps.v, c * 64, p_kv, (int)slot[0], bar);
                        if (a.page_shift == 3) {
                            tma_load_3d(dst + c * kTile + kTile / 2, &maps.k, c * 64, p_kv, (int)slot[1], bar);
                            tma_load_3d(dst + (PARTS + c) * kTile + kTile / 2, &maps.v, c * 64, p_kv, (int)slot[1], bar);
                        }
                    }
                } else {
                    s_there[warp][p_slot] = 0;
                    mbar_arrive(&s_full[warp][p_slot]);
                }
            }
            p_block++;
            p_slot = p_slot == kStages - 1 ? 0 : p_slot + 1;
        }
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; i++) produce();

    // ---- the consumer's side
    uint32_t c_seg = 0, slot = 0, parity = 0;
    bool ok = true;
    const uint32_t row = lane >> 2, quad = lane & 3u;
    // a lane's ldmatrix row in a box, and the 16-byte piece it starts with in each group of 16 elements (the swizzle XORs it with the row)
    const uint32_t krow = ((lane & 7u) + (lane >> 4) * 8) * 128, vrow = (lane & 15u) * 128;
    uint32_t kpiece[4], vpiece[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        kpiece[i] = krow + (((2 * i + ((lane >> 3) & 1u)) ^ (lane & 7u)) << 4);
        vpiece[i] = vrow + (((2 * i + (lane >> 4)) ^ (lane & 7u)) << 4);
    }
    while (c_seg < p_seg) {
        const Segment g = s_seg[warp][c_seg & 7u];
        c_seg++;
        const uint32_t pairs = g.tokens * g.heads;
        uint32_t q[KT][4];
        int pos[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = half * 8 + row, token = r / g.heads, head = r - token * g.heads;
            const bool live = r < pairs;
            pos[half] = live ? g.pos0 + (int)token : -1;
            const T *src = static_cast<const T *>(a.q) + (size_t)(g.row0 + (live ? token : 0)) * a.q_pitch + (size_t)(g.head0 + head) * d + 2 * quad;
#pragma unroll
            for (int k = 0; k < KT; k++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    q[k][half + 2 * j] = live && k * 16 + j * 8 + 2 * quad < d ? *reinterpret_cast<const uint32_t *>(src + k * 16 + j * 8) : 0u;
        }
        float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NT; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        const uint32_t blocks = max(g.end, g.begin + 1) - g.begin;
        const int last_pos = g.pos0 + (int)g.tokens - 1;
        for (uint32_t b = 0; b < blocks; b++) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(&s_full[warp][slot], parity, &s_failed, &g_decode_error)))) break;
            uint32_t there = s_there[warp][slot];
            const uint32_t kbase = ring + slot * kStage, vbase = kbase + PARTS * kTile;
            slot = slot == kStages - 1 ? 0 : slot + 1;
            parity ^= slot == 0;
            produce();
            const int key0 = (int)((g.begin + b) * kBlock + warp * kStep), upto = last_pos - key0 + 1, behind = a.window ? g.pos0 - (int)a.window + 1 - key0 : 0;
            if (upto < kStep) there &= upto > 0 ? (1u << upto) - 1 : 0u;
            if (behind > 0) there &= behind < kStep ? ~0u << behind : 0u;
            if (!there) continue;
            if (there != 0xFFFFu) {                      // values that no row sees, whatever the page holds there, become zeros
#pragma unroll
                for (uint32_t i = 0; i < PARTS * kTile / 512; i++)
                    if (!(there >> (i % 4 * 4 + lane / 8) & 1u))
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vbase + i * 512 + lane * 16), "r"(0) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // before the stage is filled again
                __syncwarp();
            }
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int k = 0; k < KT; k++) {
                uint32_t kf[4];
                ldmatrix4(kf, kbase + k / 4 * kTile + kpiece[k % 4]);
                mma<T>(s[0], q[k], kf[0], kf[1]);
                mma<T>(s[1], q[k], kf[2], kf[3]);
            }
            const bool whole = there == 0xFFFFu && key0 + kStep - 1 <= g.pos0 && (!a.window || key0 > last_pos - (int)a.window);
            bool hidden = false;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float top = m[half];
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = s[n][2 * half + e] * a.scale_log2;
                        if (!whole) {
                            const int key = key0 + n * 8 + 2 * (int)quad + e, p = pos[half];
                            const bool seen = key <= p && (there >> (n * 8 + 2 * quad + e) & 1u) && (!a.window || key > p - (int)a.window);
                            hidden |= !seen;
                            x = seen ? x : -INFINITY;
                        }
                        s[n][2 * half + e] = x;
                        top = fmaxf(top, x);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float base = top == -INFINITY ? 0.f : top;
                if (__any_sync(0xffffffffu, top > m[half])) {
                    const float keep = exp2_fast(m[half] - base);
                    l[half] *= keep;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        o[n][2 * half] *= keep;
                        o[n][2 * half + 1] *= keep;
                    }
                    m[half] = top;
                }
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float p = exp2_fast(s[n][2 * half + e] - base) * kUp;
                        s[n][2 * half + e] = p;
                        l[half] += p;
                    }
            }
            // where some row does not see a value that another one sees and that is infinite or NaN, its product with a weight of 0 must not be formed
            if (!whole && __any_sync(0xffffffffu, hidden)) {
                bool bad = false;
#pragma unroll
                for (uint32_t i = 0; i < PARTS * kTile / 512; i++) {
                    uint4 v;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(vbase + i * 512 + lane * 16) : "memory");
                    bad |= not_finite8<T>(v);
                }
                if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
                    for (uint32_t j = 0; j < kStep; j++) {
                        float p[2];
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const float even = j < 8 ? s[0][2 * half] : s[1][2 * half], oddv = j < 8 ? s[0][2 * half + 1] : s[1][2 * half + 1];
                            p[half] = __shfl_sync(0xffffffffu, j & 1u ? oddv : even, (lane & ~3u) | (j & 7u) >> 1);
                        }
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            uint32_t w;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(vbase + n / 8 * kTile + j * 128 + (((n % 8) ^ (j & 7u)) << 4) + quad * 4) : "memory");
                            const T *v = reinterpret_cast<const T *>(&w);
#pragma unroll
                            for (int half = 0; half < 2; half++)
#pragma unroll
                                for (int e = 0; e < 2; e++)
                                    o[n][2 * half + e] += p[half] != 0.f ? p[half] * to_f32(v[e]) : 0.f;
                        }
                    }
                    continue;
                }
            }
            uint32_t high[4], low[4];
#pragma unroll
            for (int i = 0; i < 4; i++) split_pair<T>(s[i >> 1][2 * (i & 1)], s[i >> 1][2 * (i & 1) + 1], high[i], low[i]);
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t vf[4];
                ldmatrix4_t(vf, vbase + n / 8 * kTile + vpiece[n / 2 % 4]);
                mma<T>(o[n], high, vf[0], vf[1]);
                mma<T>(o[n + 1], high, vf[2], vf[3]);
                mma<T>(o[n], low, vf[0], vf[1]);
                mma<T>(o[n + 1], low, vf[2], vf[3]);
            }
        }

        if (!ok) break;

        // ---- the four warps' sums
#pragma unroll
        for (int half = 0; half < 2; half++) {
            float sum = l[half];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (quad == 0) {
                s_m[warp][half * 8 + row] = m[half];
                s_l[warp][half * 8 + row] = sum;
            }
        }
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = half * 8 + row;
            const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            const float mine = s_l[warp][r] != 0.f ? exp2_fast(m[half] - top) : 0.f;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) o[n][2 * half + e] = mine != 0.f ? o[n][2 * half + e] * mine : 0.f;
        }
        const bool alone = g.first && g.last;
        float *part = a.parts + (size_t)part_index(blockIdx.x, g) * kRows * (d + 2);
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
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int half = 0; half < 2; half++)
                    *reinterpret_cast<float2 *>(s_join + (warp * kRows + half * 8 + row) * kPitch + n * 8 + 2 * quad) =
                        make_float2(o[2 * c + n][2 * half], o[2 * c + n][2 * half + 1]);
            __syncthreads();
            for (uint32_t i = t; i < pairs * (kChunk / 2); i += kThreads) {
                const uint32_t r = i / (kChunk / 2), col = i % (kChunk / 2) * 2;
                if (c * kChunk + col >= d) continue;
                float x = 0.f, y = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    const float2 v = *reinterpret_cast<const float2 *>(s_join + (w * kRows + r) * kPitch + col);
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
                    *reinterpret_cast<float2 *>(part + r * d + c * kChunk + col) = make_float2(x, y);
                }
            }
            __syncthreads();
        }
        if (!alone) {
            if (t < pairs) {
                float top;
                const float sum = total(t, top);
                part[kRows * d + 2 * t] = top;
                part[kRows * d + 2 * t + 1] = sum;
            }
            if (t == 0) name_part(a, blockIdx.x, g);
            __syncthreads();                             // before the next unit's maxima
        }
    }
    // given up: the copies in flight land before the CTA exits
    if (!ok && lane == 0)
        for (int i = 0; i < kStages - 1; i++) {
            for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&s_full[warp][slot], parity); w++) { }
            slot = slot == kStages - 1 ? 0 : slot + 1;
            parity ^= slot == 0;
        }
}

template <typename T, int D>
int launch_sized(const AttendArgs &a, const CacheMaps &maps, uint32_t pairs, cudaStream_t stream)
{
    constexpr uint32_t ctas = 148 * ctas_per_sm<D>();
    auto *kernel = decode_kernel<T, D>;
    if (int rc = allow_smem(kernel, smem_bytes<D>())) return rc;
    // left to itself the driver divides L1 and shared memory so that one CTA less fits for heads of 64: 128 single tokens of three such heads (0.4 GB)
    // took 118 us instead of 88
    MGQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (int rc = launch(kernel, dim3(ctas), dim3(kThreads), smem_bytes<D>(), stream, maps, a)) return rc;
    return launch_merge<T, kRows>(a, ctas, pairs, stream);
}

template <typename T>
int launch_typed(const AttendArgs &a, const CacheMaps &maps, uint32_t pairs, cudaStream_t stream)
{
    if (a.d <= 64) return launch_sized<T, 64>(a, maps, pairs, stream);
    if (a.d <= 128) return launch_sized<T, 128>(a, maps, pairs, stream);
    return launch_sized<T, 256>(a, maps, pairs, stream);
}

}  // namespace

bool decode_takes(const AttendArgs &a, int dtype)
{
    auto on = [](const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    return dtype != MGQ_FMT_F32 && a.d % 8 == 0 && on(a.k, 16) && on(a.v, 16) && on(a.q, 4) && on(a.out, 4) && a.q_pitch % 2 == 0 && a.out_pitch % 2 == 0 &&
           (unsigned long long)a.pages << a.page_shift < (1ull << 31);
}

uint32_t decode_ctas(uint32_t head_dim) { return 148 * (head_dim <= 64 ? ctas_per_sm<64>() : head_dim <= 128 ? ctas_per_sm<128>() : ctas_per_sm<256>()); }

int encode_caches(CacheMaps &maps, int dtype, const AttendArgs &a, uint32_t tokens)
{
    EncodeTiledFn encode = nullptr;
    if (int rc = encode_fn(encode)) return rc;
    const cuuint64_t dims[3] = {a.d, a.kv_heads, (cuuint64_t)a.pages << a.page_shift};
    const cuuint64_t strides[2] = {(cuuint64_t)a.d * 2, (cuuint64_t)a.kv_heads * a.d * 2};
    const cuuint32_t box[3] = {64, 1, tokens}, elem[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == MGQ_FMT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // a token's row of a head in whole pieces of 256 bytes, or what L2 fetches beyond it is another head's and may be gone by then: heads of 64 took 131 and
    // 118 us (128 single tokens, 0.4 GB), of 80 318 and 243 (64 single tokens, 1 GB), with 128 bytes 118 and 274
    const CUtensorMapL2promotion promotion = a.d % 128 == 0 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
    for (int i = 0; i < 2; i++) {
        const CUresult cr = encode(i ? &maps.v : &maps.k, type, 3, const_cast<void *>(i ? a.v : a.k), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) return fail(MGQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    }
    return MGQ_OK;
}

int launch_decode(const AttendArgs &a, int dtype, uint32_t pairs, cudaStream_t stream)
{
    CacheMaps maps;
    if (int rc = encode_caches(maps, dtype, a, a.page_shift == 3 ? 8 : kStep)) return rc;
    return dtype == MGQ_FMT_F16 ? launch_typed<__half>(a, maps, pairs, stream) : launch_typed<__nv_bfloat16>(a, maps, pairs, stream);
}

int paged_status()
{
    unsigned int err = 0;
    MGQ_CUDA(cudaMemcpyFromSymbol(&err, g_decode_error, sizeof err));
    if (!err) return prefill_status();
    const unsigned int zero = 0;
    MGQ_CUDA(cudaMemcpyToSymbol(g_decode_error, &zero, sizeof zero));
    return fail(MGQ_ERR_TIMEOUT, "a bounded wait inside the paged attention of few tokens ran out");
}

}  // namespace mgq
