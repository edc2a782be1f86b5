// Attention of many new tokens per sequence (portions of prompts, long drafts) over a paged cache of 8-bit codes, on tcgen05.
//
// As in mgq_paged_prefill.cu a unit is 256 pairs of token and query head of one key / value head, two tiles of 128 rows that share the codes of a block of 128
// keys; S = Q K^T and O += P V are products in 16 bits.  What is different: codes become operands on the way (four warps more), exactly, as f16 and bf16 hold
// all whole numbers up to 127; scales stay outside the products.  A block of 16 keys of a head has one scale each:
//   score    s * (scale * k_scale), a factor per 16 columns, which takes no more instructions than one for the row
//   weight   p * (v_scale / 2^e), rounded to f16, in which the values are operands whatever the queries' type: 2^-11 of a weight is lost at most, as in
//            mgq_paged_prefill.cu for f16.  e is the same for all rows; where a block's largest scale comes up to 2^e it rises and O is scaled.  The sums of weights are
//            without v_scale, in f32, and of weights before they are rounded: of rounded ones the results in f16 are off by 0.00024 instead of 0.00026 (2-norm; their own
//            rounding 0.00021), and 4 x 2048 tokens take 662 instead of 590 us.
//   warps 0-3, 4-7  softmax of tile 0 and 1, a row per thread
//   warp 8          codes: TMA boxes of a page's tokens (128 at most) by a head's dimensions, a lane each, into a ring
//   warp 9          issues the products
//   warp 10         finds the units, and loads their queries
//   warp 11         scales, two batches of four blocks, and which keys exist
//   warps 12-15     codes to operands in the 128-byte swizzle: eight lanes take two rows' opposite halves, so that neither loads nor stores meet in a bank
// Sums are kept relative to a maximum that may be 2^7 too low (2^15 where it has grown since): only where a row's maximum grows by more is O scaled.  Exponents are
// score * factor - m in one rounding; rows whose scores pass 2^20 (huge) round before they subtract, and their m is the maximum itself, so that its weight is that of a whole
// exponent however large m is: 2^8, added behind the subtraction, where m of other rows is the maximum less 8.
// 4 x 2048 tokens over up to 6144, 32 heads of 128 on 8: 589 us in bf16 (932 TFLOP/s of the 1678 that a library product reaches), 587 in f16; over 16 bits 482.  A tile's chain from scores to
// weights bounds it, beside shared memory, where codes are read and operands written, and the instruction cache: the twelve warps run four different programs, so the
// softmax reads its scores in short loops, twice (straight through with 208 registers 736 us, in 16 columns at a time 660), and what masks or huge scores need is apart.
// TMEM: S0, S1 (128 columns each, P in the first 64 of them), O0, O1.
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "mgq_paged_int8.cuh"
#include "mgq_paged_prefill.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 512;
constexpr int kExtra = 2;                                // blocks of keys that starting and ending a unit take as long as
constexpr float kHuge = 0x1p20f, kUnder = 8.f, kRoom = 15.f;          // m is 8 below a row's maximum when it is set, the maximum at most 15 above m
constexpr uint32_t kGroups = kKeys / 16, kBatch = 4;     // blocks of keys whose scales are fetched together
template <int D> __host__ __device__ constexpr uint32_t stage_bytes() { return D / 64 * kHalf; }                  // of operands
template <int D> __host__ __device__ constexpr uint32_t code_bytes() { return kKeys * D; }
template <int D> __host__ __device__ constexpr int stages() { return D == 64 ? 6 : 4; }
template <int D> __host__ __device__ constexpr int code_stages() { return D == 64 ? 4 : 2; }

__device__ unsigned int g_prefill8_error;

using Way = Walk<kPrefillRows, kKeys, kExtra>;
struct __align__(16) Shared {
    unsigned long long full[6], empty[6], code_full[4], code_empty[4], sc_full[2], sc_empty[2], q_full, q_empty, s_full[2], p_half[2], p_full[2], o_full[2];
    alignas(16) float factor[2][kBatch][kGroups], weight[2][kBatch][kGroups];          // of a block's groups of 16 keys
    float drop[2][kBatch], power[2][kBatch];             // what O is multiplied by at a block, and 2^e
    uint32_t there[2][kBatch][4];                        // keys that exist
    uint32_t odd[2][kBatch];                             // whether a scale is not finite
    Way way[3];                                          // of the producers of codes, queries, scales
    Segment kv_seg, sc_seg, next, seg[2];                // of those; of everybody else, two units in turn, no tokens behind the last
    int more;
    uint32_t last[4];                                    // whether a stage of codes says that there are no more
    uint32_t holes[2];                                   // whether the unit's keys have pages that do not exist
    uint32_t tmem;
    volatile int failed;
};
template <int D> constexpr size_t smem_bytes() { return (size_t)(2 + stages<D>()) * stage_bytes<D>() + code_stages<D>() * code_bytes<D>() + sizeof(Shared); }
static_assert(smem_bytes<128>() <= 227 * 1024 && smem_bytes<64>() <= 227 * 1024, "shared memory of an SM");

struct Maps {
    CUtensorMap k, v, q;
};

__device__ __forceinline__ pair_t pair_mul(pair_t x, pair_t y)
{
    pair_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
// The largest of 16; NaN if one is NaN.
__device__ __forceinline__ float max16(const float *y)
{
    const float a = max3(y[0], y[1], y[2]), b = max3(y[3], y[4], y[5]), c = max3(y[6], y[7], y[8]), d = max3(y[9], y[10], y[11]);
    return max3(max3(a, b, c), max3(d, y[12], y[13]), max3(y[14], y[15], y[15]));
}
// 32 columns of this lane's row; wait_quarter before they are used.
__device__ __forceinline__ void tmem_ld_quarter(uint32_t addr, float (&y)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]), "=f"(y[4]), "=f"(y[5]), "=f"(y[6]), "=f"(y[7]),
                   "=f"(y[8]), "=f"(y[9]), "=f"(y[10]), "=f"(y[11]), "=f"(y[12]), "=f"(y[13]), "=f"(y[14]), "=f"(y[15]),
                   "=f"(y[16]), "=f"(y[17]), "=f"(y[18]), "=f"(y[19]), "=f"(y[20]), "=f"(y[21]), "=f"(y[22]), "=f"(y[23]),
                   "=f"(y[24]), "=f"(y[25]), "=f"(y[26]), "=f"(y[27]), "=f"(y[28]), "=f"(y[29]), "=f"(y[30]), "=f"(y[31])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void wait_quarter(float (&y)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 32; c++) asm volatile("" : "+f"(y[c]));      // nothing that uses them moves in front of the wait
}
// Four codes as two pairs of f16 or bf16.  f16: 0x64 above a biased code reads 1024 + 128 + code.  bf16: 0x43 above seven bits reads 128 + them, and 128 or, with
// the sign, 256 is taken off.
template <typename T>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if constexpr (std::is_same<T, __half>::value) {
        const uint32_t off = 0x64806480u, u = w ^ 0x80808080u, x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 o = *reinterpret_cast<const __half2 *>(&off), a = __hsub2(*reinterpret_cast<const __half2 *>(&x), o), b = __hsub2(*reinterpret_cast<const __half2 *>(&y), o);
        lo = *reinterpret_cast<const uint32_t *>(&a);
        hi = *reinterpret_cast<const uint32_t *>(&b);
    } else {
        const uint32_t u = w & 0x7F7F7F7Fu, s = w & 0x80808080u;
        const uint32_t x = __byte_perm(u, 0x43434343u, 0x4140), y = __byte_perm(u, 0x43434343u, 0x4342), p = __byte_perm(s, 0x43434343u, 0x4140), q = __byte_perm(s, 0x43434343u, 0x4342);
        const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&x), *reinterpret_cast<const __nv_bfloat162 *>(&p));
        const __nv_bfloat162 b = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&y), *reinterpret_cast<const __nv_bfloat162 *>(&q));
        lo = *reinterpret_cast<const uint32_t *>(&a);
        hi = *reinterpret_cast<const uint32_t *>(&b);
    }
}
// 32 rows of a block's codes, [keys][D], to operands, halves of 64 dimensions in the 128-byte swizzle.
template <typename T, int D>
__device__ __forceinline__ void widen_rows(uint32_t codes, uint32_t operands, uint32_t row0)
{
    const uint32_t lane = threadIdx.x & 31u, group = lane >> 3, sub = lane >> 2 & 1u, j = lane & 3u;
    // eight lanes: rows r and r + 1, 64 dimensions each, of opposite halves where there are two
    const uint32_t half = D == 128 ? sub ^ (group & 1u) : 0u, first = row0 + sub + (D == 128 ? 2 * (group >> 1) : 2 * group);
    constexpr uint32_t kStep = D == 128 ? 4 : 8;
#pragma unroll 1
    for (uint32_t r = first; r < row0 + 32; r += kStep) {
        uint32_t w[4], o[8];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(codes + r * D + half * 64 + j * 16) : "memory");
#pragma unroll
        for (int i = 0; i < 4; i++) widen<T>(w[i], o[2 * i], o[2 * i + 1]);
        const uint32_t dst = operands + half * kHalf + r * 128, piece = (2 * j ^ (r & 7u)) << 4;
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + piece), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (piece ^ 16u)), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
    }
}
// 2^e for e from -126 to 127.
__device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <typename T, int D>                             // D: head size rounded up to 64 or 128
__global__ void __launch_bounds__(kThreads, 1) prefill8_kernel(const __grid_constant__ Maps maps, const Attend8Args a)
{
    constexpr int S = stages<D>(), C = code_stages<D>(), PARTS = D / 64;
    constexpr uint32_t kStage = stage_bytes<D>(), kCodes = code_bytes<D>();
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
    constexpr uint32_t kInstrS = (1u << 4) | kType | (kKeys >> 3 << 17) | (kTile >> 4 << 24);
    constexpr uint32_t kInstrO = (1u << 4) | (1u << 16) | ((uint32_t)D >> 3 << 17) | (kTile >> 4 << 24);                // f16
    extern __shared__ __align__(1024) uint8_t smem_raw[];                 // swizzled tiles lie on multiples of 1024
    uint8_t *s_q = smem_raw, *ring = s_q + 2 * kStage, *codes = ring + S * kStage;
    Shared &sh = *reinterpret_cast<Shared *>(codes + C * kCodes);
    if (smem_u32(smem_raw) % 1024 != 0) {                                 // cannot be with the alignment above
        if (threadIdx.x == 0) atomicExch(&g_prefill8_error, 1u);
        return;
    }
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;

    if (tid == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&sh.full[s], 4);                                    // the warps that widen codes
            mbar_init(&sh.empty[s], 2);                                   // either tile's warps
        }
        for (int s = 0; s < C; s++) {
            mbar_init(&sh.code_full[s], 1);
            mbar_init(&sh.code_empty[s], 4);
            sh.last[s] = 0;
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.sc_full[i], 1);
            mbar_init(&sh.sc_empty[i], 8);                                // the softmax warps
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_half[i], 4);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
        }
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 3);                                        // the issuer, both tiles' warps
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t slice = min(a.group, kPrefillRows), rows = kPrefillRows / slice * slice;       // heads of a unit, rows that TMA fills
    {
        Way way;
        way.begin(a, blockIdx.x, gridDim.x, reinterpret_cast<unsigned long long *>(s_q));
        if (lane == 0 && (warp == 8 || warp == 10 || warp == 11)) sh.way[warp == 8 ? 0 : warp - 9] = way;
    }
    for (uint32_t i = tid; i < (kPrefillRows - rows) * PARTS * 8; i += kThreads) {            // the others are zero for good
        const uint32_t part = i / ((kPrefillRows - rows) * 8), at = i - part * (kPrefillRows - rows) * 8;
        *reinterpret_cast<uint4 *>(s_q + part * 2 * kHalf + rows * 128 + at * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (tid == 0) clear_parts(a, blockIdx.x);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    // the tokens of the tiles' last rows
    const uint32_t last_token[2] = {(kTile - 1) / slice, (2 * kTile - 1) / slice};
    // Each lane by itself: false where the limit ran out, or another role has given up.
    auto lane_wait = [&](unsigned long long *bar, uint32_t parity) { return mbar_wait(bar, parity, &sh.failed, &g_prefill8_error); };
    auto wait = [&](unsigned long long *bar, uint32_t parity) {
        const bool done = lane_wait(bar, parity);
        __syncwarp();
        return done;
    };
    auto wait_all = [&](unsigned long long *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (warp >= 8) {
    if (warp == 8) {
        const uint32_t shift = a.page_shift, page_keys = 1u << shift, box = min(page_keys, kKeys), boxes = kKeys / box, gone = a.pages << shift;
        uint32_t slot = 0, round = 0;
        int armed = 0;
        bool ok = true;
        while (ok) {
            int more_units = 0;
            if (lane == 0) more_units = sh.way[0].next(a, sh.kv_seg);
            __syncwarp();
            if (!__shfl_sync(0xffffffffu, more_units, 0)) break;
            const Segment &g = sh.kv_seg;
            const int len = g.len, kv = (int)g.kv;
            const uint32_t *table = g.table;
            const uint32_t kb_begin = g.begin, kb_end = g.end;
            __syncwarp();                                // all lanes have read: behind a unit without blocks lane 0 writes the next one at once
            for (uint32_t kb = kb_begin; ok && kb < kb_end; kb++) {
                const uint32_t key = kb * kKeys + lane * box;             // lane = box of the block
                uint32_t y = gone;
                if (lane < boxes && (int)key < len) {
                    const uint32_t page = table[key >> shift];
                    if (page < a.pages) y = (page << shift) + (key & (page_keys - 1));
                }
                for (int what = 0; what < 2; what++) {
                    if (!(ok = wait_all(&sh.code_empty[slot], (round & 1u) ^ 1u))) break;
                    if (lane == 0) mbar_arrive_expect_tx(&sh.code_full[slot], kCodes);
                    __syncwarp();
                    if (lane < boxes) tma_load_3d(smem_u32(codes) + slot * kCodes + lane * box * D, what ? &maps.v : &maps.k, 0, kv, (int)y, &sh.code_full[slot]);
                    __syncwarp();
                    armed++;
                    if (++slot == C) { slot = 0; round++; }
                }
            }
        }
        if (ok && (ok = wait_all(&sh.code_empty[slot], (round & 1u) ^ 1u)) && lane == 0) {
            sh.last[slot] = 1;
            mbar_arrive(&sh.code_full[slot]);
        }
        // given up: the copies in flight land before the CTA exits
        if (!ok && lane == 0)
            for (int i = 0; i < min(armed, C); i++) {
                if (slot-- == 0) { slot = C - 1; round--; }
                for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&sh.code_full[slot], round & 1u); w++) { }
            }
    } else if (warp >= 12) {
        const uint32_t row0 = (warp - 12) * 32;
        uint32_t slot = 0, round = 0, from = 0, from_round = 0;           // of the operands, of the codes
        for (uint32_t what = 0;; what ^= 1u) {
            if (!wait_all(&sh.code_full[from], from_round & 1u) || sh.last[from]) break;
            if (!wait_all(&sh.empty[slot], (round & 1u) ^ 1u)) break;
            const uint32_t src = smem_u32(codes) + from * kCodes, dst = smem_u32(ring) + slot * kStage;
            if (std::is_same<T, __half>::value || what != 0) widen_rows<__half, D>(src, dst, row0);
            else                                             widen_rows<T, D>(src, dst, row0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the products read it, and the next codes come
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.full[slot]);
                mbar_arrive(&sh.code_empty[from]);
            }
            __syncwarp();
            if (++slot == S) { slot = 0; round++; }
            if (++from == C) { from = 0; from_round++; }
        }
    } else if (warp == 11) {
        // lane = block of the batch * 8 + group of 16 keys
        const uint32_t group = lane & 7u, shift = a.page_shift, within = (1u << shift) - 1;
        uint32_t batch = 0;
        bool ok = true;
        while (ok) {
            int more_units = 0;
            if (lane == 0) more_units = sh.way[2].next(a, sh.sc_seg);
            __syncwarp();
            if (!__shfl_sync(0xffffffffu, more_units, 0)) break;
            const int len = sh.sc_seg.len;
            const uint32_t *table = sh.sc_seg.table;
            const uint32_t kv = sh.sc_seg.kv, kb_begin = sh.sc_seg.begin, kb_end = sh.sc_seg.end;
            __syncwarp();
            int e2 = -1000;                              // weights are relative to 2^e2
            for (uint32_t kb0 = kb_begin; kb0 < kb_end; kb0 += kBatch, batch++) {
                const uint32_t b = batch & 1u, kb = kb0 + lane / 8, key = kb * kKeys + group * 16;
                float ks = 0.f, vs = 0.f;
                uint32_t there = 0;
                if (kb < kb_end && (int)key < len) {
                    const uint32_t page = table[key >> shift];
                    if (page < a.pages) {
                        const size_t at = (size_t)(((page << shift) + (key & within)) >> a.block_shift) * a.kv_heads + kv;
                        ks = a.k_scales[at];
                        vs = a.v_scales[at];
                        there = (1u << min(16, len - (int)key)) - 1;
                    }
                }
                // the scale's exponent: vs < 2^exponent; 129 for one that is not finite, which has no say
                int exponent = (int)(__float_as_uint(vs) >> 23 & 255u) - 126;
                int top = exponent < 129 ? exponent : -126;
#pragma unroll
                for (int o = 1; o < 8; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                int mine = e2, before = e2;
#pragma unroll
                for (uint32_t i = 0; i < kBatch; i++) {
                    const int t = __shfl_sync(0xffffffffu, top, 8 * i), was = e2;
                    if (t > e2 && kb0 + i < kb_end) e2 = min(t + 2, 127);
                    if (lane / 8 == i) {
                        mine = e2;
                        before = was;
                    }
                }
                const uint32_t odd = __ballot_sync(0xffffffffu, !(ks <= FLT_MAX && vs <= FLT_MAX));
                if (!(ok = wait_all(&sh.sc_empty[b], (batch >> 1 & 1u) ^ 1u))) break;
                if (kb < kb_end) {
                    const uint32_t i = lane / 8;
                    const float f = a.scale_log2 * fmaf(ks, 0.f, ks);      // NaN where the scale is infinite: its keys must not have scores of -infinity
                    sh.factor[b][i][group] = f < 1e-36f ? 1e-36f : f;      // a scale of 0 must not make -inf NaN
                    const int up = -mine;                // vs * 2^up in two steps, as 2^up alone may be out of range
                    sh.weight[b][i][group] = vs * power_of(max(min(up, 100), -126)) * power_of(max(up - 100, 0));
                    if (group == 0) {
                        sh.drop[b][i] = before == -1000 || before == mine ? 1.f : power_of(max(before - mine, -126));
                        sh.power[b][i] = power_of(mine);
                        sh.odd[b][i] = odd >> (8 * i) & 0xFFu;
                    }
                    reinterpret_cast<uint16_t *>(sh.there[b][i])[group] = (uint16_t)there;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.sc_full[b]);
            }
        }
    } else if (warp == 10) {
        uint32_t unit = 0;
        bool ok = true, more = true;
        for (; more; unit++) {
            if (lane == 0) {
                sh.next.tokens = 0;
                sh.more = sh.way[1].next(a, sh.next);
            }
            __syncwarp();
            more = sh.more != 0;
            bool holes = false;
            if (more && sh.next.end > sh.next.begin) {
                const uint32_t first = sh.next.begin * kKeys >> a.page_shift, last = (min(sh.next.end * kKeys, (uint32_t)sh.next.len) - 1) >> a.page_shift;
                for (uint32_t j = first + lane; j <= last; j += 32) holes |= sh.next.table[j] >= a.pages;
            }
            holes = __any_sync(0xffffffffu, holes);
            if (!(ok = wait_all(&sh.q_empty, (unit & 1u) ^ 1u))) break;
            if (lane == 0) {
                Segment &g = sh.seg[unit & 1u];
                g = sh.next;
                if (!more) g.tokens = 0;
                sh.holes[unit & 1u] = holes;
                if (more && g.end > g.begin) {
                    mbar_arrive_expect_tx(&sh.q_full, PARTS * rows * 128);
                    for (int c = 0; c < PARTS; c++) tma_load_3d(smem_u32(s_q) + c * 2 * kHalf, &maps.q, c * 64, (int)g.head0, (int)g.row0, &sh.q_full);
                } else {
                    mbar_arrive(&sh.q_full);
                }
            }
            __syncwarp();
        }
        if (!ok && lane == 0 && unit > 0)                // given up: the copy in flight lands before the CTA exits
            for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&sh.q_full, (unit - 1) & 1u); w++) { }
    } else if (warp == 9) {
        // One lane alone: a lane that ran along without issuing could fall two phases of a barrier behind, since nothing here or in the other roles waits for it, and
        // would then wait for a phase that is over.
        if (elect_one()) {
            const uint32_t q16 = smem_u32(s_q) >> 4, ring16 = smem_u32(ring) >> 4;
            uint32_t slot = 0, round = 0, p_seen = 0;                         // p_seen: parities of the two tiles in bits 0 and 1
            bool ok = true;
            auto advance = [&]() {
                if (++slot == S) { slot = 0; round++; }
            };
            auto scores = [&](uint32_t tile, uint32_t at) {
                const uint32_t q = q16 + tile * (kHalf / 16), k = ring16 + at * (kStage / 16);
                umma_step<false>(tmem + tile * 128, q, k, kInstrS);
#pragma unroll 1
                for (uint32_t i = 1; i < D / 16; i++) umma_step<true>(tmem + tile * 128, q + i / 4 * (2 * kHalf / 16) + i % 4 * 2, k + i / 4 * (kHalf / 16) + i % 4 * 2, kInstrS);
                umma_commit(&sh.s_full[tile]);
            };
            // 64 keys, 16 per product
            auto values = [&](uint32_t tile, uint32_t at, uint32_t part, bool first) {
                const uint32_t v = ring16 + at * (kStage / 16), o = tmem + 256 + tile * D, p = tmem + tile * 128;
#pragma unroll 1
                for (uint32_t i = 0; i < kKeys / 32; i++) {
                    const uint32_t step = part * 4 + i;
                    umma_f16_ts_mn(o, p + step * 8, v + step * (2048 / 16), kHalf / 16, kInstrO, !first || i > 0 || part > 0);
                }
            };
            for (uint32_t unit = 0;; unit++) {
                if (!(ok = lane_wait(&sh.q_full, unit & 1u))) break;
                const Segment &g = sh.seg[unit & 1u];
                if (g.tokens == 0) break;
                const uint32_t begin = g.begin, end = g.end, stop[2] = {tile_end(g, 0, last_token[0]), tile_end(g, 1, last_token[1])};
                if (end <= begin) {
                    mbar_arrive(&sh.q_empty);
                    continue;
                }
                // Each wait stands where products are under way: for the next keys behind the first half of tile 0's values, for the next values behind that of
                // tile 1's.  The stages are given back by the softmax warps, which learn from the scores' commits that their products are done.
                if (!(ok = lane_wait(&sh.full[slot], round & 1u))) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t tile = 0; tile < 2; tile++)
                    if (stop[tile] > begin) scores(tile, slot);
                if (begin + 1 == end) umma_commit(&sh.q_empty);
                advance();
                if (!(ok = lane_wait(&sh.full[slot], round & 1u))) break;
                for (uint32_t kb = begin; kb < end; kb++) {
                    const uint32_t v_slot = slot;
                    advance();
                    const uint32_t k_slot = slot, k_round = round;
                    const bool more = kb + 1 < end;
                    if (more) advance();                     // to the next values
#pragma unroll 1
                    for (uint32_t tile = 0; tile < 2; tile++) {
                        const bool values_now = (tile ? stop[1] : stop[0]) > kb;
                        if (values_now) {
                            if (!(ok = lane_wait(&sh.p_half[tile], p_seen >> tile & 1u))) break;
                            tc_fence_after();
                            values(tile, v_slot, 0, kb == begin);
                        }
                        if (more && !(ok = lane_wait(&sh.full[tile ? slot : k_slot], (tile ? round : k_round) & 1u))) break;
                        if (values_now) {
                            if (!(ok = lane_wait(&sh.p_full[tile], p_seen >> tile & 1u))) break;
                            p_seen ^= 1u << tile;
                            tc_fence_after();
                            values(tile, v_slot, 1, false);
                            if (kb + 1 == (tile ? stop[1] : stop[0])) umma_commit(&sh.o_full[tile]);
                        }
                        if ((tile ? stop[1] : stop[0]) > kb + 1) scores(tile, k_slot);
                    }
                    if (!ok) break;
                    if (kb + 2 == end) umma_commit(&sh.q_empty);    // no more scores of this unit
                }
                if (!ok) break;
            }
        }
        __syncwarp();
    }
    } else {
        const uint32_t tile = warp >> 2, quad = warp & 3u, r_tile = quad * 32 + lane, row = tile * kTile + r_tile, d = a.d;
        const uint32_t lanes = (quad * 32u) << 16, s_at = tmem + tile * 128 + lanes, o_at = tmem + 256 + tile * D + lanes;
        const uint32_t token = row / slice, head = row - token * slice, first_token = tile * kTile / slice;     // of this row, of the tile's first
        uint32_t slot = 0, round = 0, batch = 0;         // of the ring, as the producer counts; of the scales
        uint32_t s_seen = 0, o_seen = 0;
        // Where a wait runs out the tile's warps run on without waiting, and leave together at the next unit.
        for (uint32_t unit = 0;; unit++) {
            const bool there_is = wait(&sh.q_full, unit & 1u);
            const Segment &g = sh.seg[unit & 1u];
            if (any_of_tile(tile, !there_is)) break;
            if (g.tokens == 0) break;
            const uint32_t begin = g.begin, end = g.end, stop = tile_end(g, tile, last_token[tile]), pairs = g.tokens * g.heads;
            if (stop <= begin && r_tile == 0) mbar_arrive(&sh.q_empty);           // behind the meeting of this tile's warps
            const int first_pos = g.pos0 + (int)first_token, len = g.len;
            const int last_pos = g.pos0 + (int)min(last_token[tile], g.tokens - 1), window = (int)a.window;
            const int pos = row < pairs ? g.pos0 + (int)token : -1;
            const bool holes = sh.holes[unit & 1u] != 0;
            float m = -INFINITY, l = 0.f, power = 1.f;
            bool huge = false;
            uint32_t v_before = 0;
            bool finished = stop <= begin;               // the last product is done, its values' stage given back
            auto finish = [&]() {
                if (finished) return;
                finished = true;
                wait(&sh.o_full[tile], o_seen & 1u);
                o_seen++;
                tc_fence_after();
                if (r_tile == 0) mbar_arrive(&sh.empty[v_before]);
            };
            for (uint32_t kb = begin; kb < end; kb++) {
                const uint32_t k_slot = slot, k_round = round;
                if (++slot == S) { slot = 0; round++; }
                const uint32_t v_slot = slot, v_round = round;
                if (++slot == S) { slot = 0; round++; }
                const uint32_t in_batch = (kb - begin) % kBatch, sb = batch & 1u;
                const bool batch_ends = in_batch == kBatch - 1 || kb + 1 == end;
                if (in_batch == 0) wait(&sh.sc_full[sb], batch >> 1 & 1u);
                auto leave_batch = [&]() {               // all of this warp's reads of the block's scales are done
                    if (!batch_ends) return;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.sc_empty[sb]);
                    batch++;
                };
                if (kb >= stop) {
                    finish();
                    // Nothing for this tile: it gives the stages back as soon as they are filled, not before.  Its first warp alone, lanes together: once the stage is
                    // given back it may be filled again, and another warp that has not looked yet would wait for a phase that is over.
                    if (quad == 0) {
                        wait(&sh.full[k_slot], k_round & 1u);
                        if (lane == 0) mbar_arrive(&sh.empty[k_slot]);
                        wait(&sh.full[v_slot], v_round & 1u);
                        if (lane == 0) mbar_arrive(&sh.empty[v_slot]);
                    }
                    leave_batch();
                    continue;
                }
                wait(&sh.s_full[tile], s_seen & 1u);
                s_seen++;
                tc_fence_after();
                if (r_tile == 0) {                       // these scores are done, and the product before them; with the last ones the queries
                    if (kb + 1 == stop) mbar_arrive(&sh.q_empty);
                    mbar_arrive(&sh.empty[k_slot]);
                    if (kb != begin) mbar_arrive(&sh.empty[v_before]);
                }
                v_before = v_slot;
                const int key0 = (int)(kb * kKeys);
                const bool every = !holes && key0 + (int)kKeys <= len;
                const bool plain = every && key0 + (int)kKeys - 1 <= first_pos && !(window && key0 <= last_pos - window);      // nothing is masked
                const float *factors = sh.factor[sb][in_batch], *by = sh.weight[sb][in_batch];
                const float drop = sh.drop[sb][in_batch];
                power = sh.power[sb][in_batch];
                auto signal = [&](unsigned long long *bar) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                // Both passes over the scores stand twice in the code: for blocks where something is masked (or huge), and for those where nothing is.  In one
                // loop the first kind's instructions lie between the second's, and what runs on the SM at the same time no longer fits its instruction cache.
                // Of 32 keys: those that the row sees, the factors or weights of their two groups, and scores without what it does not see.  Where a scale is not finite,
                // one that this row does not see must have no say.
                const bool odd = !plain && sh.odd[sb][in_batch];
                auto sees = [&](int w) { return sh.there[sb][in_batch][w] & bits(window ? pos - window + 1 : 0, pos + 1, key0 + 32 * w); };
                auto of_groups = [&](auto simple, const float *p, int w, float otherwise) {
                    float2 v = *reinterpret_cast<const float2 *>(p + 2 * w);
                    if (!decltype(simple)::value && odd) {
                        const uint32_t seen = sees(w);
                        if (!(seen & 0xFFFFu)) v.x = otherwise;
                        if (!(seen >> 16)) v.y = otherwise;
                    }
                    return v;
                };
                auto mask = [&](auto simple, float (&s)[32], int w) {
                    if (decltype(simple)::value || plain) return;
                    const uint32_t seen = sees(w);
#pragma unroll
                    for (int e = 0; e < 32; e++) s[e] = seen >> e & 1u ? s[e] : -INFINITY;
                    __syncwarp();
                };
                // Scores are read twice, for the maximum and for the weights, in loops that are short in the code; the next 32 are on their way as soon as these are used.
                float s[32], top = -INFINITY;
                tmem_ld_quarter(s_at, s);
                auto find_top = [&](auto simple) {
#pragma unroll 1
                    for (int w = 0; w < 4; w++) {
                        wait_quarter(s);
                        mask(simple, s, w);
                        const float2 f = of_groups(simple, factors, w, 1.f);
                        const float a0 = max16(s), a1 = max16(s + 16);
                        tmem_ld_quarter(s_at + (32 * w + 32) % 128, s);      // in the end the first ones again
                        top = max3(top, a0 * f.x, a1 * f.y);
                    }
                };
                if (plain) find_top(std::true_type());
                else       find_top(std::false_type());
                // Nothing to do where the maximum stays at or below m + kRoom (finite behind the first block); -inf and NaN come here, too.
                const float room = m + (huge ? kRoom - kUnder : kRoom);
                const bool calm = top <= room && top >= -FLT_MAX && drop == 1.f;
                if (__any_sync(0xffffffffu, !calm)) {
                    const bool up = !(top <= room) && top > -INFINITY;                      // also where m is still -inf
                    const bool was = huge;
                    huge |= up && fabsf(top) > kHuge;
                    const float under = up ? (huge ? top : top - kUnder) : m, keep = up ? exp2_fast(m - under + (huge && !was ? kUnder : 0.f)) : 1.f;
                    l *= keep;
                    m = under;
                    if (kb != begin && __any_sync(0xffffffffu, up || drop != 1.f)) {
                        const float both = keep * drop;
#pragma unroll 1
                        for (uint32_t c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_at + c, o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * both);
                            tmem_st16(o_at + c, o);
                        }
                    }
                }
                const bool scaled = __any_sync(0xffffffffu, huge);
                const float base = m == -INFINITY ? 0.f : -m;
                const pair_t bases = pair_of(base, base);
                pair_t sum[2] = {0, 0};
                // Exponentials, sums, P, which takes the place of scores that have been read.
                auto all_weights = [&](auto simple) {
#pragma unroll 1
                    for (int w = 0; w < 4; w++) {
                        wait_quarter(s);
                        mask(simple, s, w);
                        float2 f = of_groups(simple, factors, w, 1.f);
                        const float2 v = of_groups(simple, by, w, 0.f);
                        pair_t minus = bases;
                        if (!decltype(simple)::value && scaled) {            // the products with the factors are rounded first, so that the maximum's weight is 2^8 however large m is
                            const float lift = huge ? kUnder : 0.f;
#pragma unroll
                            for (int e = 0; e < 32; e++) s[e] = __fadd_rn(__fadd_rn(__fmul_rn(s[e], e < 16 ? f.x : f.y), base), lift);
                            f = make_float2(1.f, 1.f);
                            minus = 0;
                        }
                        pair_t e[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) e[i] = pair_fma(pair_of(s[2 * i], s[2 * i + 1]), i < 8 ? pair_of(f.x, f.x) : pair_of(f.y, f.y), minus);
                        if (w < 3) tmem_ld_quarter(s_at + 32 * w + 32, s);
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            float a0, a1;
                            parts_of(e[i], a0, a1);
                            const pair_t both = pair_of(exp2_fast(a0), exp2_fast(a1));
                            sum[i & 1] = pair_add(sum[i & 1], both);
                            parts_of(pair_mul(both, i < 8 ? pair_of(v.x, v.x) : pair_of(v.y, v.y)), a0, a1);
                            p[i] = pack<__half>(a0, a1);
                        }
                        tmem_st16(s_at + 16 * w, p);
                        if (w == 1) signal(&sh.p_half[tile]);
                    }
                };
                if (plain && !scaled) all_weights(std::true_type());
                else                  all_weights(std::false_type());
                float a0, a1;
                parts_of(pair_add(sum[0], sum[1]), a0, a1);
                l += a0 + a1;
                leave_batch();
                signal(&sh.p_full[tile]);
            }
            finish();
            if (huge) {                                  // sums and O are relative to m again, as parts are joined
                l *= 1.f / (1 << (int)kUnder);
                power *= 1.f / (1 << (int)kUnder);
            }
            if (tile * kTile < pairs) {
                // 128 bytes of eight rows at a time, turned so that a store covers whole lines of few rows
                const bool alone = g.first && g.last;
                const unsigned long long at = (unsigned long long)(g.row0 + token) * a.out_pitch + (unsigned long long)(g.head0 + head) * d;
                float *part = a.parts + (size_t)part_index(blockIdx.x, g) * kPrefillRows * (d + 2);
                const float inv = alone ? (l == 0.f ? 0.f : power / l) : power;
                const uint32_t first_row = tile * kTile + quad * 32 + (lane & 24u), piece = lane & 7u;
#pragma unroll 1
                for (uint32_t c = 0; c < D; c += 32) {
                    float o[32];
                    auto columns = [&](uint32_t c) {
                        tmem_ld32(o_at + c, o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = stop > begin && l != 0.f ? o[e] * inv : 0.f;
                    };
                    columns(c);
                    if (alone) {                         // 64 bytes of a row, two such steps make a line
                        uint32_t v[8][4];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e / 4][e % 4] = pack<T>(o[2 * e], o[2 * e + 1]);
                        columns(min(c + 32, (uint32_t)D - 32));
#pragma unroll
                        for (int e = 0; e < 16; e++) v[4 + e / 4][e % 4] = pack<T>(o[2 * e], o[2 * e + 1]);
                        transpose8(v);
#pragma unroll
                        for (int r = 0; r < 8; r++) {
                            const unsigned long long there = __shfl_sync(0xffffffffu, at, (lane & 24u) + r);
                            if (first_row + r < pairs && c + 8 * piece < d)
                                *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + there + c + 8 * piece) = make_uint4(v[r][0], v[r][1], v[r][2], v[r][3]);
                        }
                        c += 32;
                    } else {
                        uint32_t v[8][4];
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e / 4][e % 4] = __float_as_uint(o[e]);
                        transpose8(v);
#pragma unroll
                        for (int r = 0; r < 8; r++)
                            if (first_row + r < pairs && c + 4 * piece < d)
                                *reinterpret_cast<uint4 *>(part + (first_row + r) * d + c + 4 * piece) = make_uint4(v[r][0], v[r][1], v[r][2], v[r][3]);
                    }
                    __syncwarp();                        // the next columns are read by the whole warp
                }
                if (!alone && row < pairs) *reinterpret_cast<float2 *>(part + kPrefillRows * d + 2 * row) = make_float2(m, l);
                if (!alone && tid == 0) name_part(a, blockIdx.x, g);
            }
            tc_fence_before();
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

template <typename T, int D>
int launch_sized(const Attend8Args &a, const Maps &maps, cudaStream_t stream)
{
    auto *kernel = prefill8_kernel<T, D>;
    if (int rc = allow_smem(kernel, smem_bytes<D>())) return rc;
    if (int rc = launch(kernel, dim3(kPrefillCtas), dim3(kThreads), smem_bytes<D>(), stream, maps, a)) return rc;
    return launch_merge<T, (int)kPrefillRows>(a, kPrefillCtas, kPrefillRows, stream);
}

// Codes: {head_dim, kv_heads, pages * page_size}, boxes of a head's dimensions (64 or 128) by the tokens of a page, as they lie.  What lies outside reads as zero.
// Queries: {head_dim, heads, rows}, boxes of 64 elements by the heads of a key / value head by the tokens of a unit: the pairs of token and head are the rows.
int encode_maps(Maps &maps, int dtype, const Attend8Args &a)
{
    EncodeTiledFn encode = nullptr;
    if (int rc = encode_fn(encode)) return rc;
    const cuuint32_t elem[3] = {1, 1, 1};
    for (int i = 0; i < 2; i++) {
        const cuuint64_t dims[3] = {a.d, a.kv_heads, (cuuint64_t)a.pages << a.page_shift}, strides[2] = {a.d, (cuuint64_t)a.kv_heads * a.d};
        const cuuint32_t box[3] = {a.d <= 64 ? 64u : 128u, 1, min(1u << a.page_shift, kKeys)};
        const CUresult cr = encode(i ? &maps.v : &maps.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(i ? a.v : a.k), dims, strides, box, elem,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) return fail(MGQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
    }
    const cuuint64_t dims[3] = {a.d, (cuuint64_t)a.kv_heads * a.group, a.rows}, strides[2] = {(cuuint64_t)a.d * 2, (cuuint64_t)a.q_pitch * 2};
    const cuuint32_t box[3] = {64, a.group, kPrefillRows / a.group};
    const CUresult cr = encode(&maps.q, dtype == MGQ_FMT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(a.q), dims, strides, box,
                               elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? MGQ_OK : fail(MGQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
}

}  // namespace

bool prefill8_takes(const Attend8Args &a)
{
    auto on = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    // scores are masked and compared before they are scaled: a scale of 0 would make -inf NaN, a negative one turn the order around
    return a.d <= 128 && a.group <= kPrefillRows && a.scale_log2 >= 1e-30f && a.scale_log2 <= 1e30f && on(a.q) && on(a.out) && a.q_pitch % 8 == 0 && a.out_pitch % 8 == 0;
}

int launch_prefill8(const Attend8Args &a, int dtype, cudaStream_t stream)
{
    Maps maps;
    if (int rc = encode_maps(maps, dtype, a)) return rc;
    if (dtype == MGQ_FMT_F16) return a.d <= 64 ? launch_sized<__half, 64>(a, maps, stream) : launch_sized<__half, 128>(a, maps, stream);
    return a.d <= 64 ? launch_sized<__nv_bfloat16, 64>(a, maps, stream) : launch_sized<__nv_bfloat16, 128>(a, maps, stream);
}

int prefill8_status()
{
    unsigned int err = 0;
    MGQ_CUDA(cudaMemcpyFromSymbol(&err, g_prefill8_error, sizeof err));
    if (!err) return int8_status();
    const unsigned int zero = 0;
    MGQ_CUDA(cudaMemcpyToSymbol(g_prefill8_error, &zero, sizeof zero));
    return fail(MGQ_ERR_TIMEOUT, "a bounded wait inside the attention of many tokens over 8-bit codes ran out");
}

}  // namespace mgq
