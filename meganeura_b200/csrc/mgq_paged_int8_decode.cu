// Attention of few new tokens per sequence (single tokens, drafted ones) over a paged cache of 8-bit codes: reads every code once, so HBM bounds it, and what
// the codes need before they can be multiplied has to fit beside that.
//
// A unit's pairs of token and head (8 or 16: heads of one key / value head share its keys) are the columns of m16n8k16 products in f16 whose rows are 16 keys of a
// head (scores) or 16 of its dimensions (results): codes are the left operand of both, eight pairs cost no more than they are, and the accumulators of eight
// pairs of 128 are 32 registers.  The order of k inside a product, and of the results' rows, is free, so a lane takes 16 consecutive codes of a key with one
// load.  A biased byte code + 128 with a zero above it is an f16, subnormal and exact: (code + 128) 2^-24.  From the scores the bias is taken off by where their sums
// begin, at -128 2^-24 times the sum of q; from values by a subtraction per pair of them, so that no sum ever grows with the bias.  (The same for keys would
// cost a fourteenth of the instructions, which are what this kernel has to save.)
// Scores: q enters as f16, times a power of two that bf16 rows need to fit its range; a row's is undone in f32 with the block's scale.  Weights: times the
// block's scale, as the sum of two f16, 2^-22 of each is lost at most, so that only the result is rounded (2-norm against 64 bits: f16 0.00020, bf16 0.0016, as the rounded
// exact result).  One f16 alone, 2^-11, left 0.00026 to 0.00031 in f16; with a product of the bias in the place of the second part's and of the subtraction 64 single tokens of the
// Qwen3-8B shape took as long and 32 times 1 to 5 3 % less.  Weights are relative to a maximum that may be 2^8 too low (kRoom), and to a power of two of the blocks' scales (`e2`)
// which rises when a larger scale comes; sums of weights are f32.  Weights that move from the scores' layout to the right operand's are transposed 8 x 8 at a time (movmatrix).
// Four warps of a CTA split a unit, and each takes 32 keys of a block at a time, from a ring that a fifth warp fills across the borders of units: a lane brings 16
// keys or values with a TMA box and their scales with 4-byte copies.  (Where every warp filled its own, that was a quarter of its instructions: 64 single
// tokens of the Qwen3-8B shape took 117 us.)  At a unit's end the sums are joined in shared memory.
// Heads of up to 128 in pairs (H = 2): a token's codes of one head are 128 bytes or less, a kilobyte apart, and HBM gives 5.0 TB/s of such pieces (107 us, as long without
// any arithmetic).  So where it can be a unit is two neighbouring key / value heads, whose codes come in one box, and two warps work for either: 64 single tokens over
// up to 8100 take 97 us, 5.5 TB/s with the join of the parts (5 us), 94 without any arithmetic.  32 times 1 to 5 tokens of four heads each over up to 4000 take 58 to 62:
// above 16 pairs two units read the same keys, and two warps of a scheduler do not hide each other's chains.
#include <cstdint>

#include "mgq_paged_int8.cuh"
#include "mgq_tcgen05.cuh"

namespace mgq {
namespace {

constexpr int kWarps = 4, kStep = 32;             // keys of a warp's step
constexpr int kGroups = kStep / 16;                      // 16 keys lie in one page and one block
constexpr int kExtra = 2;                                // blocks of keys that starting and ending a unit take as long as
// Cost of a piece, blocks of keys and kExtra for a unit: with less the join of the parts takes longer than the blocks.  1, 2, 3, 4: one token over 8000 cached 25.7, 23.1, 21.8, 19.9 us,
// two over 3000 19.0, 16.3, 17.4, 17.1, four of nine heads of 64 over up to 500 9.5, 9.8, 10.5, 11.7.
constexpr uint32_t kLeastBlocks = 3;
// Which kernels serve more than kDecode8Pairs pairs.  The one for many tokens takes 20 us for the least, this one as long as it reads and joins: it takes everything where the
// units, by what the tables let them read, are little work (kLittle: units of 16 pairs times keys, kPlace more for each), and no sequence has so many units that finding one's place
// among them takes long (kMostUnits).  32 heads on 8 of 128, all here and all there, us: 9 tokens over 300 19.7 and 23.3, 40 over 1500 26.2 and 26.0, 12 times 9 over 1500 45.8 and 44.5, 12
// times 40 over 300 52.2 and 32.6, 200 over 1500 62.1 and 34.4; 8 on 1, 500 over none 41.0 and 26.8.  The tables' width is all that is known here of the lengths: with tables of 131072
// tokens the first and the fourth of these take both kernels, 30 and 39.
// Else each kernel takes its sequences, but where most have many tokens and none can be long the other one takes all, as a launch of this one costs more than it saves (12 times
// 40 over 300 39.3 and 32.5, three single tokens over 8000 beside 128 85.7 and 67.9); single tokens over long sequences are slow there (three over 32000 beside 512 103 and 126).
constexpr unsigned long long kLittle = 175000, kPlace = 100, kShort = 32768;
constexpr uint32_t kMostUnits = 64, kManyRows = 32;
constexpr float kRoom = 8.f;
constexpr int kUp = 7;                                   // weights are 2^kUp times what they should be: 2^15 at most, and all of their bits down to 2^-21 of the largest

template <int D> __host__ __device__ constexpr uint32_t row_bytes() { return D < 128 ? D : 128; }                  // of a box: 64 or 128, in the swizzle of that size
template <int D> __host__ __device__ constexpr uint32_t box_bytes() { return 16 * row_bytes<D>(); }
template <int D> __host__ __device__ constexpr uint32_t group_bytes() { return D / row_bytes<D>() * box_bytes<D>(); }
template <int D> __host__ __device__ constexpr uint32_t stage_bytes() { return 2 * kGroups * group_bytes<D>(); }   // keys of all groups, then values
template <int D> __host__ __device__ constexpr int ctas_per_sm() { return D == 64 ? 3 : D == 128 ? 2 : 1; }
constexpr int kStages = 3;
// Heads of 128 by 16 pairs need more registers than the 168 that the ten warps of two CTAs of 160 threads leave each: 128 * 208 + 128 * 48 = 256 * 128, for the
// warps that compute and for the one that fills the rings with three idle ones beside it.  32 sequences of up to 20 pairs take 59 us so, 64 with 90 bytes in local
// memory; eight pairs are slower by it, 103 and 101 us.  (Three blocks of pairs, which would read the keys of 20 pairs once, took 77 us.)
template <int D, int NP> __host__ __device__ constexpr bool splits_registers() { return D == 128 && NP == 2; }
template <int D, int NP> __host__ __device__ constexpr int threads() { return splits_registers<D, NP>() ? 256 : 160; }
// Blocks of 16 columns joined at a time, as shared memory has room for.
template <int D, int NP> __host__ __device__ constexpr int join_blocks() { return D == 128 && NP == 2 ? 2 : 4; }
template <int D, int NP> __host__ __device__ constexpr uint32_t join_pitch() { return join_blocks<D, NP>() * 16 + 2; }
template <int D, int NP> constexpr size_t smem_bytes() { return 1024 + (size_t)kWarps * kStages * stage_bytes<D>() + kWarps * NP * 8 * join_pitch<D, NP>() * 4; }

__device__ unsigned int g_decode8_error;

struct Maps {
    CUtensorMap k, v;
};
// Of the keys in a ring's stage.
template <int H> struct __align__(8) Step {
    int have[kGroups];                                   // how many of each 16 exist
    float scale[H][kGroups][2];                          // of keys and values
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
constexpr uint32_t kBias = 0x80808080u;                  // of four bytes
constexpr float kUnit = 0x1p-24f;                        // of the codes as operands
// Two codes as operands without their bias, exact as well.
__device__ __forceinline__ uint32_t unbiased(uint32_t v)
{
    const uint32_t bias = 0x00800080u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&bias));
    return *reinterpret_cast<const uint32_t *>(&h);
}
// 2^e for e from -126 to 127.
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <typename T, int D, int NP, int H>              // D: head size rounded up to 64, 128 or 256; NP: blocks of 8 pairs; H: key / value heads of a unit
__global__ void __launch_bounds__(threads<D, NP>(), ctas_per_sm<D>()) decode8_kernel(const __grid_constant__ Maps maps, const Attend8Args a, bool wide)
{
    constexpr int KT = D / 16, S = kStages, PARTS = D / row_bytes<D>();
    constexpr uint32_t kStage = stage_bytes<D>(), kRow = row_bytes<D>(), kBox = box_bytes<D>(), kGroup = group_bytes<D>();
    constexpr uint32_t kPer = kRow / 4;                  // consecutive codes of a key that a lane takes for the scores
    constexpr uint32_t kOwn = kRow / 8;                  // and of a value for the results
    constexpr uint32_t kWords = kPer / 4;
    constexpr int kRings = kWarps / H, kBlock = kRings * kStep, kRows = 8 * NP * H;
    static_assert(H == 1 || PARTS == 1, "two heads in one box");
    using Way = Walk<kRows, kBlock, kExtra>;
    extern __shared__ uint8_t s_raw[];
    __shared__ unsigned long long s_walk[40];
    __shared__ __align__(8) unsigned long long s_full[kRings][S], s_empty[kRings][S];
    __shared__ Way s_way;
    __shared__ Segment s_seg[8];                         // the last units begun; no tokens behind the last
    __shared__ Step<H> s_step[kRings][S];
    __shared__ float s_m[kWarps][8 * NP], s_l[kWarps][8 * NP];
    __shared__ volatile int s_failed;
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = __shfl_sync(0xffffffffu, t >> 5, 0), d = a.d;
    uint8_t *s_mem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t ring = warp % kRings, sub = warp / kRings;            // whose keys this warp takes, of which of the unit's heads
    const uint8_t *codes = s_mem + ring * (S * H * kStage);
    float *s_join = reinterpret_cast<float *>(s_mem + (size_t)kWarps * S * kStage);
    if (t == 0) {
        for (int i = 0; i < kRings * S; i++) {
            mbar_init(&s_full[i / S][i % S], 4 * kGroups);       // a box and scales of keys and of values each
            mbar_init(&s_empty[i / S][i % S], H);
        }
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_launch_dependents();
    pdl_wait();
    {
        Way way;
        way.begin(a, blockIdx.x, gridDim.x, s_walk);
        if (t == kWarps * 32) s_way = way;
    }
    if (t == 0) clear_parts(a, blockIdx.x);
    __syncthreads();

    if (warp >= kWarps) {
        if constexpr (splits_registers<D, NP>()) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp > kWarps) return;
        // lane = ring * 4 + group of 16 keys * 2 + (keys or values); a segment without keys is a step without loads, and so is the end
        const uint32_t to = (lane >> 2) % kRings, group = lane >> 1 & 1u, values = lane & 1u, within = (1u << a.page_shift) - 1;
        const bool mine = lane < 4 * kRings;
        uint32_t seg = 0, slot = 0, round = 0, armed = 0;
        bool ok = true, more = true;
        while (more && ok) {
            if (lane == 0) {
                Segment g;
                if (!s_way.next(a, g)) g.tokens = g.begin = g.end = 0;
                s_seg[seg & 7u] = g;
            }
            __syncwarp();
            const Segment &g = s_seg[seg & 7u];
            seg++;
            more = g.tokens != 0;
            const uint32_t *table = g.table;
            const uint32_t begin = g.begin, end = max(g.end, g.begin + 1);
            const int len = more && g.end > g.begin ? g.len : 0, kv = (int)g.kv * H;
            uint32_t key = begin * kBlock + to * kStep + group * 16;
            uint32_t page = mine && (int)key < len ? table[key >> a.page_shift] : 0xFFFFFFFFu;
            for (uint32_t b = begin; b < end; b++) {
                const uint32_t next_key = key + kBlock, next_page = mine && b + 1 < end && (int)next_key < len ? table[next_key >> a.page_shift] : 0xFFFFFFFFu;      // a step ahead
                if (!(ok = mbar_wait_lanes(&s_empty[to][slot], (round & 1u) ^ 1u, mine, &s_failed, &g_decode8_error))) break;
                if (mine) {
                    const bool real = page < a.pages;            // also: in front of the sequence's end
                    unsigned long long *bar = &s_full[to][slot];
                    Step<H> &step = s_step[to][slot];
                    if (!values) step.have[group] = real ? min(16, len - (int)key) : 0;      // written before the arrivals that publish it
                    if (real) {
                        const uint32_t at = (page << a.page_shift) + (key & within), dst = smem_u32(s_mem) + ((to * S + slot) * 2 * kGroups + values * kGroups + group) * (H * kGroup);
                        const float *from = (values ? a.v_scales : a.k_scales) + (size_t)(at >> a.block_shift) * (a.kv_heads * H) + kv;
#pragma unroll
                        for (int h = 0; h < H; h++) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&step.scale[h][group][values])), "l"(from + h) : "memory");
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
                        mbar_arrive_expect_tx(bar, H * kGroup);
#pragma unroll
                        for (int c = 0; c < PARTS; c++) tma_load_3d(dst + c * kBox, values ? &maps.v : &maps.k, c * 128, kv, (int)at, bar);
                    } else {
#pragma unroll
                        for (int h = 0; h < H; h++) step.scale[h][group][values] = 0.f;
                        mbar_arrive(bar);
                        mbar_arrive(bar);
                    }
                }
                __syncwarp();
                key = next_key;
                page = next_page;
                armed++;
                if (++slot == S) { slot = 0; round++; }
            }
        }
        // given up: the copies in flight land before the CTA exits
        if (!ok && lane < kRings)
            for (uint32_t i = 0; i < min(armed, (uint32_t)S); i++) {
                if (slot-- == 0) { slot = S - 1; round--; }
                for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&s_full[lane][slot], round & 1u); w++) { }
            }
        return;
    }

    // ---- the warps that use them
    if constexpr (splits_registers<D, NP>()) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // A warp whose wait ran out meets the others once more, behind the unit, and all four leave: nobody waits for one that is gone.
    auto meet = [] { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); };
    auto any = [](bool mine) {
        uint32_t r;
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)mine) : "memory");
        return r != 0;
    };
    uint32_t c_seg = 0, slot = 0, parity = 0;
    bool ok = true;
    const uint32_t row = lane >> 2, quad = lane & 3u;
    // byte `at` of key r of this warp's head in a box, as the swizzle of 64 or 128 bytes places its 16-byte pieces
    auto place = [&](uint32_t r, uint32_t at) {
        const uint32_t line = r * H + sub;
        return line * kRow + (at ^ (kRow == 128 ? (line & 7u) << 4 : (line >> 1 & 3u) << 4));
    };
    // The key of a product's row r (of 8), and the 16 codes that are a lane's c-th: any order will do that is the same for all operands.  With one head a
    // quarter of a warp reads pieces of two lines that differ in their last bit, with two heads lines of one parity: keys 0 2 1 3 6 4 7 5 and a lane's pieces four
    // apart leave no two pieces of eight lanes in the same banks, neither of keys nor of values (heads of 64 in pairs: two).
    auto key_of = [](uint32_t r) { return H == 1 ? r : 0x57463120u >> (4 * r) & 7u; };
    auto piece = [&](uint32_t c) { return H == 1 || kWords == 4 ? quad * (kPer / 16) + c : quad + 4 * c; };
    const uint32_t my_key = key_of(row);
    for (;; c_seg++) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[ring][slot], parity, &s_failed, &g_decode8_error));
        const Segment g = s_seg[c_seg & 7u];
        if (!ok || g.tokens == 0) {
            any(!ok);
            break;
        }
        const uint32_t heads = g.heads / H, pairs = g.tokens * heads;        // of a key / value head
        // queries of pair `row` of each block of 8: for part c of 128 dimensions those from c * 128 + quad * kPer on
        uint32_t q[NP][KT][2];
        float factor[NP][2], bias[NP][2];                // of the pairs 2 quad and 2 quad + 1, whose scores this lane has
        int pos[NP][2];
#pragma unroll
        for (int n = 0; n < NP; n++) {
            const uint32_t r = n * 8 + row, token = r / heads, head = r - token * heads + sub * heads;
            const bool live = r < pairs;
            const T *src = static_cast<const T *>(a.q) + (size_t)(g.row0 + (live ? token : 0)) * a.q_pitch + (size_t)(g.head0 + (live ? head : 0)) * d;
            float up = 1.f, total = 0.f;
            T v[PARTS][kPer];
#pragma unroll
            for (int c = 0; c < PARTS; c++)
#pragma unroll
                for (uint32_t e = 0; e < kPer; e += 8) {
                    const uint32_t at = c * 128 + piece(e / 16) * 16 + e % 16;   // d is a multiple of 16: all eight or none
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (live && at < d) {
                        if (wide) {
                            w = *reinterpret_cast<const uint4 *>(src + at);
                        } else {
                            uint16_t x[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) x[i] = reinterpret_cast<const uint16_t *>(src)[at + i];
                            w = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16);
                        }
                    }
                    *reinterpret_cast<uint4 *>(&v[c][e]) = w;
                }
            if constexpr (!std::is_same<T, __half>::value) {
                uint32_t top = 0;                        // exponents of bf16
#pragma unroll
                for (int c = 0; c < PARTS; c++)
#pragma unroll
                    for (uint32_t e = 0; e < kPer; e++) top = max(top, (uint32_t)__bfloat16_as_ushort(v[c][e]) & 0x7FFFu);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int exponent = min(max((int)(top >> 7) - 127 - 13, -100), 112);     // the largest becomes 2^13 to 2^14
                up = power(-exponent);
                const float f = power(exponent);
                factor[n][0] = __shfl_sync(0xffffffffu, f, 8 * quad) * (a.scale_log2 / kUnit);
                factor[n][1] = __shfl_sync(0xffffffffu, f, 8 * quad + 4) * (a.scale_log2 / kUnit);
            } else {
                factor[n][0] = factor[n][1] = a.scale_log2 / kUnit;
            }
#pragma unroll
            for (int c = 0; c < PARTS; c++)
#pragma unroll
                for (uint32_t w = 0; w < kWords; w++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const T x = v[c][4 * w + 2 * h], y = v[c][4 * w + 2 * h + 1];
                        const __half2 both = __floats2half2_rn(to_f32(x) * up, to_f32(y) * up);
                        q[n][c * kWords + w][h] = *reinterpret_cast<const uint32_t *>(&both);
                        total += __low2float(both) + __high2float(both);
                    }
            total += __shfl_xor_sync(0xffffffffu, total, 1);
            total += __shfl_xor_sync(0xffffffffu, total, 2);
            bias[n][0] = __shfl_sync(0xffffffffu, total, 8 * quad) * (-128.f * kUnit);
            bias[n][1] = __shfl_sync(0xffffffffu, total, 8 * quad + 4) * (-128.f * kUnit);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t p = n * 8 + 2 * quad + e;
                pos[n][e] = p < pairs ? g.pos0 + (int)(p / heads) : -1;
            }
        }
        float o[NP][KT][4], m[NP][2], l[NP][2];
        int e2 = -124;                                   // results are relative to 2^e2, the blocks' scales below it; up1 * up2 = 2^(kUp - e2)
        float limit = 0.f, up1 = 0.f, up2 = 0.f;
#pragma unroll
        for (int n = 0; n < NP; n++) {
#pragma unroll
            for (int j = 0; j < KT; j++) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
        const uint32_t blocks = max(g.end, g.begin + 1) - g.begin;
        const int last_pos = g.pos0 + (int)g.tokens - 1;
        for (uint32_t b = 0; b < blocks; b++) {
            if (b > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&s_full[ring][slot], parity, &s_failed, &g_decode8_error)))) break;
            const uint8_t *base = codes + slot * (H * kStage);
            const Step<H> &step = s_step[ring][slot];
            unsigned long long *const empty = &s_empty[ring][slot];
            int have[kGroups];
            float ks[kGroups], vs[kGroups];
#pragma unroll
            for (int i = 0; i < kGroups; i++) {
                have[i] = step.have[i];
                // An infinite one becomes NaN: where codes are zeros the bias leaves a rest of either sign, and -infinity would be a key that has no weight.
                ks[i] = fmaf(step.scale[sub][i][0], 0.f, step.scale[sub][i][0]);
                vs[i] = step.scale[sub][i][1];
            }
            slot = slot == S - 1 ? 0 : slot + 1;
            parity ^= slot == 0;
            auto leave = [&]() {                         // all lanes have read
                __syncwarp();
                if (lane == 0) mbar_arrive(empty);
            };
            const int key0 = (int)((g.begin + b) * kBlock + ring * kStep);
            if (have[0] + have[kGroups - 1] == 0 || key0 > last_pos) {
                leave();
                continue;
            }
            float s[kGroups][NP][4];
#pragma unroll
            for (int i = 0; i < kGroups; i++) {
#pragma unroll
                for (int n = 0; n < NP; n++) {
                    s[i][n][0] = s[i][n][2] = bias[n][0];
                    s[i][n][1] = s[i][n][3] = bias[n][1];
                }
#pragma unroll
                for (int c = 0; c < PARTS; c++) {
                    const uint8_t *k = base + i * (H * kGroup) + c * kBox;
                    uint32_t w[2][kWords];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (uint32_t e = 0; e < kWords; e += 4) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(k + place(my_key + 8 * h, piece(e / 4) * 16));
                            w[h][e] = x.x ^ kBias; w[h][e + 1] = x.y ^ kBias; w[h][e + 2] = x.z ^ kBias; w[h][e + 3] = x.w ^ kBias;
                        }
#pragma unroll
                    for (uint32_t e = 0; e < kWords; e++) {
                        const uint32_t f[4] = {__byte_perm(w[0][e], 0, 0x4140), __byte_perm(w[1][e], 0, 0x4140), __byte_perm(w[0][e], 0, 0x4342), __byte_perm(w[1][e], 0, 0x4342)};
#pragma unroll
                        for (int n = 0; n < NP; n++) mma(s[i][n], f, q[n][c * kWords + e][0], q[n][c * kWords + e][1]);
                    }
                }
            }
            // keys my_key and my_key + 8 of a group by pairs 2 quad and 2 quad + 1
            const bool whole = have[0] + have[kGroups - 1] == kStep && key0 + kStep - 1 <= g.pos0 && (!a.window || key0 > last_pos - (int)a.window);
            bool up = false;
#pragma unroll
            for (int i = 0; i < kGroups; i++)
#pragma unroll
                for (int n = 0; n < NP; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = __fmul_rn(s[i][n][e], factor[n][e & 1] * ks[i]);
                        if (!whole) {
                            const int at = (int)my_key + e / 2 * 8, key = key0 + i * 16 + at, p = pos[n][e & 1];
                            x = at < have[i] && key <= p && (!a.window || key > p - (int)a.window) ? x : -INFINITY;
                        }
                        s[i][n][e] = x;
                        up |= x > m[n][e & 1] + kRoom;   // never where x is -inf or NaN
                    }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int n = 0; n < NP; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float top = m[n][e];
#pragma unroll
                        for (int i = 0; i < kGroups; i++) top = fmaxf(top, fmaxf(s[i][n][e], s[i][n][e + 2]));
#pragma unroll
                        for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        const float keep = top > m[n][e] ? exp2_fast(m[n][e] - top) : 1.f;
                        m[n][e] = top;
                        l[n][e] *= keep;
#pragma unroll
                        for (int j = 0; j < KT; j++) {
                            o[n][j][e] *= keep;
                            o[n][j][e + 2] *= keep;
                        }
                    }
            }
#pragma unroll
            for (int i = 0; i < kGroups; i++) {
                // the block's scale below 2^e2: from 2^-3 on where e2 follows it
                if (!(vs[i] < limit)) {
                    const int exponent = (int)(__float_as_uint(vs[i]) >> 23 & 255u) - 126;          // vs < 2^exponent; 129 for one that is not finite, which has no say
                    if (exponent < 129) {
                        const int next = min(exponent + 2, 127);
                        const float keep = limit > 0.f ? power(max(e2 - next, -126)) : 0.f;
#pragma unroll
                        for (int n = 0; n < NP; n++)
#pragma unroll
                            for (int j = 0; j < KT; j++)
#pragma unroll
                                for (int e = 0; e < 4; e++) o[n][j][e] *= keep;
                        e2 = next;
                        limit = power(e2);
                        const int shift = kUp - e2;      // in two steps, as 2^shift alone may be out of range
                        up1 = power(max(min(shift, 100), -126));
                        up2 = power(max(shift - 100, 0));
                    }
                }
                const float by = vs[i] * up1 * up2;
                uint32_t weight[NP][2], low[NP][2];
#pragma unroll
                for (int n = 0; n < NP; n++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float x = s[i][n][2 * h + e], p = exp2_fast(__fsub_rn(x, m[n][e] == -INFINITY ? 0.f : m[n][e]));
                            l[n][e] += p;
                            w[e] = whole || x != -INFINITY ? p * by : 0.f;                           // no product where nothing is seen: the scale may be anything
                        }
                        const __half2 both = __floats2half2_rn(w[0], w[1]);
                        weight[n][h] = transpose(*reinterpret_cast<const uint32_t *>(&both));
                        const __half2 rest = __floats2half2_rn(w[0] - __low2float(both), w[1] - __high2float(both));
                        low[n][h] = transpose(*reinterpret_cast<const uint32_t *>(&rest));
                    }
                // values of the keys of rows 2 quad, 2 quad + 1, and eight on, dimensions row * kOwn on: a product's rows are two of them each
#pragma unroll
                for (int c = 0; c < PARTS; c++) {
                    const uint8_t *v = base + (kGroups + i) * (H * kGroup) + c * kBox;
                    uint32_t w[4][kOwn / 4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint8_t *at = v + place(key_of(2 * quad + (k & 1)) + (k >> 1) * 8, row * kOwn);
                        if constexpr (kOwn == 16) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(at);
                            w[k][0] = x.x; w[k][1] = x.y; w[k][2] = x.z; w[k][3] = x.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2 *>(at);
                            w[k][0] = x.x; w[k][1] = x.y;
                        }
                    }
#pragma unroll
                    for (uint32_t e = 0; e < kOwn / 4; e++) {
                        // [a0 b0 a1 b1] and [a2 b2 a3 b3] of the keys a, b
                        const uint32_t x0 = __byte_perm(w[0][e], w[1][e], 0x5140) ^ kBias, x1 = __byte_perm(w[0][e], w[1][e], 0x7362) ^ kBias;
                        const uint32_t y0 = __byte_perm(w[2][e], w[3][e], 0x5140) ^ kBias, y1 = __byte_perm(w[2][e], w[3][e], 0x7362) ^ kBias;
                        const uint32_t f[2][4] = {
                            {unbiased(__byte_perm(x0, 0, 0x4140)), unbiased(__byte_perm(x0, 0, 0x4342)), unbiased(__byte_perm(y0, 0, 0x4140)), unbiased(__byte_perm(y0, 0, 0x4342))},
                            {unbiased(__byte_perm(x1, 0, 0x4140)), unbiased(__byte_perm(x1, 0, 0x4342)), unbiased(__byte_perm(y1, 0, 0x4140)), unbiased(__byte_perm(y1, 0, 0x4342))}};
#pragma unroll
                        for (int n = 0; n < NP; n++)
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                float (&acc)[4] = o[n][c * (kOwn / 2) + 2 * e + j];
                                mma(acc, f[j], weight[n][0], weight[n][1]);
                                mma(acc, f[j], low[n][0], low[n][1]);
                            }
                    }
                }
            }
            leave();
        }

        if (any(!ok)) break;

        // ---- the sums of the warps of a head
#pragma unroll
        for (int n = 0; n < NP; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float sum = l[n][e];
#pragma unroll
                for (int x = 4; x < 32; x *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                if (row == 0) {
                    s_m[warp][n * 8 + 2 * quad + e] = m[n][e];
                    s_l[warp][n * 8 + 2 * quad + e] = sum;
                }
            }
        meet();
        auto top_of = [&](uint32_t h, uint32_t r) {
            float top = s_m[h * kRings][r];
#pragma unroll
            for (int w = 1; w < kRings; w++) top = fmaxf(top, s_m[h * kRings + w][r]);
            return top;
        };
        auto total = [&](uint32_t h, uint32_t r, float &top) {
            top = top_of(h, r);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kRings; w++) sum += s_l[h * kRings + w][r] != 0.f ? s_l[h * kRings + w][r] * exp2_fast(s_m[h * kRings + w][r] - top) : 0.f;
            return sum;
        };
        const float scale2 = power(e2) * (1.f / (1 << kUp) / kUnit);
#pragma unroll
        for (int n = 0; n < NP; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t r = n * 8 + 2 * quad + e;
                const float top = top_of(sub, r), mine = s_l[warp][r] != 0.f ? exp2_fast(m[n][e] - top) : 0.f;
#pragma unroll
                for (int j = 0; j < KT; j++) {
                    o[n][j][e] = mine != 0.f ? o[n][j][e] * mine * scale2 : 0.f;
                    o[n][j][e + 2] = mine != 0.f ? o[n][j][e + 2] * mine * scale2 : 0.f;
                }
            }
        const bool alone = g.first && g.last;
        float *part = a.parts + (size_t)part_index(blockIdx.x, g) * kRows * (d + 2);
        // of every lane row's kOwn dimensions (of 128) kSpan at a time
        constexpr uint32_t kJoinPitch = join_pitch<D, NP>();
        constexpr int kAt = join_blocks<D, NP>(), kSpan = 2 * kAt;
#pragma unroll
        for (int j0 = 0; j0 < KT; j0 += kAt) {
#pragma unroll
            for (int n = 0; n < NP; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float *dst = s_join + (warp * (8 * NP) + n * 8 + 2 * quad + e) * kJoinPitch + row * kSpan;
#pragma unroll
                    for (int j = 0; j < kAt; j++) *reinterpret_cast<float2 *>(dst + 2 * j) = make_float2(o[n][j0 + j][e], o[n][j0 + j][e + 2]);
                }
            meet();
            for (uint32_t i = t; i < H * pairs * 8; i += kWarps * 32) {
                const uint32_t h = H == 1 ? 0u : i / (pairs * 8), r = i / 8 - h * pairs, at = i % 8, token = r / heads, head = h * heads + r - token * heads;
                const uint32_t per = kOwn / 2, column = j0 / per * 128 + at * kOwn + j0 % per * 2;
                if (column >= d) continue;
                float x[kSpan];
#pragma unroll
                for (int c = 0; c < kSpan; c += 2) {
                    x[c] = x[c + 1] = 0.f;
#pragma unroll
                    for (int w = 0; w < kRings; w++) {
                        const float2 v = *reinterpret_cast<const float2 *>(s_join + ((h * kRings + w) * (8 * NP) + r) * kJoinPitch + at * kSpan + c);
                        x[c] += v.x;
                        x[c + 1] += v.y;
                    }
                }
                if (alone) {
                    float top;
                    const float sum = total(h, r, top), inv = sum == 0.f ? 0.f : 1.f / sum;
                    T *dst = static_cast<T *>(a.out) + (size_t)(g.row0 + token) * a.out_pitch + (size_t)(g.head0 + head) * d + column;
                    T y[kSpan];
#pragma unroll
                    for (int c = 0; c < kSpan; c++) y[c] = rounded<T>(x[c] * inv);
                    if (wide) {
#pragma unroll
                        for (int c = 0; c < kSpan; c += 4) *reinterpret_cast<uint2 *>(dst + c) = *reinterpret_cast<const uint2 *>(y + c);
                    } else {
#pragma unroll
                        for (int c = 0; c < kSpan; c++) dst[c] = y[c];
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kSpan; c += 2) *reinterpret_cast<float2 *>(part + (token * g.heads + head) * d + column + c) = make_float2(x[c], x[c + 1]);
                }
            }
            meet();
        }
        if (!alone) {
            if (t < H * pairs) {
                const uint32_t token = t / g.heads, head = t - token * g.heads, h = head / heads;
                float top;
                const float sum = total(h, token * heads + head - h * heads, top);
                part[kRows * d + 2 * t] = top;
                part[kRows * d + 2 * t + 1] = sum;
            }
            if (t == 0) name_part(a, blockIdx.x, g);
            meet();                                      // before the next unit's maxima
        }
    }
}

template <typename T, int D, int NP, int H>
int launch_sized(const Attend8Args &a, const Maps &maps, bool wide, uint32_t pairs, cudaStream_t stream)
{
    constexpr uint32_t ctas = 148 * ctas_per_sm<D>();
    auto *kernel = decode8_kernel<T, D, NP, H>;
    if (int rc = allow_smem(kernel, smem_bytes<D, NP>())) return rc;
    MGQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (int rc = launch(kernel, dim3(ctas), dim3(threads<D, NP>()), smem_bytes<D, NP>(), stream, maps, a, wide)) return rc;
    return launch_merge<T, 8 * NP * H>(a, ctas, H * min(pairs, 8u * NP), stream);      // no unit has more; `pairs` may be any bound
}

template <typename T, int H>
int launch_heads(const Attend8Args &a, const Maps &maps, bool wide, uint32_t pairs, cudaStream_t stream)
{
    if (pairs <= 8) return a.d <= 64 ? launch_sized<T, 64, 1, H>(a, maps, wide, pairs, stream) : launch_sized<T, 128, 1, H>(a, maps, wide, pairs, stream);
    return a.d <= 64 ? launch_sized<T, 64, 2, H>(a, maps, wide, pairs, stream) : launch_sized<T, 128, 2, H>(a, maps, wide, pairs, stream);
}
// Two key / value heads to a unit: as one with the query heads of both.
bool in_pairs(const Attend8Args &a) { return a.d <= 128 && a.kv_heads % 2 == 0 && a.group <= 16; }
template <typename T>
int launch_typed(const Attend8Args &a, const Maps &maps, bool wide, uint32_t pairs, cudaStream_t stream)
{
    if (a.d > 128) return launch_sized<T, 256, 1, 1>(a, maps, wide, pairs, stream);
    if (!in_pairs(a)) return launch_heads<T, 1>(a, maps, wide, pairs, stream);
    Attend8Args b = a;
    b.kv_heads /= 2;
    b.group *= 2;
    b.rows_to = a.rows_to < 0x80000000u ? 2 * a.rows_to + 1 : a.rows_to;
    return launch_heads<T, 2>(b, maps, wide, pairs, stream);
}

// {head_dim, kv_heads, pages * page_size} of a cache, for boxes of 64 or 128 codes by 16 tokens of one head or two, in the swizzle of that size.  What lies outside
// reads as zero.
int encode_codes(CUtensorMap &map, const void *base, const Attend8Args &a)
{
    EncodeTiledFn encode = nullptr;
    if (int rc = encode_fn(encode)) return rc;
    const cuuint64_t dims[3] = {a.d, a.kv_heads, (cuuint64_t)a.pages << a.page_shift};
    const cuuint64_t strides[2] = {a.d, (cuuint64_t)a.kv_heads * a.d};
    const cuuint32_t box[3] = {a.d <= 64 ? 64u : 128u, in_pairs(a) ? 2u : 1u, 16}, elem[3] = {1, 1, 1};
    const CUresult cr = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               a.d <= 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                               a.d % 128 == 0 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? MGQ_OK : fail(MGQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
}

}  // namespace

uint32_t decode8_ctas(uint32_t head_dim) { return 148 * (head_dim <= 64 ? ctas_per_sm<64>() : head_dim <= 128 ? ctas_per_sm<128>() : ctas_per_sm<256>()); }

int launch_decode8(const Attend8Args &a, int dtype, uint32_t pairs, cudaStream_t stream)
{
    Maps maps;
    if (int rc = encode_codes(maps.k, a.k, a)) return rc;
    if (int rc = encode_codes(maps.v, a.v, a)) return rc;
    auto on = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool wide = on(a.q) && on(a.out) && a.q_pitch % 8 == 0 && a.out_pitch % 8 == 0;
    return dtype == MGQ_FMT_F16 ? launch_typed<__half>(a, maps, wide, pairs, stream) : launch_typed<__nv_bfloat16>(a, maps, wide, pairs, stream);
}

int decode8_status()
{
    unsigned int err = 0;
    MGQ_CUDA(cudaMemcpyFromSymbol(&err, g_decode8_error, sizeof err));
    if (!err) return prefill8_status();
    const unsigned int zero = 0;
    MGQ_CUDA(cudaMemcpyToSymbol(g_decode8_error, &zero, sizeof zero));
    return fail(MGQ_ERR_TIMEOUT, "a bounded wait inside the attention of few tokens over 8-bit codes ran out");
}

size_t paged_attention_int8_workspace(uint32_t head_dim)
{
    const uint32_t ctas = decode8_ctas(head_dim);
    const size_t many = head_dim <= 128 ? kPrefillCtas * 2 * (sizeof(PartHead) + (size_t)kPrefillRows * (head_dim + 2) * sizeof(float)) : 0;
    return ctas * 2 * (sizeof(PartHead) + (size_t)kDecode8Rows * (head_dim + 2) * sizeof(float)) + many;
}

int launch_paged_attention_int8(const void *q, const int8_t *k_cache, const int8_t *v_cache, const float *k_scales, const float *v_scales, int dtype, const uint32_t *table,
                                const uint32_t *starts, const uint32_t *lengths, void *out, uint32_t sequences, uint32_t rows, uint32_t max_fresh, uint32_t heads,
                                uint32_t kv_heads, uint32_t head_dim, uint32_t page_size, uint32_t pages, uint32_t block, uint32_t table_width, uint32_t q_pitch,
                                uint32_t out_pitch, float scale, uint32_t window, void *workspace, void *stream)
{
    Attend8Args a{};
    a.q = q; a.k = k_cache; a.v = v_cache; a.out = out;
    a.k_scales = k_scales; a.v_scales = v_scales; a.block_shift = page_shift(block);
    a.starts = starts; a.lengths = lengths; a.table = table;
    a.sequences = sequences; a.rows = rows; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.d = head_dim;
    a.page_shift = page_shift(page_size); a.pages = pages; a.table_width = table_width;
    a.window = window < (1u << 31) ? window : 0u;                      // no sequence is longer
    a.q_pitch = q_pitch; a.out_pitch = out_pitch;
    a.rows_from = 1; a.rows_to = 0xFFFFFFFFu;
    a.least = kLeastBlocks;
    a.scale_log2 = scale * 1.4426950408889634f;
    const uint32_t pairs = (uint32_t)min((unsigned long long)max_fresh * a.group, 0xFFFFFFFFull);
    a.heads = static_cast<PartHead *>(workspace);
    a.parts = reinterpret_cast<float *>(a.heads + 2 * decode8_ctas(a.d));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (pairs <= kDecode8Pairs || !prefill8_takes(a)) return launch_decode8(a, dtype, pairs, s);
    const unsigned long long reach = (unsigned long long)table_width * page_size, units = ((unsigned long long)rows * a.group / 16 + sequences) * kv_heads;
    if (max_fresh <= kMostUnits * max(16 / a.group, 1u) && units <= kLittle / (reach + kPlace)) return launch_decode8(a, dtype, pairs, s);
    const bool many = (unsigned long long)rows * a.group > (unsigned long long)kDecode8Pairs * sequences;
    const bool alone = many && (sequences * reach <= kShort || (sequences == 1 && rows >= kManyRows));
    if (!alone) {
        a.rows_to = kDecode8Pairs;
        if (int rc = launch_decode8(a, dtype, kDecode8Pairs, s)) return rc;
        a.rows_from = kDecode8Pairs + 1;
        a.rows_to = 0xFFFFFFFFu;
        a.heads = reinterpret_cast<PartHead *>(a.parts + (size_t)decode8_ctas(a.d) * 2 * kDecode8Rows * (a.d + 2));
    }
    a.least = 0;
    a.parts = reinterpret_cast<float *>(a.heads + 2 * kPrefillCtas);
    return launch_prefill8(a, dtype, s);
}

}  // namespace mgq
