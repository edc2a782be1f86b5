// Attention of many new tokens per sequence (portions of prompts, long drafts) over a paged cache of f16 or bf16, on tcgen05.
//
// A unit is 256 pairs of token and query head of one key / value head, two tiles of 128 rows that share the keys and values of a block
// of 128.  Per block and tile S = Q K^T and O += P V are four to eight products of K = 16 each way; the tensor cores need 512 cycles for either (heads
// of 128; a product of 128 x 128 x 16 takes 64), and the exponentials of a tile, 16 per cycle on the SM, 1024: two tiles in turn keep both busy.  A tile's chain
// takes 3200 per block (4 x 2048 tokens behind up to 6144, 549 GFLOP: 562 us and 977 TFLOP/s call after call, where the clock falls; 505 to 530 us for a few).
//   warps 0-3, 4-7  softmax of tile 0 and 1, a row per thread: S from TMEM, running maximum and sum in f32, P back into TMEM over S (as the
//                   16-bit left operand of the second product), results out of TMEM.  Two warps per row need a barrier per block (280 cycles, 671 us for
//                   4 x 2048 tokens); four lanes per row read TMEM at half the rate (500 cycles of a block, 653 us).
//   warp 8          keys and values: TMA boxes of a page's tokens (128 at most) by 64 elements, a lane each, into a ring of stages that hold
//                   128 keys or 128 values.
//   warp 9          issues S(j + 1) of a tile right behind O(j) of the same tile: products run in order, so P is read before S overwrites it, and whoever sees
//                   S(j + 1) done knows that O(j) is.  O(j) begins when the weights of the first 64 keys are there.
//   warp 10         finds the units, and loads their queries by TMA as soon as the last scores of the unit before are done.
// Sums are kept relative to a maximum that may be 2^8 too low, in f16 2^7: only where a row's maximum grows by more is O scaled.
// Weights are rounded to the values' type, as the tensor cores take both operands in one type; their sum is of the unrounded ones in f32.  In bf16 that leaves the
// results of 4 x 2048 tokens 2.19e-3 (2-norm) off the exact ones, where rounding these alone leaves 1.65e-3; with what is dropped as a second operand it
// was 1.65e-3, too, but 742 us.  f16 weights are relative to 2^-8 of the maximum, so that they go up to 2^15, have all their bits down to 2^-22 of it
// and are not lost above 2^-33 (relative to 2^-11, with a maximum that may grow by 2^4 only, calls took 8 % longer).
// TMEM: S0, S1 (128 columns each, P in the first 64 of them), O0, O1.
#include <cfloat>
#include <cstdint>

#include "mgq_paged.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 384;
constexpr int kExtra = 2;                                // blocks of keys that starting and ending a unit take as long as
// Exponents are score * scale - m in one rounding, m is rounded before, by up to 2^-24 of its size.  That is a factor which all weights of a row have in common, but
// beyond some size it takes them out of their type's range (from 2^27 on infinite f16 weights, from 2^34 rows of zeros): such rows are computed again.
constexpr float kHuge = 0x1p20f;
// How far below a row's maximum m lies when it is set, and how far above m the maximum may grow, in powers of two.
template <typename T> constexpr float kUnder = std::is_same<T, __half>::value ? 8.f : 0.f;
template <typename T> constexpr float kRoom = std::is_same<T, __half>::value ? 15.f : 8.f;
constexpr uint32_t kKeys = 128, kTile = 128;             // keys of a block, rows of a tile
constexpr uint32_t kHalf = kKeys * 128;                  // 128 rows of 64 elements
template <int D> __host__ __device__ constexpr uint32_t stage_bytes() { return D / 64 * kHalf; }
template <int D> __host__ __device__ constexpr int stages() { return D == 64 ? 8 : 5; }

__device__ unsigned int g_prefill_error;

using Way = Walk<kPrefillRows, kKeys, kExtra>;
struct __align__(16) Shared {
    unsigned long long full[8], empty[8], q_full, q_empty, s_full[2], p_half[2], p_full[2], o_full[2];
    Way way[2];                                          // of the producers of keys and of queries
    Segment kv_seg, next, seg[2];                        // of the producer of keys; of that of queries; of everybody else, two units in turn, no tokens behind the last
    int more;
    uint32_t there[8][4];                                // keys of a block that exist, for the last eight blocks
    uint32_t holes[2];                                   // whether the unit's keys have pages that do not exist
    uint32_t tmem;
    volatile int failed;
    volatile uint32_t again;                             // counts on while rows are computed again
};
template <int D> constexpr size_t smem_bytes() { return (size_t)(2 + stages<D>()) * stage_bytes<D>() + sizeof(Shared); }
static_assert(smem_bytes<128>() <= 227 * 1024 && smem_bytes<64>() <= 227 * 1024, "shared memory of an SM");

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

// mbar_wait for roles that may wait for rows that are computed again: that takes as long as there are keys, and while `again` counts on nobody gives up.
__device__ __forceinline__ bool wait_for(Shared &sh, unsigned long long *bar, uint32_t parity)
{
    uint32_t again = sh.again;
    for (uint32_t i = 0; i < kWaitLimit; i++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (sh.failed) return false;
        const uint32_t now = sh.again;
        if (now != again) {
            again = now;
            i = 0;
        }
    }
    sh.failed = 1;
    atomicExch(&g_prefill_error, 1u);
    return false;
}

// Key blocks of one tile of a segment: [g.begin, what is returned).  last_token: that of the tile's last row, were all tokens there.
__device__ __forceinline__ uint32_t tile_end(const Segment &g, uint32_t tile, uint32_t last_token)
{
    if (tile * kTile >= g.tokens * g.heads) return g.begin;
    const int last = min(g.pos0 + (int)min(last_token, g.tokens - 1), g.len - 1);
    return last < 0 ? g.begin : max(g.begin, min(g.end, (uint32_t)last / kKeys + 1));
}

// 8 values of T as f32.
template <typename T>
__device__ __forceinline__ void unpack(const uint4 &v, float (&f)[8])
{
    const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = to_f32(e[i]);
}
// One row of a segment again, on the CUDA cores and without what it does not see: where a value that only other rows see is infinite or NaN, its
// product with a weight of 0 has spoilt the row, and where scores are huge their weights have left the type's range.  A whole warp: eight lanes share a key, each with 8 of
// 64 columns, and the four groups of lanes have maxima and sums of their own, joined at the end, when all of them hold the row.  Loads' latency bounds it: eight keys at
// a time, fetched while the eight before are used, their pages looked up another step ahead.
template <typename T, int D>
__device__ __noinline__ void row_again(const AttendArgs &a, Shared &sh, const Segment &g, uint32_t r, uint32_t end, float &m_out, float &l_out, float (&out)[D / 64][8])
{
    constexpr int C = D / 64, kStep = 8, N = kStep / 4;
    const uint32_t lane = threadIdx.x & 31u, token = r / g.heads, head = g.head0 + r - token * g.heads, column = lane % 8 * 8;
    const int pos = g.pos0 + (int)token, first = (int)(g.begin * kKeys), stop = min(min((int)(end * kKeys), pos + 1), g.len);
    float q[C][8], acc[C][8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const bool in = column + 64 * c < a.d;
        const T *src = static_cast<const T *>(a.q) + (size_t)(g.row0 + token) * a.q_pitch + (size_t)head * a.d + column + 64 * c;
        unpack<T>(in ? *reinterpret_cast<const uint4 *>(src) : make_uint4(0u, 0u, 0u, 0u), q[c]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            q[c][e] *= a.scale_log2;
            acc[c][e] = 0.f;
        }
    }
    uint4 k[N][C], v[N][C];
    uint32_t page[N];
    bool seen[N];
    auto look_up = [&](int key0) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int key = key0 + 4 * n + (int)(lane / 8);
            page[n] = key < stop && !(a.window && key <= pos - (int)a.window) ? g.table[(uint32_t)key >> a.page_shift] : 0xFFFFFFFFu;
        }
    };
    auto fetch = [&](int key0) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int key = key0 + 4 * n + (int)(lane / 8);
            seen[n] = page[n] < a.pages;
            const size_t at = seen[n] ? ((((size_t)page[n] << a.page_shift) + (key & ((1u << a.page_shift) - 1))) * a.kv_heads + g.kv) * a.d + column : 0;
#pragma unroll
            for (int c = 0; c < C; c++) {
                k[n][c] = v[n][c] = make_uint4(0u, 0u, 0u, 0u);
                if (seen[n] && column + 64 * c < a.d) {
                    k[n][c] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.k) + at + 64 * c);
                    v[n][c] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.v) + at + 64 * c);
                }
            }
        }
    };
    look_up(first);
    fetch(first);
    look_up(first + kStep);
    for (int key0 = first; key0 < stop; key0 += kStep) {
        if (lane == 0 && (key0 - first) % 1024 == 0) sh.again = sh.again + 1;     // other warps may do so at once: only that it changes counts
        float x[N], w[N][C][8];
#pragma unroll
        for (int n = 0; n < N; n++) {
            x[n] = 0.f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                unpack<T>(k[n][c], w[n][c]);
#pragma unroll
                for (int e = 0; e < 8; e++) x[n] = fmaf(q[c][e], w[n][c][e], x[n]);
                unpack<T>(v[n][c], w[n][c]);
            }
        }
        bool real[N];
#pragma unroll
        for (int n = 0; n < N; n++) real[n] = seen[n];
        fetch(key0 + kStep);
        look_up(key0 + 2 * kStep);
#pragma unroll
        for (int o = 1; o < 8; o *= 2)
#pragma unroll
            for (int n = 0; n < N; n++) x[n] += __shfl_xor_sync(0xffffffffu, x[n], o);
        float top = m;
#pragma unroll
        for (int n = 0; n < N; n++) {
            x[n] = real[n] ? x[n] : -INFINITY;
            top = fmaxf(top, x[n]);
        }
        const float base = top == -INFINITY ? 0.f : top, keep = exp2_fast(m - base);
        m = top;
        l *= keep;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) acc[c][e] *= keep;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const float p = exp2_fast(x[n] - base);
            l += p;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) acc[c][e] = fmaf(p, w[n][c][e], acc[c][e]);
        }
    }
#pragma unroll
    for (int o = 8; o < 32; o *= 2) {
        const float top = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o)), keep = l != 0.f ? exp2_fast(m - top) : 0.f;      // a NaN is a weight
        m = top;
        l *= keep;
        l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float mine = keep != 0.f ? acc[c][e] * keep : 0.f;
                acc[c][e] = mine + __shfl_xor_sync(0xffffffffu, mine, o);
            }
    }
    m_out = m;
    l_out = l;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) out[c][e] = acc[c][e];
}

template <typename T, int D>                             // D: head size rounded up to 64 or 128
__global__ void __launch_bounds__(kThreads, 1) prefill_kernel(const __grid_constant__ CacheMaps maps, const __grid_constant__ CUtensorMap q_map, const AttendArgs a)
{
    constexpr int S = stages<D>(), PARTS = D / 64;
    constexpr uint32_t kStage = stage_bytes<D>();
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
    constexpr uint32_t kInstrS = (1u << 4) | kType | (kKeys >> 3 << 17) | (kTile >> 4 << 24);
    constexpr uint32_t kInstrO = (1u << 4) | kType | (1u << 16) | ((uint32_t)D >> 3 << 17) | (kTile >> 4 << 24);
    extern __shared__ __align__(1024) uint8_t smem_raw[];                 // swizzled tiles lie on multiples of 1024
    uint8_t *s_q = smem_raw, *ring = s_q + 2 * kStage;
    Shared &sh = *reinterpret_cast<Shared *>(ring + S * kStage);
    if (smem_u32(smem_raw) % 1024 != 0) {                                 // cannot be with the alignment above
        if (threadIdx.x == 0) atomicExch(&g_prefill_error, 1u);
        return;
    }
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;

    if (tid == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 2);                                   // either tile's warps
        }
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 3);                                        // the issuer, both tiles' warps
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_half[i], 4);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
        }
        sh.failed = 0;
        sh.again = 0;
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
        if (lane == 0 && (warp == 8 || warp == 10)) sh.way[warp == 10] = way;
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
    auto lane_wait = [&](unsigned long long *bar, uint32_t parity) {
        return mbar_try_wait(bar, parity) || wait_for(sh, bar, parity);
    };
    auto wait = [&](unsigned long long *bar, uint32_t parity) {
        const bool done = lane_wait(bar, parity);
        __syncwarp();
        return done;
    };
    auto wait_all = [&](unsigned long long *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    // Registers where they are needed: 256 * 216 + 128 * 72 = 384 * 168.
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
        const uint32_t shift = a.page_shift, page_keys = 1u << shift, box = min(page_keys, kKeys), boxes = kKeys / box, gone = a.pages << shift;
        uint32_t slot = 0, round = 0, block = 0;
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
            for (uint32_t kb = kb_begin; ok && kb < kb_end; kb++, block++) {
                // lane = box of the block + boxes * group of 64 elements
                const uint32_t b = lane % boxes, part = lane / boxes, key = kb * kKeys + b * box;
                uint32_t y = gone, have = 0;
                if ((int)key < len) {
                    const uint32_t page = table[key >> shift];
                    if (page < a.pages) {
                        y = (page << shift) + (key & (page_keys - 1));
                        have = min(box, (uint32_t)len - key);
                    }
                }
                uint32_t there[4];
#pragma unroll
                for (int w = 0; w < 4; w++) there[w] = __reduce_or_sync(0xffffffffu, bits(b * box, b * box + have, 32 * w));
#pragma unroll
                for (int what = 0; what < 2 && ok; what++) {
                    if (!(ok = wait_all(&sh.empty[slot], (round & 1u) ^ 1u))) break;
                    if (lane == 0) {
                        if (what == 0)
                            for (int w = 0; w < 4; w++) sh.there[block & 7u][w] = there[w];
                        mbar_arrive_expect_tx(&sh.full[slot], kStage);
                    }
                    __syncwarp();
                    if (part < PARTS)
                        tma_load_3d(smem_u32(ring) + slot * kStage + part * kHalf + b * box * 128, what ? &maps.v : &maps.k, (int)part * 64, kv, (int)y, &sh.full[slot]);
                    __syncwarp();
                    armed++;
                    if (++slot == S) { slot = 0; round++; }
                }
            }
        }
        // given up: the copies in flight land before the CTA exits
        if (!ok && lane == 0)
            for (int i = 0; i < min(armed, S); i++) {
                if (slot-- == 0) { slot = S - 1; round--; }
                for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&sh.full[slot], round & 1u); w++) { }
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
                    for (int c = 0; c < PARTS; c++) tma_load_3d(smem_u32(s_q) + c * 2 * kHalf, &q_map, c * 64, (int)g.head0, (int)g.row0, &sh.q_full);
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
#pragma unroll
                for (uint32_t i = 1; i < D / 16; i++) umma_step<true>(tmem + tile * 128, q + i / 4 * (2 * kHalf / 16) + i % 4 * 2, k + i / 4 * (kHalf / 16) + i % 4 * 2, kInstrS);
                umma_commit(&sh.s_full[tile]);
            };
            // 64 keys, 16 per product
            auto values = [&](uint32_t tile, uint32_t at, uint32_t part, bool first) {
                const uint32_t v = ring16 + at * (kStage / 16), o = tmem + 256 + tile * D, p = tmem + tile * 128;
#pragma unroll
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
                // A wait takes the warp 100 cycles and more even where all is there already, so each stands where products are under way: for the next keys
                // behind the first half of tile 0's values, for the next values behind that of tile 1's.  A commit takes 200: the stages are given back by the
                // softmax warps, which learn from the scores' commits that their products are done.
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
#pragma unroll
                    for (uint32_t tile = 0; tile < 2; tile++) {
                        const bool values_now = stop[tile] > kb;
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
                            if (kb + 1 == stop[tile]) umma_commit(&sh.o_full[tile]);
                        }
                        if (stop[tile] > kb + 1) scores(tile, k_slot);
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const uint32_t tile = warp >> 2, quad = warp & 3u, r_tile = quad * 32 + lane, row = tile * kTile + r_tile, d = a.d;
        const uint32_t lanes = (quad * 32u) << 16, s_at = tmem + tile * 128 + lanes, o_at = tmem + 256 + tile * D + lanes;
        const float scale = a.scale_log2;
        const uint32_t token = row / slice, head = row - token * slice, first_token = tile * kTile / slice;     // of this row, of the tile's first
        uint32_t slot = 0, round = 0, block = 0;         // of the ring, as the producer counts
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
            float m = -INFINITY, l = 0.f;
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
            for (uint32_t kb = begin; kb < end; kb++, block++) {
                const uint32_t k_slot = slot, k_round = round;
                if (++slot == S) { slot = 0; round++; }
                const uint32_t v_slot = slot, v_round = round;
                if (++slot == S) { slot = 0; round++; }
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
                uint32_t there[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                if (!every) {
                    // For sight of `there`, and to write into the values.  Not the keys' barrier: their stage is free by now and may have been
                    // filled again, two phases on, where this parity would wait for a third.  The values' stage is free behind this tile's product only.
                    wait(&sh.full[v_slot], v_round & 1u);
#pragma unroll
                    for (int w = 0; w < 4; w++) there[w] = sh.there[block & 7u][w];
                    // values that nobody sees, whatever the page holds there, become zeros
                    uint8_t *v = ring + v_slot * kStage;
                    for (uint32_t i = r_tile; i < kKeys * PARTS * 8; i += 128) {
                        const uint32_t key = i / 8 % kKeys, w = key / 32, word = w == 0 ? there[0] : w == 1 ? there[1] : w == 2 ? there[2] : there[3];
                        if (!(word >> (key % 32) & 1u)) *reinterpret_cast<uint4 *>(v + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    any_of_tile(tile, false);            // all of them have, before the first weights are signalled
                }
                // 64 keys: what the row does not see
                auto mask = [&](float (&s)[64], int c) {
                    if (plain) return;
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const uint32_t seen = there[2 * c + w] & bits(window ? pos - window + 1 : 0, pos + 1, key0 + 64 * c + 32 * w);
#pragma unroll
                        for (int e = 0; e < 32; e++) s[32 * w + e] = seen >> e & 1u ? s[32 * w + e] : -INFINITY;
                    }
                    __syncwarp();
                };
                float s[64], t[64];
                tmem_ld_row(s_at, s);
                wait_row(s);
                tmem_ld_row(s_at + 64, t);               // on its way while the first half's maximum is found
                mask(s, 0);
                const float first = row_max(s);
                wait_row(t);
                mask(t, 1);
                const float second = row_max(t), top = max3(first, second, second) * scale;
                // Nothing to do where the maximum stays at or below m + kRoom (finite behind the first block); -inf and NaN come here, too.
                if (__any_sync(0xffffffffu, !(top <= m + kRoom<T> && top >= -FLT_MAX))) {
                    const bool up = !(top <= m + kRoom<T>) && top > -INFINITY;              // also where m is still -inf
                    const float under = up ? top - kUnder<T> : m, keep = up ? exp2_fast(m - under) : 1.f;
                    l *= keep;
                    m = under;
                    huge |= up && fabsf(top) > kHuge;
                    if (kb != begin && __any_sync(0xffffffffu, up)) {
#pragma unroll 1
                        for (uint32_t c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_at + c, o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st16(o_at + c, o);
                        }
                    }
                }
                const pair_t scales = pair_of(scale, scale);
                const float base = m == -INFINITY ? 0.f : -m;
                const pair_t bases = pair_of(base, base);
                pair_t sum[2] = {0, 0};
                // A quarter of the keys: exponentials, sums, P.  The first half is signalled in front of the third quarter's stores, when its own are long
                // done: waiting for them at once cost the row 100 cycles, and the products of the first half have time.
                auto weights = [&](const float (&s)[64], int quarter, auto before_stores) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int i = quarter % 2 * 32 + 2 * e;
                        float x, y;
                        parts_of(pair_fma(pair_of(s[i], s[i + 1]), scales, bases), x, y);
                        x = exp2_fast(x);
                        y = exp2_fast(y);
                        sum[e & 1] = pair_add(sum[e & 1], pair_of(x, y));
                        p[e] = pack<T>(x, y);
                    }
                    before_stores();
                    tmem_st16(s_at + 16 * quarter, p);
                };
                auto signal = [&](unsigned long long *bar) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                weights(s, 0, [] {});
                weights(s, 1, [] {});
                weights(t, 2, [&] { signal(&sh.p_half[tile]); });
                weights(t, 3, [] {});
                signal(&sh.p_full[tile]);
                float x, y;
                parts_of(pair_add(sum[0], sum[1]), x, y);
                l += x + y;
            }
            finish();
            if (tile * kTile < pairs) {
                // 128 bytes of eight rows at a time, turned so that a store covers whole lines of few rows: a thread storing its own row piece by piece
                // took 5000 cycles of a unit, 12000 where it is a part.
                const bool alone = g.first && g.last;
                const unsigned long long at = (unsigned long long)(g.row0 + token) * a.out_pitch + (unsigned long long)(g.head0 + head) * d;
                float *part = a.parts + (size_t)part_index(blockIdx.x, g) * kPrefillRows * (d + 2);
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const uint32_t first_row = tile * kTile + quad * 32 + (lane & 24u), piece = lane & 7u;
                bool bad = false;
#pragma unroll 1
                for (uint32_t c = 0; c < D; c += 32) {
                    float o[32];
                    if (stop > begin) {
                        tmem_ld32(o_at + c, o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e++) bad |= !(fabsf(o[e]) <= FLT_MAX);
                    if (alone) {                         // 64 bytes of a row, two such steps make a line
                        uint32_t v[8][4];
#pragma unroll
                        for (int e = 0; e < 16; e++) v[e / 4][e % 4] = pack<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
                        tmem_ld32(o_at + min(c + 32, (uint32_t)D - 32), o);
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            if (stop <= begin) o[e] = 0.f;
                            bad |= !(fabsf(o[e]) <= FLT_MAX);
                        }
#pragma unroll
                        for (int e = 0; e < 16; e++) v[4 + e / 4][e % 4] = pack<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
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
                bad = row < pairs && (huge || (bad && l == l));          // a NaN among the seen scores makes all of the row NaN, as it should be
                if (!alone && row < pairs) *reinterpret_cast<float2 *>(part + kPrefillRows * d + 2 * row) = make_float2(m, l);
                for (uint32_t left = __ballot_sync(0xffffffffu, bad); left; left &= left - 1) {
                    const uint32_t r = tile * kTile + quad * 32 + __ffs(left) - 1;
                    float rm, rl, acc[D / 64][8];
                    row_again<T, D>(a, sh, g, r, stop, rm, rl, acc);
                    const uint32_t tok = r / g.heads, hd = r - tok * g.heads;
                    __syncwarp();                        // behind the row's own stores
#pragma unroll
                    for (int c = 0; c < D / 64; c++) {
                        const uint32_t column = lane * 8 + 64 * c;
                        if (lane >= 8 || column >= d) continue;
                        if (alone) {
                            uint32_t v[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) v[e] = rl == 0.f ? 0u : pack<T>(acc[c][2 * e] / rl, acc[c][2 * e + 1] / rl);
                            *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + (size_t)(g.row0 + tok) * a.out_pitch + (size_t)(g.head0 + hd) * d + column) =
                                make_uint4(v[0], v[1], v[2], v[3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; e += 4)
                                *reinterpret_cast<float4 *>(part + r * d + column + e) = make_float4(acc[c][e], acc[c][e + 1], acc[c][e + 2], acc[c][e + 3]);
                        }
                    }
                    if (!alone && lane == 0) *reinterpret_cast<float2 *>(part + kPrefillRows * d + 2 * r) = make_float2(rm, rl);
                    __syncwarp();
                }
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
int launch_sized(const AttendArgs &a, const CacheMaps &maps, const CUtensorMap &q_map, cudaStream_t stream)
{
    auto *kernel = prefill_kernel<T, D>;
    if (int rc = allow_smem(kernel, smem_bytes<D>())) return rc;
    if (int rc = launch(kernel, dim3(kPrefillCtas), dim3(kThreads), smem_bytes<D>(), stream, maps, q_map, a)) return rc;
    return launch_merge<T, (int)kPrefillRows>(a, kPrefillCtas, kPrefillRows, stream);
}

// {head_dim, heads, rows} of the queries, for boxes of 64 elements by the heads of a key / value head by the tokens of a unit: as they lie in
// shared memory then, the pairs of token and head are the rows.
int encode_queries(CUtensorMap &map, int dtype, const AttendArgs &a)
{
    EncodeTiledFn encode = nullptr;
    if (int rc = encode_fn(encode)) return rc;
    const cuuint64_t dims[3] = {a.d, (cuuint64_t)a.kv_heads * a.group, a.rows};
    const cuuint64_t strides[2] = {(cuuint64_t)a.d * 2, (cuuint64_t)a.q_pitch * 2};
    const cuuint32_t box[3] = {64, a.group, kPrefillRows / a.group}, elem[3] = {1, 1, 1};
    const CUresult cr = encode(&map, dtype == MGQ_FMT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(a.q), dims, strides, box,
                               elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? MGQ_OK : fail(MGQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
}

}  // namespace

bool prefill_takes(const AttendArgs &a, int dtype)
{
    auto on = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    // scores are masked and compared before they are scaled: a scale of 0 would make -inf NaN, a negative one turn the order around
    return decode_takes(a, dtype) && a.d <= 128 && a.group <= kPrefillRows && a.scale_log2 >= 1e-30f && on(a.q) && on(a.out) && a.q_pitch % 8 == 0 && a.out_pitch % 8 == 0;
}

int launch_prefill(const AttendArgs &a, int dtype, cudaStream_t stream)
{
    CacheMaps maps;
    if (int rc = encode_caches(maps, dtype, a, min(1u << a.page_shift, kKeys))) return rc;
    CUtensorMap q_map;
    if (int rc = encode_queries(q_map, dtype, a)) return rc;
    if (dtype == MGQ_FMT_F16) return a.d <= 64 ? launch_sized<__half, 64>(a, maps, q_map, stream) : launch_sized<__half, 128>(a, maps, q_map, stream);
    return a.d <= 64 ? launch_sized<__nv_bfloat16, 64>(a, maps, q_map, stream) : launch_sized<__nv_bfloat16, 128>(a, maps, q_map, stream);
}

int prefill_status()
{
    unsigned int err = 0;
    MGQ_CUDA(cudaMemcpyFromSymbol(&err, g_prefill_error, sizeof err));
    if (!err) return MGQ_OK;
    const unsigned int zero = 0;
    MGQ_CUDA(cudaMemcpyToSymbol(g_prefill_error, &zero, sizeof zero));
    return fail(MGQ_ERR_TIMEOUT, "a bounded wait inside the paged attention of many tokens ran out");
}

}  // namespace mgq
