// Attention of many new tokens per sequence (portions of prompts, long drafts) over a paged cache of f16 or bf16, on tcgen05.
//
// A unit is 256 pairs of token and query head of one key / value head, two tiles of 128 rows that share the keys and values of a block
// of 128.  Per block and tile S = Q K^T and O += P V are four to eight products of K = 16 each way; the tensor cores need 512 cycles for either (heads of 128),
// and the exponentials of a tile, 16 per cycle on the SM, 1024: two tiles in turn keep both busy.
//   warps 0-7, 8-15 softmax of tile 0 and 1, two threads per row with 64 keys of a block each (one per row took 3200 cycles per block, most of them
//                   waiting for its own results): S from TMEM, running maximum and sum in f32, P back into TMEM over S (as the
//                   16-bit left operand of the second product); queries into shared memory, results out of TMEM.
//   warp 16         keys and values: TMA boxes of a page's tokens (128 at most) by 64 elements, a lane each, into a ring of stages that hold
//                   128 keys or 128 values.
//   warp 17         issues S(j + 1) of a tile right behind O(j) of the same tile: products run in order, so P is read before S overwrites it, and whoever sees
//                   S(j + 1) done knows that O(j) is.
// Sums are kept relative to a maximum that may be 2^8 too low: only where a row's maximum grows by more do its threads agree on a new one and scale O.  Weights are
// rounded to the values' type, as the tensor cores take both operands in one type; their sum is of the unrounded ones in f32.
// TMEM: S0, S1 (128 columns each, P in the first 32 of either half), O0, O1.
#include <cfloat>
#include <cstdint>

#include "mgq_paged.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 576;
constexpr int kExtra = 2;                                // blocks of keys that starting and ending a unit take as long as
constexpr uint32_t kKeys = 128, kTile = 128;             // keys of a block, rows of a tile
constexpr uint32_t kHalf = kKeys * 128;                  // 128 rows of 64 elements
template <int D> __host__ __device__ constexpr uint32_t stage_bytes() { return D / 64 * kHalf; }
template <int D> __host__ __device__ constexpr int stages() { return D == 64 ? 8 : 5; }

__device__ unsigned int g_prefill_error;

using Way = Walk<kPrefillRows, kKeys, kExtra>;
struct __align__(16) Shared {
    float top[2][2][kTile];                              // of a row's two threads: maximum, at the end sum of weights
    unsigned long long full[8], empty[8], q_full[2], s_full[2], p_full[2], o_full[2];
    Way way[4];                                          // of the tiles' warps, the producer, the issuer
    Segment seg[6];                                      // two of either tile's warps, then the producer's and the issuer's
    uint32_t there[8][4];                                // keys of a block that exist, for the last eight blocks
    uint32_t tmem;
    int more[2];
    volatile int failed;
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
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float x, float y, float z)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// (x, y) * s - b and (x, y) += (z, w), two elements per instruction.
__device__ __forceinline__ void scaled_pair(float &x, float &y, float s, float minus_b)
{
    asm("{\n\t.reg .b64 v, s, b;\n\t"
        "mov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %2};\n\tmov.b64 b, {%3, %3};\n\t"
        "fma.rn.f32x2 v, v, s, b;\n\t"
        "mov.b64 {%0, %1}, v;\n\t}" : "+f"(x), "+f"(y) : "f"(s), "f"(minus_b));
}
__device__ __forceinline__ void add_pair(float &x, float &y, float z, float w)
{
    asm("{\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "add.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}" : "+f"(x), "+f"(y) : "f"(z), "f"(w));
}
// 64 columns of this lane's row, one wait for all of them.
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float (&y)[64])
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
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 64; c++) asm volatile("" : "+f"(y[c]));     // nothing that uses them moves in front of the wait
}
// All 256 threads of a tile's warps: whether any of them says so.
__device__ __forceinline__ bool any_of_tile(uint32_t tile, bool mine)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
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

// Key blocks of one tile of a segment: [g.begin, what is returned).
__device__ __forceinline__ uint32_t tile_end(const Segment &g, uint32_t tile)
{
    const uint32_t pairs = g.tokens * g.heads;
    if (tile * kTile >= pairs) return g.begin;
    const int last = min(g.pos0 + (int)((min(pairs, (tile + 1) * kTile) - 1) / g.heads), g.len - 1);
    return last < 0 ? g.begin : max(g.begin, min(g.end, (uint32_t)last / kKeys + 1));
}

// One row of a segment again, on the CUDA cores and without what it does not see: where a value that only other rows see is infinite or NaN, its
// product with a weight of 0 has spoilt the row.  A whole warp; lane i has columns i, i + 32, ...
template <typename T, int D>
__device__ __noinline__ void row_again(const AttendArgs &a, const Segment &g, uint32_t r, uint32_t end, float &m, float &l, float (&acc)[D / 32])
{
    const uint32_t lane = threadIdx.x & 31u, token = r / g.heads, head = g.head0 + r - token * g.heads;
    const int pos = g.pos0 + (int)token;
    float q[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
        const uint32_t c = lane + 32 * i;
        q[i] = c < a.d ? to_f32(static_cast<const T *>(a.q)[(size_t)(g.row0 + token) * a.q_pitch + (size_t)head * a.d + c]) * a.scale_log2 : 0.f;
        acc[i] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    const int stop = min(min((int)(end * kKeys), pos + 1), g.len);
    for (int key = (int)(g.begin * kKeys); key < stop; key++) {
        if (a.window && key <= pos - (int)a.window) continue;
        const uint32_t page = g.table[(uint32_t)key >> a.page_shift];
        if (page >= a.pages) continue;
        const size_t at = ((((size_t)page << a.page_shift) + (key & ((1u << a.page_shift) - 1))) * a.kv_heads + g.kv) * a.d;
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
            if (lane + 32 * i < a.d) x = fmaf(q[i], to_f32(static_cast<const T *>(a.k)[at + lane + 32 * i]), x);
        x = warp_sum(x);
        const float top = fmaxf(m, x), base = top == -INFINITY ? 0.f : top, keep = exp2_fast(m - base), p = exp2_fast(x - base);
        l = l * keep + p;
        m = top;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
            if (lane + 32 * i < a.d) acc[i] = acc[i] * keep + (p != 0.f ? p * to_f32(static_cast<const T *>(a.v)[at + lane + 32 * i]) : 0.f);
    }
}

template <typename T, int D>                             // D: head size rounded up to 64 or 128
__global__ void __launch_bounds__(kThreads, 1) prefill_kernel(const __grid_constant__ CacheMaps maps, const AttendArgs a)
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
            mbar_init(&sh.empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.q_full[i], 8);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 8);
            mbar_init(&sh.o_full[i], 1);
        }
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t role = warp < 16 ? warp >> 3 : warp - 14;              // 0, 1: softmax of a tile, 2: producer, 3: issuer
    {
        Way way;
        way.begin(a, blockIdx.x, gridDim.x, 1, reinterpret_cast<unsigned long long *>(s_q));
        if (lane == 0 && (warp & 7u) == (role < 2 ? 0 : role - 2)) sh.way[role] = way;
    }
    if (tid == 0) clear_parts(a, blockIdx.x);
    __syncwarp();
    // The next segment of the producer or the issuer, if there is one.
    auto fetch = [&]() {
        int more = 0;
        if (lane == 0) more = sh.way[role].next(a, sh.seg[role + 2]);
        __syncwarp();
        return __shfl_sync(0xffffffffu, more, 0) != 0;
    };
    auto wait = [&](unsigned long long *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, &sh.failed, &g_prefill_error)) != 0; };

    if (role == 2) {
        const uint32_t shift = a.page_shift, page_keys = 1u << shift, box = min(page_keys, kKeys), boxes = kKeys / box, gone = a.pages << shift;
        uint32_t slot = 0, round = 0, block = 0;
        int armed = 0;
        bool ok = true;
        while (ok && fetch()) {
            const Segment &g = sh.seg[4];
            const int len = g.len, kv = (int)g.kv;
            const uint32_t *table = g.table;
            for (uint32_t kb = g.begin; ok && kb < g.end; kb++, block++) {
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
                    if (!(ok = wait(&sh.empty[slot], (round & 1u) ^ 1u))) break;
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
    } else if (role == 3) {
        const bool leader = elect_one();
        const uint32_t q16 = smem_u32(s_q) >> 4, ring16 = smem_u32(ring) >> 4;
        uint32_t slot = 0, round = 0, q_seen = 0, p_seen = 0;             // parities of the two tiles in bits 0 and 1
        bool ok = true;
        auto advance = [&]() {
            if (++slot == S) { slot = 0; round++; }
        };
        auto scores = [&](uint32_t tile, uint32_t at) {
            if (leader) {
                const uint32_t q = q16 + tile * (kStage / 16), k = ring16 + at * (kStage / 16);
                umma_step<false>(tmem + tile * 128, q, k, kInstrS);
#pragma unroll
                for (uint32_t i = 1; i < D / 16; i++) umma_step<true>(tmem + tile * 128, q + i / 4 * (kHalf / 16) + i % 4 * 2, k + i / 4 * (kHalf / 16) + i % 4 * 2, kInstrS);
                umma_commit(&sh.s_full[tile]);
            }
            __syncwarp();
        };
        auto values = [&](uint32_t tile, uint32_t at, bool first) {
            if (leader) {
                const uint32_t v = ring16 + at * (kStage / 16), o = tmem + 256 + tile * D, p = tmem + tile * 128;
#pragma unroll
                for (uint32_t i = 0; i < kKeys / 16; i++) umma_f16_ts_mn(o, p + i / 4 * 64 + i % 4 * 8, v + i * (2048 / 16), kHalf / 16, kInstrO, !first || i > 0);
            }
            __syncwarp();
        };
        while (ok && fetch()) {
            const Segment &g = sh.seg[5];
            const uint32_t begin = g.begin, end = g.end, stop[2] = {tile_end(g, 0), tile_end(g, 1)};
            if (end <= begin) continue;
            if (!(ok = wait(&sh.full[slot], round & 1u))) break;
            tc_fence_after();
#pragma unroll
            for (uint32_t tile = 0; tile < 2; tile++)
                if (ok && stop[tile] > begin) {
                    if (!(ok = wait(&sh.q_full[tile], q_seen >> tile & 1u))) break;
                    q_seen ^= 1u << tile;
                    tc_fence_after();
                    scores(tile, slot);
                }
            if (!ok) break;
            if (leader) umma_commit(&sh.empty[slot]);
            __syncwarp();
            advance();
            for (uint32_t kb = begin; ok && kb < end; kb++) {
                const uint32_t v_slot = slot;
                if (!(ok = wait(&sh.full[slot], round & 1u))) break;
                tc_fence_after();
                advance();
                const bool more = kb + 1 < end;
                bool waited = false;
#pragma unroll
                for (uint32_t tile = 0; tile < 2; tile++) {
                    if (stop[tile] > kb) {
                        if (!(ok = wait(&sh.p_full[tile], p_seen >> tile & 1u))) break;
                        p_seen ^= 1u << tile;
                        tc_fence_after();
                        values(tile, v_slot, kb == begin);
                        if (kb + 1 == stop[tile] && leader) umma_commit(&sh.o_full[tile]);
                        __syncwarp();
                    }
                    if (stop[tile] > kb + 1) {
                        if (!waited) {
                            if (!(ok = wait(&sh.full[slot], round & 1u))) break;
                            tc_fence_after();
                            waited = true;
                        }
                        scores(tile, slot);
                    }
                }
                if (!ok) break;
                if (leader) umma_commit(&sh.empty[v_slot]);
                if (more) {
                    if (!waited && !(ok = wait(&sh.full[slot], round & 1u))) break;
                    if (leader) umma_commit(&sh.empty[slot]);
                    advance();
                }
                __syncwarp();
            }
        }
    } else {
        // thread = row of the tile and half of a block's keys, of O's columns, of the query's pieces
        const uint32_t tile = role, half = warp >> 2 & 1u, quad = warp & 3u, r_tile = quad * 32 + lane, row = tile * kTile + r_tile;
        const uint32_t lanes = (quad * 32u) << 16, s_at = tmem + tile * 128 + half * 64 + lanes, o_at = tmem + 256 + tile * D + half * (D / 2) + lanes, d = a.d;
        const float scale = fabsf(a.scale_log2);
        const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;      // a negative scale turns the queries' signs
        uint32_t slot = 0, round = 0, block = 0;         // of the ring, as the producer counts
        uint32_t s_seen = 0, o_seen = 0, turn = 0;
        bool ok = true;
        // the tile's next segment: one thread looks for it, all meet
        auto fetch_tile = [&]() {
            if (half == 0 && r_tile == 0) sh.more[tile] = sh.way[tile].next(a, sh.seg[2 * tile + (turn & 1u)]);
            turn++;
            any_of_tile(tile, false);
            return sh.more[tile] != 0;
        };
        // this thread's half of a query into the swizzled tile; heads beyond d and rows behind the last pair are zero
        auto load_q = [&](const Segment &g) {
            if (tile_end(g, tile) <= g.begin) return;
            const uint32_t token = row / g.heads, head = row - token * g.heads;
            const bool live = row < g.tokens * g.heads;
            const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (size_t)(g.row0 + (live ? token : 0)) * a.q_pitch + (size_t)(g.head0 + head) * d);
#pragma unroll
            for (uint32_t i = 0; i < D / 16; i++) {
                const uint32_t c = half * (D / 16) + i;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (live && c * 8 < d) v = src[c];
                v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
                *reinterpret_cast<uint4 *>(s_q + tile * kStage + c / 8 * kHalf + r_tile * 128 + ((c % 8) ^ (r_tile & 7u)) * 16) = v;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[tile]);
        };
        // A wait that runs out is noted and carried to the next meeting of the tile's warps, where all of them leave.
        bool live_seg = fetch_tile();
        if (live_seg) load_q(sh.seg[2 * tile]);
        while (live_seg) {
            const Segment &g = sh.seg[2 * tile + ((turn - 1) & 1u)];
            const uint32_t begin = g.begin, end = g.end, stop = tile_end(g, tile), pairs = g.tokens * g.heads;
            const int pos = row < pairs ? g.pos0 + (int)(row / g.heads) : -1, first_pos = g.pos0 + (int)(tile * kTile / g.heads);
            const int last_pos = g.pos0 + (int)((min(pairs, (tile + 1) * kTile) - 1) / g.heads), window = (int)a.window;
            float m = -INFINITY, l = 0.f;
            for (uint32_t kb = begin; kb < end; kb++, block++) {
                if (++slot == S) { slot = 0; round++; }
                const uint32_t v_slot = slot, v_round = round;
                if (++slot == S) { slot = 0; round++; }
                if (kb >= stop) continue;
                ok = wait(&sh.s_full[tile], s_seen & 1u);
                s_seen++;
                tc_fence_after();
                // For sight of `there`, and to write into the values below.  Not the keys' barrier: their stage is free by now and may have been filled
                // again, two phases on, where this parity would wait for a third.  The values' stage is free behind this tile's product only.
                ok = wait(&sh.full[v_slot], v_round & 1u) && ok;
                uint32_t there[4];
#pragma unroll
                for (int w = 0; w < 4; w++) there[w] = sh.there[block & 7u][w];
                float s[64];
                tmem_ld64(s_at, s);
                const int key0 = (int)(kb * kKeys);
                const bool every = (there[0] & there[1] & there[2] & there[3]) == 0xFFFFFFFFu;
                if (!every || key0 + (int)kKeys - 1 > first_pos || (window && key0 <= last_pos - window)) {
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const uint32_t seen = (half ? there[2 + w] : there[w]) & bits(window ? pos - window + 1 : 0, pos + 1, key0 + 64 * (int)half + 32 * w);
#pragma unroll
                        for (int e = 0; e < 32; e++) s[32 * w + e] = seen >> e & 1u ? s[32 * w + e] : -INFINITY;
                    }
                }
                float tops[4];
#pragma unroll
                for (int i = 0; i < 4; i++) tops[i] = max3(s[i], s[4 + i], s[8 + i]);
#pragma unroll
                for (int e = 12; e < 60; e += 8)
#pragma unroll
                    for (int i = 0; i < 4; i++) tops[i] = max3(tops[i], s[e + i], s[e + 4 + i]);
                float top = fmaxf(max3(tops[0], tops[1], s[60]), max3(max3(tops[2], tops[3], s[61]), s[62], s[63])) * scale;
                if (any_of_tile(tile, !ok || (!(top <= m + 8.f) && top > -INFINITY))) {
                    sh.top[tile][half][r_tile] = top;
                    if (any_of_tile(tile, !ok)) {
                        ok = false;
                        break;
                    }
                    top = fmaxf(top, sh.top[tile][half ^ 1u][r_tile]);
                    const bool up = !(top <= m + 8.f) && top > -INFINITY;             // also where m is still -inf
                    const float keep = up ? exp2_fast(m - top) : 1.f;
                    l *= keep;
                    m = up ? top : m;
                    if (kb != begin && __any_sync(0xffffffffu, up)) {
#pragma unroll 1
                        for (uint32_t c = 0; c < D / 2; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_at + c, o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st16(o_at + c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        float x = s[32 * c + 2 * e], y = s[32 * c + 2 * e + 1];
                        scaled_pair(x, y, scale, -base);
                        x = exp2_fast(x);
                        y = exp2_fast(y);
                        add_pair(sum[e % 2 * 2], sum[e % 2 * 2 + 1], x, y);
                        p[e] = pack<T>(x, y);
                    }
                    tmem_st16(s_at + 16 * c, p);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (!every) {                            // values that nobody sees, whatever the page holds there, become zeros
                    uint8_t *v = ring + v_slot * kStage;
                    for (uint32_t i = half * 128 + r_tile; i < kKeys * PARTS * 8; i += 256) {
                        const uint32_t key = i / 8 % kKeys, w = key / 32, word = w == 0 ? there[0] : w == 1 ? there[1] : w == 2 ? there[2] : there[3];
                        if (!(word >> (key % 32) & 1u)) *reinterpret_cast<uint4 *>(v + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[tile]);
            }
            if (!ok) break;
            // the next unit's queries, while the last product runs: the scores of this one are done with them
            const bool more = fetch_tile();
            if (more) load_q(sh.seg[2 * tile + ((turn - 1) & 1u)]);
            if (stop > begin) {
                ok = wait(&sh.o_full[tile], o_seen & 1u);
                o_seen++;
                tc_fence_after();
            }
            sh.top[tile][half][r_tile] = l;
            if (any_of_tile(tile, !ok)) {
                ok = false;
                break;
            }
            l += sh.top[tile][half ^ 1u][r_tile];
            if (tile * kTile < pairs) {
                const bool alone = g.first && g.last;
                const uint32_t token = row / g.heads, head = row - token * g.heads, c0 = half * (D / 2);
                T *out = static_cast<T *>(a.out) + (size_t)(g.row0 + token) * a.out_pitch + (size_t)(g.head0 + head) * d + c0;
                float *part = a.parts + (size_t)part_index(blockIdx.x, g) * kPrefillRows * (d + 2);
                const float inv = l == 0.f ? 0.f : 1.f / l;
                bool bad = false;
#pragma unroll 1
                for (uint32_t c = 0; c < D / 2; c += 16) {
                    uint32_t b[16];
                    if (stop > begin) {
                        tmem_ld16(o_at + c, b);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) b[e] = 0u;
                    }
                    if (row < pairs) {
#pragma unroll
                        for (int e = 0; e < 16; e += 8) {
                            if (c0 + c + e >= d) break;
                            float o[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                o[i] = __uint_as_float(b[e + i]);
                                bad |= !(fabsf(o[i]) <= FLT_MAX);
                            }
                            if (alone) {
                                *reinterpret_cast<uint4 *>(out + c + e) =
                                    make_uint4(pack<T>(o[0] * inv, o[1] * inv), pack<T>(o[2] * inv, o[3] * inv), pack<T>(o[4] * inv, o[5] * inv), pack<T>(o[6] * inv, o[7] * inv));
                            } else {
                                *reinterpret_cast<float4 *>(part + row * d + c0 + c + e) = make_float4(o[0], o[1], o[2], o[3]);
                                *reinterpret_cast<float4 *>(part + row * d + c0 + c + e + 4) = make_float4(o[4], o[5], o[6], o[7]);
                            }
                        }
                    }
                    __syncwarp();                        // the next columns are read by the whole warp
                }
                if (!alone && half == 0 && row < pairs) *reinterpret_cast<float2 *>(part + kPrefillRows * d + 2 * row) = make_float2(m, l);
                // a row that either thread finds spoilt is computed again by the first one's warp, behind both threads' stores
                if (any_of_tile(tile, bad)) {
                    sh.top[tile][half][r_tile] = bad ? 1.f : 0.f;
                    any_of_tile(tile, false);
                    const bool redo = half == 0 && (sh.top[tile][0][r_tile] != 0.f || sh.top[tile][1][r_tile] != 0.f);
                    for (uint32_t left = __ballot_sync(0xffffffffu, redo); left; left &= left - 1) {
                        const uint32_t r = tile * kTile + quad * 32 + __ffs(left) - 1;
                        float rm, rl, acc[D / 32];
                        row_again<T, D>(a, g, r, stop, rm, rl, acc);
                        const uint32_t tok = r / g.heads, hd = r - tok * g.heads;
#pragma unroll
                        for (int i = 0; i < D / 32; i++) {
                            const uint32_t c = lane + 32 * i;
                            if (c >= d) continue;
                            if (alone) static_cast<T *>(a.out)[(size_t)(g.row0 + tok) * a.out_pitch + (size_t)(g.head0 + hd) * d + c] = rounded<T>(rl == 0.f ? 0.f : acc[i] / rl);
                            else       part[r * d + c] = acc[i];
                        }
                        if (!alone && lane == 0) *reinterpret_cast<float2 *>(part + kPrefillRows * d + 2 * r) = make_float2(rm, rl);
                    }
                }
                if (!alone && tid == 0) name_part(a, blockIdx.x, g);
            }
            any_of_tile(tile, false);                    // sums read, before the next unit's maxima
            tc_fence_before();
            __syncwarp();
            live_seg = more;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        __syncwarp();
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

template <typename T, int D>
int launch_sized(const AttendArgs &a, const CacheMaps &maps, cudaStream_t stream)
{
    auto *kernel = prefill_kernel<T, D>;
    if (int rc = allow_smem(kernel, smem_bytes<D>())) return rc;
    if (int rc = launch(kernel, dim3(kPrefillCtas), dim3(kThreads), smem_bytes<D>(), stream, maps, a)) return rc;
    return launch(merge_kernel<T, (int)kPrefillRows>, dim3(kPrefillCtas, 16), dim3(kMergeThreads), 0, stream, a, kPrefillCtas);
}

}  // namespace

bool prefill_takes(const AttendArgs &a, int dtype)
{
    auto on = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    // masked scores are -inf before they are scaled: a scale of 0 would make them NaN
    return decode_takes(a, dtype) && a.d <= 128 && fabsf(a.scale_log2) >= 1e-30f && on(a.q) && on(a.out) && a.q_pitch % 8 == 0 && a.out_pitch % 8 == 0;
}

int launch_prefill(const AttendArgs &a, int dtype, cudaStream_t stream)
{
    CacheMaps maps;
    if (int rc = encode_caches(maps, dtype, a, min(1u << a.page_shift, kKeys))) return rc;
    if (dtype == MGQ_FMT_F16) return a.d <= 64 ? launch_sized<__half, 64>(a, maps, stream) : launch_sized<__half, 128>(a, maps, stream);
    return a.d <= 64 ? launch_sized<__nv_bfloat16, 64>(a, maps, stream) : launch_sized<__nv_bfloat16, 128>(a, maps, stream);
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
