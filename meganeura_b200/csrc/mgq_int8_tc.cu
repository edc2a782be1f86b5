// Products of rows of 8-bit codes on tcgen05: out[m, n] = (sum over k of a[m, k] w[n, k]) a_scales[m] w_scales[n] (+ addend[m, n]).
//
// The weight rows are the products' rows (TMEM lanes), the activation rows their columns: a thread of the epilogue has one weight row and its scale, a store
// covers 32 consecutive columns of an output row, and few activation rows cost as few columns.  Sums are whole numbers in 32 bits, exact and free of order.
// Both operands lie k-major in the 128-byte swizzle: 128 k per stage, four products of 32.
//
// pair_kernel: many tiles.  Two CTAs of a cluster share tiles of 256 weight rows by `tn` activation rows (cta_group::2): each holds its 128 weight rows and half of
// the activation rows, and has its 128 rows' sums in its TMEM.  One CTA's copies would fill and feed its shared memory at 192 bytes per cycle with 128 x 256
// tiles, a pair needs 128.  Persistent, one accumulator is read while the other is filled.
// 2048 x 4096 by 12288 columns: 69 to 82 us, 2.5 to 3.0 POP/s.  Power bounds it: codes of all the range hold the clock at 1.26 to 1.45 of 1.97 GHz, and 8192 cubed
// takes 340 to 390 us (2.8 to 3.2 POP/s); with operands of zeros the same instructions take 250 (4.40), as fast as products alone out of shared memory (4.33).  So stages of 256 k, tiles of
// 256 x 512, which read a quarter less from L2 (405 us), and smaller tiles for the last round gave nothing.
//   warp 0      TMA of this CTA's boxes, completing on full[s] of the pair's first CTA
//   warp 1      (first CTA) issues the products, and gives stages and accumulators to both CTAs
//   warps 2-9   epilogue: 32 rows by every other 32 columns each
// split_kernel: few tiles.  A cluster shares out the k of a tile of 128 by `tn`; sums meet through distributed shared memory, each CTA finishing its part of
// the columns.  Two CTAs per SM.
#include "mgq_int8.cuh"
#include "mgq_tcgen05.cuh"

namespace mgq {
namespace {

constexpr uint32_t kRows = 128, kChunk = 128;            // weight rows of a CTA's tile, k of a stage
constexpr uint32_t kBytesW = kRows * kChunk;
constexpr uint32_t kMostCols = 256;
constexpr int kPairThreads = 320, kPairStages = 6, kSplitThreads = 256;
constexpr uint32_t kPairStage = kBytesW + kMostCols / 2 * kChunk;
constexpr uint32_t kMostSplit = 8;

__device__ unsigned int g_int8_error;

struct Maps {
    CUtensorMap w, a;
};

// kind::i8: D s32, A and B signed 8-bit, both K-major.
__host__ __device__ constexpr uint32_t instr_i8(uint32_t m, uint32_t n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }

template <int GROUP>
__device__ __forceinline__ void mma_i8(uint32_t d, uint32_t a16, uint32_t b16, uint32_t instr, bool accumulate)
{
    if constexpr (GROUP == 2)
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
                     "setp.ne.b32 p, %5, 0;\n\t"
                     "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
                     "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, p;\n\t}"
                     ::"r"(d), "r"(a16 | 0x10000u), "r"(b16 | 0x10000u), "r"(instr), "r"(kDescHigh), "r"((uint32_t)accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
                     "setp.ne.b32 p, %5, 0;\n\t"
                     "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
                     "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n\t}"
                     ::"r"(d), "r"(a16 | 0x10000u), "r"(b16 | 0x10000u), "r"(instr), "r"(kDescHigh), "r"((uint32_t)accumulate) : "memory");
}
// The products issued so far are done: arrives on this barrier in both CTAs of the pair.
__device__ __forceinline__ void commit_pair(unsigned long long *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
// The same variable in another CTA of the cluster.
__device__ __forceinline__ uint32_t cluster_address(const void *p, uint32_t rank)
{
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
    return addr;
}
__device__ __forceinline__ void load_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void prefetch_box(const CUtensorMap *map, int x, int y)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// C columns of this thread's weight row n: `count` activation rows from m0 on.  All values are ready before the first is stored, so that nothing waits in
// between: element by element the warps took 360 cycles a column, three times as long as the products of a 256 x 256 tile with k = 4096.
template <typename T, int C>
__device__ __forceinline__ void finish_columns(const ProductArgs &a, uint32_t m0, uint32_t n, const int (&sum)[C], float w_scale, uint32_t count)
{
    const uint32_t lane = threadIdx.x & 31u;
    const float scales = lane < count ? a.a_scales[m0 + lane] : 0.f;
    const bool live = n < a.n;
    float y[C];
#pragma unroll
    for (int e = 0; e < C; e++) y[e] = (float)sum[e] * __shfl_sync(0xffffffffu, scales, e) * w_scale;
    if (a.addend) {
        const T *p = static_cast<const T *>(a.addend) + (size_t)m0 * a.addend_pitch + n;
        constexpr int B = C < 16 ? C : 16;
#pragma unroll
        for (int b = 0; b < C; b += B) {
            T add[B];
#pragma unroll
            for (int e = 0; e < B; e++)
                if (live && (uint32_t)(b + e) < count) add[e] = p[(size_t)(b + e) * a.addend_pitch];
#pragma unroll
            for (int e = 0; e < B; e++)
                if (live && (uint32_t)(b + e) < count) y[b + e] += to_f32(add[e]);
        }
    }
    T *p = static_cast<T *>(a.out) + (size_t)m0 * a.out_pitch + n;
    if (!live) return;
    if (count == C) {
#pragma unroll
        for (int e = 0; e < C; e++, p += a.out_pitch) *p = to_type<T>(y[e]);
    } else {
#pragma unroll
        for (int e = 0; e < C; e++, p += a.out_pitch)
            if ((uint32_t)e < count) *p = to_type<T>(y[e]);
    }
}
__device__ __forceinline__ int load_cluster(uint32_t addr)
{
    int v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void load32(uint32_t addr, int (&v)[32])
{
    float f[32];
    tmem_ld32(addr, f);
#pragma unroll
    for (int e = 0; e < 32; e++) v[e] = __float_as_int(f[e]);
}

// ---------------------------------------------------------------- many tiles
struct PairShared {
    unsigned long long full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2];
    uint32_t tmem;
    volatile int failed;
};

// Tiles of eight blocks of columns one behind another, then the next weight rows: what runs at the same time reads few different rows of either.
__device__ __forceinline__ void place(uint32_t tile, uint32_t m_tiles, uint32_t n_tiles, uint32_t &nt, uint32_t &mt)
{
    const uint32_t band = tile / (8 * n_tiles), wide = min(m_tiles - 8 * band, 8u), at = tile - band * 8 * n_tiles;
    nt = at / wide;
    mt = 8 * band + at - nt * wide;
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1) pair_kernel(const __grid_constant__ Maps maps, const ProductArgs a, uint32_t tn)
{
    constexpr int S = kPairStages;
    extern __shared__ uint8_t s_raw[];
    __shared__ PairShared sh;
    // the same offset in both CTAs
    const uint32_t ring = (smem_u32(s_raw) + 1023) & ~1023u;
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u, rank = blockIdx.x & 1u, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t m_tiles = (a.m + tn - 1) / tn, n_tiles = (a.n + 2 * kRows - 1) / (2 * kRows), tiles = n_tiles * m_tiles, chunks = (a.k + kChunk - 1) / kChunk;
    if (tid == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&sh.acc_full[b], 1);
            mbar_init(&sh.acc_empty[b], 16);             // the epilogue warps of both CTAs
        }
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    pdl_launch_dependents();
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t bytes_a = tn / 2 * kChunk;
            uint32_t slot = 0, round = 0, armed = 0;
            bool ok = true;
            for (uint32_t tile = pair; tile < tiles && ok; tile += pairs) {
                uint32_t nt, mt;
                place(tile, m_tiles, n_tiles, nt, mt);
                const int n0 = (int)(nt * 2 * kRows + rank * kRows), m0 = (int)(mt * tn + rank * (tn / 2));
                for (uint32_t c = 0; c < chunks; c++) {
                    if (!(ok = mbar_wait(&sh.empty[slot], (round & 1u) ^ 1u, &sh.failed, &g_int8_error))) break;
                    const uint32_t bar = cluster_address(&sh.full[slot], 0), dst = ring + slot * kPairStage;
                    if (rank == 0) mbar_arrive_expect_tx(&sh.full[slot], 2 * (kBytesW + bytes_a));      // of both CTAs
                    load_pair(dst, &maps.w, (int)(c * kChunk), n0, bar);
                    load_pair(dst + kBytesW, &maps.a, (int)(c * kChunk), m0, bar);
                    armed++;
                    if (++slot == S) { slot = 0; round++; }
                }
            }
            // given up: the copies in flight land before the CTAs exit
            if (!ok && rank == 0)
                for (uint32_t i = 0; i < min(armed, (uint32_t)S); i++) {
                    if (slot-- == 0) { slot = S - 1; round--; }
                    for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&sh.full[slot], round & 1u); w++) { }
                }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint32_t ring16 = ring >> 4, instr = instr_i8(2 * kRows, tn);
            uint32_t slot = 0, round = 0, at = 0;
            bool ok = true;
            for (uint32_t tile = pair; tile < tiles && ok; tile += pairs, at++) {
                const uint32_t b = at & 1u, acc = tmem + b * kMostCols;
                if (!(ok = mbar_wait(&sh.acc_empty[b], ((at >> 1) & 1u) ^ 1u, &sh.failed, &g_int8_error))) break;
                tc_fence_after();
                for (uint32_t c = 0; c < chunks; c++) {
                    if (!(ok = mbar_wait(&sh.full[slot], round & 1u, &sh.failed, &g_int8_error))) break;
                    tc_fence_after();
                    const uint32_t w = ring16 + slot * (kPairStage / 16), x = w + kBytesW / 16;
#pragma unroll
                    for (uint32_t j = 0; j < kChunk / 32; j++) mma_i8<2>(acc, w + 2 * j, x + 2 * j, instr, c > 0 || j > 0);
                    commit_pair(&sh.empty[slot]);
                    if (++slot == S) { slot = 0; round++; }
                }
                if (ok) commit_pair(&sh.acc_full[b]);
            }
        }
        __syncwarp();
    } else {
        const uint32_t quad = warp & 3u, half = (warp - 2) / 4;
        uint32_t at = 0;
        for (uint32_t tile = pair; tile < tiles; tile += pairs, at++) {
            uint32_t nt, mt;
            place(tile, m_tiles, n_tiles, nt, mt);
            const uint32_t b = at & 1u, m0 = mt * tn;
            const bool ok = mbar_wait(&sh.acc_full[b], (at >> 1) & 1u, &sh.failed, &g_int8_error);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint32_t n = nt * 2 * kRows + rank * kRows + quad * 32 + lane, acc = tmem + ((quad * 32u) << 16) + b * kMostCols;
            const float w_scale = n < a.n ? a.w_scales[n] : 0.f;
#pragma unroll 1
            for (uint32_t c0 = half * 32; c0 < tn && m0 + c0 < a.m; c0 += 64) {
                int sum[32];
                load32(acc + c0, sum);
                finish_columns<T, 32>(a, m0 + c0, n, sum, w_scale, min(min(tn - c0, 32u), a.m - m0 - c0));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_cluster(cluster_address(&sh.acc_empty[b], 0));
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // the pair's copies, products and arrivals have landed
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------- few tiles
struct SplitShared {
    unsigned long long full[8], empty[8], done;
    uint32_t tmem;
    volatile int failed;
};

// Columns [first, last) of a tile, C at a time: their loads from all CTAs first, as each takes longer than what follows.
template <typename T, int C>
__device__ __forceinline__ void gather(const ProductArgs &a, const int *sums, uint32_t split, uint32_t first, uint32_t last, uint32_t m0, uint32_t n, float w_scale)
{
    const uint32_t row = (threadIdx.x / 32 % 4) * 32 + threadIdx.x % 32;
    for (uint32_t c0 = first; c0 < last; c0 += C) {
        int sum[C] = {};
#pragma unroll
        for (uint32_t r = 0; r < kMostSplit; r++) {
            if (r >= split) break;
            const uint32_t from = cluster_address(&sums[c0 * kRows + row], r);
#pragma unroll
            for (int e = 0; e < C; e++) sum[e] += c0 + e < last ? load_cluster(from + e * kRows * 4) : 0;
        }
        finish_columns<T, C>(a, m0 + c0, n, sum, w_scale, min(last - c0, (uint32_t)C));
    }
}

template <typename T>
__global__ void __launch_bounds__(kSplitThreads, 2) split_kernel(const __grid_constant__ Maps maps, const ProductArgs a, uint32_t tn, uint32_t split, uint32_t stages, uint32_t columns)
{
    extern __shared__ uint8_t s_raw[];
    __shared__ SplitShared sh;
    uint8_t *mem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t ring = smem_u32(mem), tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
    const uint32_t rank = blockIdx.y % split, m0 = blockIdx.y / split * tn, n0 = blockIdx.x * kRows, all = (a.k + kChunk - 1) / kChunk;
    const uint32_t from = all * rank / split, to = all * (rank + 1) / split, stage = kBytesW + tn * kChunk;
    if (tid == 0) {
        for (uint32_t s = 0; s < stages; s++) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
            if (from + s < to) prefetch_box(&maps.w, (int)((from + s) * kChunk), (int)n0);      // L2 holds what the kernels in front write
        }
        mbar_init(&sh.done, 1);
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(&sh.tmem, columns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    pdl_launch_dependents();
    pdl_wait();
    if (warp == 0 && lane == 0) {
        uint32_t slot = 0, round = 0, armed = 0;
        bool ok = true;
        for (uint32_t c = from; c < to; c++) {
            if (!(ok = mbar_wait(&sh.empty[slot], (round & 1u) ^ 1u, &sh.failed, &g_int8_error))) break;
            mbar_arrive_expect_tx(&sh.full[slot], stage);
            tma_load_2d(mem + slot * stage, &maps.w, (int)(c * kChunk), (int)n0, &sh.full[slot]);
            tma_load_2d(mem + slot * stage + kBytesW, &maps.a, (int)(c * kChunk), (int)m0, &sh.full[slot]);
            armed++;
            if (++slot == stages) { slot = 0; round++; }
        }
        if (!ok)                                         // given up: the copies in flight land before the CTA exits
            for (uint32_t i = 0; i < min(armed, stages); i++) {
                if (slot-- == 0) { slot = stages - 1; round--; }
                for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&sh.full[slot], round & 1u); w++) { }
            }
    }
    if (warp == 1 && elect_one()) {
        const uint32_t instr = instr_i8(kRows, tn);
        uint32_t slot = 0, round = 0;
        bool ok = true;
        for (uint32_t c = from; c < to; c++) {
            if (!(ok = mbar_wait(&sh.full[slot], round & 1u, &sh.failed, &g_int8_error))) break;
            tc_fence_after();
            const uint32_t w = (ring + slot * stage) >> 4, x = w + kBytesW / 16;
#pragma unroll
            for (uint32_t j = 0; j < kChunk / 32; j++) mma_i8<1>(tmem, w + 2 * j, x + 2 * j, instr, c > from || j > 0);
            umma_commit(&sh.empty[slot]);
            if (++slot == stages) { slot = 0; round++; }
        }
        if (ok) umma_commit(&sh.done);
    }
    __syncwarp();
    const bool ok = __syncthreads_and(mbar_wait(&sh.done, 0, &sh.failed, &g_int8_error));      // behind it the ring is free
    tc_fence_after();
    const uint32_t quad = warp & 3u, half = warp / 4, row = quad * 32 + lane, n = n0 + row, acc = tmem + ((quad * 32u) << 16);
    const float w_scale = n < a.n ? a.w_scales[n] : 0.f;
    if (split == 1) {
        for (uint32_t c0 = half * 32; ok && c0 < tn && m0 + c0 < a.m; c0 += 64) {
            int sum[32];
            load32(acc + c0, sum);
            finish_columns<T, 32>(a, m0 + c0, n, sum, w_scale, min(min(tn - c0, 32u), a.m - m0 - c0));
        }
    } else {
        int *sums = reinterpret_cast<int *>(mem);        // [tn rounded up to 32][128]
        for (uint32_t c0 = half * 32; c0 < tn; c0 += 64) {
            int sum[32];
            load32(acc + c0, sum);
#pragma unroll
            for (int e = 0; e < 32; e++) sums[(c0 + e) * kRows + row] = sum[e];
        }
        cluster_sync();
        // a half's share of the columns
        const uint32_t share = (tn + 2 * split - 1) / (2 * split), first = min((2 * rank + half) * share, tn), last = min(min(first + share, tn), a.m - m0);
        if (ok && share <= 2) gather<T, 2>(a, sums, split, first, last, m0, n, w_scale);
        else if (ok)          gather<T, 8>(a, sums, split, first, last, m0, n, w_scale);
        cluster_sync();                                  // the others have read this CTA's sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(tmem, columns);
    }
}

int encode(CUtensorMap &map, const int8_t *base, uint32_t k, uint32_t rows, uint32_t box_rows)
{
    EncodeTiledFn fn = nullptr;
    if (int rc = encode_fn(fn)) return rc;
    const cuuint64_t dims[2] = {k, rows}, strides[1] = {k};
    const cuuint32_t box[2] = {kChunk, box_rows}, elem[2] = {1, 1};
    const CUresult cr = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? MGQ_OK : fail(MGQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)cr);
}

constexpr uint32_t kPairs = 74, kMostCtas = 296;          // one and two per SM

template <typename T>
int launch_pair(const ProductArgs &a, uint32_t tn, cudaStream_t stream)
{
    Maps maps;
    if (int rc = encode(maps.w, a.w, a.k, a.n, kRows)) return rc;
    if (int rc = encode(maps.a, a.a, a.k, a.m, tn / 2)) return rc;
    const size_t smem = 1024 + (size_t)kPairStages * kPairStage;
    if (int rc = allow_smem(pair_kernel<T>, smem)) return rc;
    return launch_clusters(pair_kernel<T>, dim3(2 * kPairs), dim3(kPairThreads), dim3(2), smem,      // along x: a pair along y is refused
                           stream, maps, a, tn);
}

template <typename T>
int launch_split(const ProductArgs &a, uint32_t tn, uint32_t split, cudaStream_t stream)
{
    Maps maps;
    if (int rc = encode(maps.w, a.w, a.k, a.n, kRows)) return rc;
    if (int rc = encode(maps.a, a.a, a.k, a.m, tn)) return rc;
    const uint32_t stage = kBytesW + tn * kChunk, stages = min(max((104u * 1024) / stage, 2u), 8u);
    uint32_t columns = 32;
    while (columns < tn) columns *= 2;
    const size_t smem = 1024 + max((size_t)stages * stage, split > 1 ? (size_t)((tn + 31) / 32 * 32) * kRows * 4 : 0);
    if (int rc = allow_smem(split_kernel<T>, smem)) return rc;
    return launch_clustered(split_kernel<T>, dim3((a.n + kRows - 1) / kRows, (a.m + tn - 1) / tn * split), dim3(kSplitThreads), split, smem, stream, maps, a, tn, split, stages,
                            columns);
}

template <typename T>
int launch_typed(const ProductArgs &a, cudaStream_t stream)
{
    const uint32_t n_tiles = (a.n + kRows - 1) / kRows, chunks = (a.k + kChunk - 1) / kChunk;
    // Few tiles: narrow ones, and a cluster for each that shares out a long k, as long as all run at once, two CTAs to an SM (in clusters 264 or so find room, of eight 256).
    // Beyond that, and for many rows where wide tiles or a long k make reads from L2 count, pairs.  Some 1600 shapes of 9 to 2048 rows, k of 128 to 12288 and 100 to 24576
    // columns were timed with all widths and splits; with these bounds they take 1 % longer than with the best for each.  256 x 576 x 1536 with 32, 64, 128 columns
    // 3.7, 3.8, 4.7 us; 200 x 4096 x 576 with 32 columns by 8, 4, 2 CTAs 10.7 (more than fit at once), 6.1, 7.8; 256 x 12288 x 100 by 8, 4 7.2, 8.9, with 128 columns by 4 13.3;
    // 512 x 256 x 8192 with 128 columns 5.2, in pairs 7.2; 512 x 2560 x 8192 12.5, 12.8, 512 x 8192 x 8192 31.8, 28.3.  Rows that begin in the middle of 32 bytes cost more
    // reads: 355 x 1024 x 11008 with 128 columns 7.9, in pairs 9.5, of k = 1040 13.1 and 10.9.
    const uint32_t least = a.m <= 16 ? 16 : 32, most = min(a.m <= 64 ? max((a.m + 15) / 16 * 16, least) : (a.m + 31) / 32 * 32, kMostCols), few_chunks = a.k % 32 ? 4 : 12;
    auto ctas = [&](uint32_t tn) { return (unsigned long long)n_tiles * ((a.m + tn - 1) / tn); };
    for (uint32_t split = kMostSplit; split > 1; split /= 2) {
        if (chunks < (split == 4 ? 16 : 32)) continue;
        const uint32_t widest = min(most, split == 8 || chunks < 40 ? 32u : split == 4 ? 128u : 96u);
        for (uint32_t tn = least; tn <= widest; tn += tn < 64 ? 16 : 32)
            if (ctas(tn) * split <= (split == 8 ? 256 : 264)) return launch_split<T>(a, tn, split, stream);
    }
    for (uint32_t tn = least; tn <= (a.m <= 256 ? most : kMostCols / 2); tn += tn < 64 ? 16 : 32)
        if (ctas(tn) <= kMostCtas && (tn <= 64 || a.m <= 256 || chunks <= few_chunks) && (a.m < 96 || chunks < 40)) return launch_split<T>(a, tn, 1, stream);
    // The columns of a tile with the shortest rounds of tiles, which take as long as tn + 64 columns: 2048 x 12288 x 4096 with 128, 160, 192, 224, 256 took 101, 86, 95, 98,
    // 79 us, 300 x 4096 x 24576 47, 40, 42, 42, 44.
    uint32_t best = kMostCols, cost = 0xFFFFFFFFu;
    for (uint32_t cols = kMostCols; cols >= min(max((a.m + 31) / 32 * 32, 64u), 128u); cols -= 32) {
        const uint32_t tiles = (a.m + cols - 1) / cols * ((a.n + 2 * kRows - 1) / (2 * kRows)), c = (tiles + kPairs - 1) / kPairs * (cols + 64);
        if (c < cost) {
            best = cols;
            cost = c;
        }
    }
    return launch_pair<T>(a, best, stream);
}

}  // namespace

int launch_product_tc(const ProductArgs &a, int dtype, void *stream)
{
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case MGQ_FMT_F32: return launch_typed<float>(a, s);
        case MGQ_FMT_F16: return launch_typed<__half>(a, s);
        default: return launch_typed<__nv_bfloat16>(a, s);
    }
}

int int8_status()
{
    unsigned int err = 0;
    MGQ_CUDA(cudaMemcpyFromSymbol(&err, g_int8_error, sizeof err));
    if (!err) return MGQ_OK;
    const unsigned int zero = 0;
    MGQ_CUDA(cudaMemcpyToSymbol(g_int8_error, &zero, sizeof zero));
    return fail(MGQ_ERR_TIMEOUT, "a bounded wait inside the product of 8-bit integers ran out");
}

}  // namespace mgq
