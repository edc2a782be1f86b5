// Bookkeeping of one cache shared by many sequences: which pages a step needs and where its rows go (mgq_paged_plan), pages given
// back (mgq_paged_trim), the rotated keys and the values of new tokens on their way into the cache (mgq_paged_append).
//
// Plan and trim move a few KB and are bound by latency: global round trips, two block scans, one barrier.  Everything that decides
// (running sums of rows and pages) is computed by every CTA for itself, so the only exchange is a barrier between the reads of the
// pool's words and their update.
#include <cstdint>

#include "mgq_launch.cuh"
#include "mgq_paged.cuh"

namespace mgq {
namespace {

constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;
constexpr uint32_t kPerThread = MGQ_PAGED_MAX_SEQUENCES / kPlanThreads;         // a block has at least a thread per four sequences

// Exclusive sums over the block in thread order; `total` is everybody's sum.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long &total, unsigned long long *s_warp)
{
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    unsigned long long sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long below = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= (uint32_t)o) sum += below;
    }
    if (lane == 31) s_warp[warp] = sum;
    __syncthreads();
    unsigned long long w = lane < blockDim.x / 32 ? s_warp[lane] : 0ull;
    const unsigned long long own = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long below = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= (uint32_t)o) w += below;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const unsigned long long base = __shfl_sync(0xffffffffu, w - own, warp);
    __syncthreads();                                     // s_warp may be used again
    return base + sum - v;
}

struct PlanArgs {
    const uint32_t *cached, *fresh;
    uint32_t sequences, page_size, page_shift;
    uint32_t *table, table_width, *held, *free_count;
    const uint32_t *free_pages;
    uint32_t pages, rows;
    uint32_t *starts, *lengths, *positions, *slots, *lacking;
};

// Sequence s has rows [start[s], start[s + 1]).  Its new pages are free[count - 1 - (before[s] + i)], i = 0, 1, ...: the top of the stack
// first, sequence after sequence.  The running need only grows, so those that are served come before the first that is not, and
// before[s] counts served pages only.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a)
{
    extern __shared__ uint32_t s_plan[];
    __shared__ unsigned long long s_warp[kPlanWarps];
    __shared__ uint32_t s_given;
    uint32_t *s_start = s_plan, *s_before = s_start + a.sequences + 1, *s_held = s_before + a.sequences, *s_got = s_held + a.sequences, *s_cached = s_got + a.sequences;
    const uint32_t t = threadIdx.x, lane = t & 31u, part = blockIdx.y, parts = gridDim.y, threads = blockDim.x, warp = part * (threads / 32) + (t >> 5);
    if (t == 0) s_given = 0;
    pdl_launch_dependents();
    pdl_wait();

    const uint32_t count = min(*a.free_count, a.pages), each = (a.sequences + threads - 1) / threads, s0 = t * each;
    uint32_t cached[kPerThread], fresh[kPerThread], held[kPerThread];
    unsigned long long sum = 0, total;
#pragma unroll
    for (uint32_t i = 0; i < kPerThread; i++) {
        const bool live = i < each && s0 + i < a.sequences;
        cached[i] = live ? a.cached[s0 + i] : 0;
        fresh[i] = live ? a.fresh[s0 + i] : 0;
        held[i] = live ? min(a.held[s0 + i], a.table_width) : 0;
        sum += fresh[i];
    }
    unsigned long long at = block_scan(sum, total, s_warp);
    uint32_t need[kPerThread];
    bool narrow[kPerThread];
    unsigned long long wanted = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPerThread; i++) {
        const uint32_t begin = (uint32_t)min(at, (unsigned long long)a.rows);
        at += fresh[i];
        const uint32_t n = (uint32_t)min(at, (unsigned long long)a.rows) - begin;        // tokens behind the last row have none
        fresh[i] = n;
        const unsigned long long after = ((unsigned long long)cached[i] + n + a.page_size - 1) >> a.page_shift;
        narrow[i] = after > a.table_width;
        need[i] = narrow[i] || after <= held[i] ? 0u : (uint32_t)after - held[i];
        if (i < each && s0 + i < a.sequences) s_start[s0 + i] = begin;
        wanted += need[i];
    }
    const uint32_t last_row = (uint32_t)min(total, (unsigned long long)a.rows);
    unsigned long long before = block_scan(wanted, total, s_warp);
#pragma unroll
    for (uint32_t i = 0; i < kPerThread; i++) {
        const bool served = !narrow[i] && (need[i] == 0 || before + need[i] <= count);
        const uint32_t s = s0 + i;
        if (i < each && s < a.sequences) {
            s_before[s] = (uint32_t)before;
            s_held[s] = held[i];
            s_cached[s] = cached[i];
            s_got[s] = served ? need[i] : 0xFFFFFFFFu;
            if (served && need[i]) atomicMax(&s_given, (uint32_t)before + need[i]);         // those that are served come first
            if (part == 0) a.starts[s] = s_start[s];
        }
        before += need[i];
    }
    if (t == 0) s_start[a.sequences] = last_row;
    if (parts > 1) cluster_sync();                       // every CTA has read cached (which may be lengths), held and free_count
    else           __syncthreads();
    if (part == 0) {
        if (t == 0) {
            a.starts[a.sequences] = last_row;
            *a.free_count = count - s_given;
            *a.lacking = (uint32_t)min(total > count ? total - count : 0ull, 0xFFFFFFFFull);
        }
        for (uint32_t s = t; s < a.sequences; s += threads) {
            const bool served = s_got[s] != 0xFFFFFFFFu;
            if (served) a.held[s] = s_held[s] + s_got[s];
            a.lengths[s] = s_cached[s] + (served ? s_start[s + 1] - s_start[s] : 0u);
        }
    }
    for (uint32_t s = warp; s < a.sequences; s += parts * (threads / 32)) {
        const uint32_t got = s_got[s] == 0xFFFFFFFFu ? 0u : s_got[s];
        for (uint32_t i = lane; i < got; i += 32)
            a.table[(size_t)s * a.table_width + s_held[s] + i] = a.free_pages[count - 1 - (s_before[s] + i)];
    }
    for (uint32_t r = part * threads + t; r < a.rows; r += parts * threads) {
        uint32_t slot = MGQ_NO_SLOT, position = 0;
        if (r < last_row) {
            uint32_t lo = 0, hi = a.sequences;           // the last sequence that starts at or before r, empty ones passed over
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (s_start[mid] <= r) lo = mid;
                else                   hi = mid;
            }
            position = s_cached[lo] + r - s_start[lo];
            const uint32_t j = position >> a.page_shift;
            if (s_got[lo] != 0xFFFFFFFFu) {
                const uint32_t page = j < s_held[lo] ? a.table[(size_t)lo * a.table_width + j] : a.free_pages[count - 1 - (s_before[lo] + j - s_held[lo])];
                if (page < a.pages) slot = (page << a.page_shift) + (position & (a.page_size - 1));
            }
        }
        a.positions[r] = position;
        a.slots[r] = slot;
    }
}

// The k-th page given back, sequences and their pages in order, goes to free[count + all - 1 - k]: a trim to the lengths before a
// plan leaves the stack as it was before the plan.
__global__ void __launch_bounds__(kPlanThreads) trim_kernel(const uint32_t *lengths, uint32_t sequences, uint32_t page_size, uint32_t page_shift, uint32_t *table,
                                                            uint32_t table_width, uint32_t *held, uint32_t *free_pages, uint32_t pages, uint32_t *free_count)
{
    extern __shared__ uint32_t s_plan[];
    __shared__ unsigned long long s_warp[kPlanWarps];
    uint32_t *s_before = s_plan, *s_keep = s_before + sequences, *s_gone = s_keep + sequences;
    const uint32_t t = threadIdx.x, lane = t & 31u, part = blockIdx.y, parts = gridDim.y, threads = blockDim.x, warp = part * (threads / 32) + (t >> 5);
    const uint32_t each = (sequences + threads - 1) / threads, s0 = t * each;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t count = min(*free_count, pages);
    uint32_t gone[kPerThread];
    unsigned long long sum = 0, total;
#pragma unroll
    for (uint32_t i = 0; i < kPerThread; i++) {
        gone[i] = 0;
        const uint32_t s = s0 + i;
        if (i < each && s < sequences) {
            const uint32_t have = min(held[s], table_width);
            const unsigned long long keep = ((unsigned long long)lengths[s] + page_size - 1) >> page_shift;
            if (keep < have) gone[i] = have - (uint32_t)keep;
            s_keep[s] = have - gone[i];
            s_gone[s] = gone[i];
        }
        sum += gone[i];
    }
    unsigned long long before = block_scan(sum, total, s_warp);
#pragma unroll
    for (uint32_t i = 0; i < kPerThread; i++) {
        const uint32_t s = s0 + i;
        if (i < each && s < sequences) {
            s_before[s] = (uint32_t)before;
        }
        before += gone[i];
    }
    if (parts > 1) cluster_sync();                       // every CTA has read held and free_count
    else           __syncthreads();
    if (part == 0)
        for (uint32_t s = t; s < sequences; s += threads)
            if (s_gone[s]) held[s] = s_keep[s];
    if (part == 0 && t == 0) *free_count = (uint32_t)min(count + total, (unsigned long long)pages);
    for (uint32_t s = warp; s < sequences; s += parts * (threads / 32)) {
        uint32_t *row = table + (size_t)s * table_width + s_keep[s];
        for (uint32_t i = lane; i < s_gone[s]; i += 32) {
            const unsigned long long place = count + total - 1 - (s_before[s] + i);
            if (place < pages) free_pages[place] = row[i];
            row[i] = MGQ_NO_PAGE;
        }
    }
}

// ---------------------------------------------------------------- keys and values into the cache
// A CTA takes a row at a time, four CTAs per SM (4096 rows of the Qwen3-8B shape, 151 MB: 26.7 us, with three 31.3).  Its angles (position *
// theta^(-2i/d), product and reduction to one turn in 64 bits: at position 100000 an f32 product is off by up to 0.004) are computed once for
// all heads, then a thread rotates four pairs of a head per step.
constexpr int kAppendThreads = 256, kBatch = 4;

struct AppendArgs {
    const void *q, *k, *v;
    const uint32_t *positions, *slots;
    void *q_out, *k_cache, *v_cache;
    uint32_t rows, q_heads, kv_heads, d, q_pitch, k_pitch, v_pitch;
    unsigned long long cache_rows;
    double log2_theta;
    bool rotate;
};

template <int N, typename T>
__device__ __forceinline__ void read_values(const T *p, float (&f)[N])
{
    if constexpr (N == 4 && sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else if constexpr (N == 4) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = to_f32(e[i]);
    } else {
        f[0] = to_f32(p[0]);
    }
}
template <int N, typename T>
__device__ __forceinline__ void write_values(T *p, const float (&f)[N])
{
    if constexpr (N == 4 && sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else if constexpr (N == 4) {
        T e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = rounded<T>(f[i]);
        *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(e);
    } else {
        p[0] = rounded<T>(f[0]);
    }
}

template <typename S, typename T, int N>      // source, cache; N values at a time
__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(const AppendArgs a)
{
    __shared__ float2 s_turn[MGQ_PAGED_MAX_HEAD / 2];
    const uint32_t t = threadIdx.x, half = a.d / 2, steps = half / N;
    const double frequency = a.rotate && t < half ? exp2(-a.log2_theta * (double)t / (double)half) : 0.0;
    pdl_launch_dependents();
    pdl_wait();
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const uint32_t slot = a.slots[r];
        const bool stored = slot < a.cache_rows;
        const uint32_t q_items = a.q ? a.q_heads * steps : 0, k_items = a.kv_heads * steps, items = q_items + (stored ? 2 * k_items : 0);
        // item: N pairs (p, p + half) of a head of q or k, 2 N values of v
        for (uint32_t i0 = 0; i0 < items || i0 == 0; i0 += kBatch * kAppendThreads) {
            float lo[kBatch][N], hi[kBatch][N];
#pragma unroll
            for (int b = 0; b < kBatch; b++) {           // all of a batch's loads first, for the first batch in front of the angles
                const uint32_t i = i0 + b * kAppendThreads + t;
                if (i >= items) continue;
                const S *src;
                uint32_t far = half;
                if (i < q_items + k_items) {
                    const bool is_q = i < q_items;
                    const uint32_t j = is_q ? i : i - q_items, head = j / steps, p = (j - head * steps) * N;
                    src = (is_q ? static_cast<const S *>(a.q) + (size_t)r * a.q_pitch : static_cast<const S *>(a.k) + (size_t)r * a.k_pitch) + head * a.d + p;
                } else {
                    src = static_cast<const S *>(a.v) + (size_t)r * a.v_pitch + (i - q_items - k_items) * 2 * N;
                    far = N;
                }
                read_values(src, lo[b]);
                read_values(src + far, hi[b]);
            }
            if (i0 == 0 && a.rotate) {
                if (t < half) {
                    const double angle = (double)a.positions[r] * frequency, turn = 6.283185307179586476925286766559;
                    float2 w;
                    sincosf((float)fma(-rint(angle * (1.0 / turn)), turn, angle), &w.y, &w.x);
                    s_turn[t] = w;
                }
                __syncthreads();
            }
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const uint32_t i = i0 + b * kAppendThreads + t;
                if (i >= items) continue;
                T *dst;
                uint32_t far = half;
                if (i < q_items + k_items) {
                    const bool is_q = i < q_items;
                    const uint32_t j = is_q ? i : i - q_items, head = j / steps, p = (j - head * steps) * N;
                    dst = (is_q ? static_cast<T *>(a.q_out) + (size_t)r * a.q_heads * a.d : static_cast<T *>(a.k_cache) + (size_t)slot * a.kv_heads * a.d) + head * a.d + p;
                    if (a.rotate) {
#pragma unroll
                        for (int e = 0; e < N; e++) {
                            const float2 w = s_turn[p + e];
                            const float x = lo[b][e] * w.x - hi[b][e] * w.y;
                            hi[b][e] = lo[b][e] * w.y + hi[b][e] * w.x;
                            lo[b][e] = x;
                        }
                    }
                } else {
                    dst = static_cast<T *>(a.v_cache) + (size_t)slot * a.kv_heads * a.d + (i - q_items - k_items) * 2 * N;
                    far = N;
                }
                write_values(dst, lo[b]);
                write_values(dst + far, hi[b]);
            }
        }
        if (a.rotate) __syncthreads();                   // the angles have been used
    }
}

template <typename S, typename T>
int launch_append_typed(const AppendArgs &a, bool wide, cudaStream_t stream)
{
    const dim3 grid(min(a.rows, 148u * 4u));
    return wide ? launch(append_kernel<S, T, 4>, grid, dim3(kAppendThreads), 0, stream, a) : launch(append_kernel<S, T, 1>, grid, dim3(kAppendThreads), 0, stream, a);
}

}  // namespace

// Barriers of few threads are quick: 256 where that is a thread per sequence and a few rows each.
static uint32_t plan_threads(uint32_t sequences, uint32_t rows) { return sequences <= 256 && rows <= 1024 ? 256 : kPlanThreads; }

int launch_paged_plan(const uint32_t *cached, const uint32_t *fresh, uint32_t sequences, uint32_t page_size, uint32_t *table, uint32_t table_width, uint32_t *held,
                      const uint32_t *free_pages, uint32_t pages, uint32_t *free_count, uint32_t rows, uint32_t *starts, uint32_t *lengths, uint32_t *positions,
                      uint32_t *slots, uint32_t *lacking, void *stream)
{
    const PlanArgs a{cached, fresh, sequences, page_size, page_shift(page_size), table, table_width, held, free_count, free_pages, pages, rows, starts, lengths, positions,
                     slots, lacking};
    const size_t smem = (5 * (size_t)sequences + 1) * 4;
    if (int rc = allow_smem(plan_kernel, smem)) return rc;
    // one CTA while its threads have few rows and its warps few sequences each, a cluster of eight beyond
    const uint32_t threads = plan_threads(sequences, rows), parts = rows <= 2 * threads && sequences <= 2 * threads / 32 ? 1 : 8;
    return launch_clustered(plan_kernel, dim3(1, parts), dim3(threads), parts, smem, static_cast<cudaStream_t>(stream), a);
}

int launch_paged_trim(const uint32_t *lengths, uint32_t sequences, uint32_t page_size, uint32_t *table, uint32_t table_width, uint32_t *held, uint32_t *free_pages,
                      uint32_t pages, uint32_t *free_count, void *stream)
{
    const size_t smem = 3 * (size_t)sequences * 4;
    if (int rc = allow_smem(trim_kernel, smem)) return rc;
    const uint32_t threads = plan_threads(sequences, 0), parts = sequences <= 2 * threads / 32 ? 1 : 8;
    return launch_clustered(trim_kernel, dim3(1, parts), dim3(threads), parts, smem, static_cast<cudaStream_t>(stream), lengths, sequences, page_size, page_shift(page_size),
                            table, table_width, held, free_pages, pages, free_count);
}

int launch_paged_append(const void *q, const void *k, const void *v, int src_dtype, const uint32_t *positions, const uint32_t *slots, void *q_out, void *k_cache,
                        void *v_cache, int cache_dtype, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t q_pitch, uint32_t k_pitch,
                        uint32_t v_pitch, unsigned long long cache_rows, float theta, void *stream)
{
    const AppendArgs a{q, k, v, positions, slots, q_out, k_cache, v_cache, rows, q ? q_heads : 0u, kv_heads, head_dim, q_pitch, k_pitch, v_pitch, cache_rows,
                       theta > 0.f ? log2((double)theta) : 0.0, theta > 0.f};
    auto fits = [](const void *p, uint32_t pitch, int dtype) { return !p || (reinterpret_cast<uintptr_t>(p) % (4 * element_bytes(dtype)) == 0 && pitch % 4 == 0); };
    const bool wide = head_dim % 8 == 0 && fits(q, q_pitch, src_dtype) && fits(k, k_pitch, src_dtype) && fits(v, v_pitch, src_dtype) && fits(q_out, 0, cache_dtype) &&
                      fits(k_cache, 0, cache_dtype) && fits(v_cache, 0, cache_dtype);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (cache_dtype) {
        case MGQ_FMT_F32: return launch_append_typed<float, float>(a, wide, s);
        case MGQ_FMT_F16: return src_dtype == MGQ_FMT_F32 ? launch_append_typed<float, __half>(a, wide, s) : launch_append_typed<__half, __half>(a, wide, s);
        default: return src_dtype == MGQ_FMT_F32 ? launch_append_typed<float, __nv_bfloat16>(a, wide, s) : launch_append_typed<__nv_bfloat16, __nv_bfloat16>(a, wide, s);
    }
}

}  // namespace mgq
