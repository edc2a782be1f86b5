// Attention of new tokens over a paged cache, any types and sizes: the form that the others stand beside, and the one for f32.
#include <cstdint>

#include "mgq_paged.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kKeys = 32;                                // of a block
constexpr int kRows = 16, kFewRows = 4;                  // pairs of token and head of a unit

__device__ __forceinline__ void copy16(float *dst, const void *src, bool real)
{
    const uint32_t bytes = real ? 16 : 0;                // the rest is zero-filled
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(bytes) : "memory");
}

// out[row, col] (+)= over a tile of 32 keys: a warp scores a quarter of the rows with a key per lane, a thread sums one or two columns for all rows.
// Single tokens of up to four heads per key / value head take four rows, a warp each: with sixteen a block of keys took 11 us instead of 2.
// Four threads fetch a key and its value; with 16-byte rows in f32 (WIDE) asynchronously, a tile ahead.  Single tokens are bound by these loads,
// portions by the multiply-adds' operands from shared memory.
template <typename T, int ROWS, int COLS, bool WIDE>     // COLS: columns per thread, heads of up to 128 * COLS
__global__ void __launch_bounds__(kThreads) attend_kernel(const AttendArgs a)
{
    constexpr int kRowsPerWarp = ROWS / kWarps;
    extern __shared__ __align__(16) float s_mem[];
    __shared__ unsigned long long s_walk[40];
    __shared__ float s_p[ROWS][kKeys], s_scale[ROWS];
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, d = a.d, d4 = (d + 3) / 4 * 4, pitch = d4 + 4, tile = 2 * kKeys * pitch;
    float *s_q = s_mem, *s_tiles = s_q + ROWS * d4;
    pdl_launch_dependents();
    pdl_wait();
    Walk<ROWS, kKeys, 0> walk;
    walk.begin(a, blockIdx.x, gridDim.x, 1, s_walk);
    if (t == 0) clear_parts(a, blockIdx.x);

    Segment g;
    while (walk.next(a, g)) {
        const uint32_t pairs = g.tokens * g.heads;
        auto fetch = [&](uint32_t kb) {
            const uint32_t j = t / 4, key = kb * kKeys + j;
            const uint32_t page = (int)key < g.len ? g.table[key >> a.page_shift] : 0xFFFFFFFFu;
            const bool real = page < a.pages;
            const size_t at = real ? ((((size_t)page << a.page_shift) + (key & ((1u << a.page_shift) - 1))) * a.kv_heads + g.kv) * d : 0;
            float *k = s_tiles + (WIDE && kb & 1u ? tile : 0) + j * pitch, *v = k + kKeys * pitch;
            const T *k_src = static_cast<const T *>(a.k) + at, *v_src = static_cast<const T *>(a.v) + at;
            if constexpr (WIDE) {
                for (uint32_t c = t % 4 * 4; c < d; c += 16) {
                    copy16(k + c, k_src + c, real);
                    copy16(v + c, v_src + c, real);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            } else {
                for (uint32_t c = t % 4; c < d4; c += 4) {
                    k[c] = real && c < d ? to_f32(k_src[c]) : 0.f;
                    v[c] = real && c < d ? to_f32(v_src[c]) : 0.f;
                }
            }
        };
        __syncthreads();
        if (WIDE && g.begin < g.end) fetch(g.begin);
        for (uint32_t r = warp; r < ROWS; r += kWarps) {
            const uint32_t token = r / g.heads, head = r - token * g.heads;
            const T *src = static_cast<const T *>(a.q) + (size_t)(g.row0 + (r < pairs ? token : 0)) * a.q_pitch + (size_t)(g.head0 + head) * d;
            for (uint32_t c = lane; c < d4; c += 32) s_q[r * d4 + c] = r < pairs && c < d ? to_f32(src[c]) : 0.f;
        }
        float m[kRowsPerWarp], l[kRowsPerWarp], acc[COLS][ROWS];
        int pos[kRowsPerWarp];
#pragma unroll
        for (int i = 0; i < kRowsPerWarp; i++) {
            const uint32_t r = warp * kRowsPerWarp + i;
            m[i] = -INFINITY;
            l[i] = 0.f;
            pos[i] = r < pairs ? g.pos0 + (int)(r / g.heads) : -1;
        }
#pragma unroll
        for (int c = 0; c < COLS; c++)
#pragma unroll
            for (int r = 0; r < ROWS; r++) acc[c][r] = 0.f;

        for (uint32_t kb = g.begin; kb < g.end; kb++) {
            if constexpr (WIDE) {
                if (kb + 1 < g.end) {
                    fetch(kb + 1);
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                } else {
                    asm volatile("cp.async.wait_group 0;" ::: "memory");
                }
            } else {
                fetch(kb);
            }
            __syncthreads();
            const float *s_k = s_tiles + (WIDE && kb & 1u ? tile : 0), *s_v = s_k + kKeys * pitch;
            const int key = (int)(kb * kKeys + lane);
            const bool there = key < g.len && g.table[(uint32_t)key >> a.page_shift] < a.pages;
            float s[kRowsPerWarp], s2[kRowsPerWarp];     // two chains of multiply-adds per row
#pragma unroll
            for (int i = 0; i < kRowsPerWarp; i++) s[i] = s2[i] = 0.f;
#pragma unroll 4
            for (uint32_t c = 0; c < d4; c += 4) {
                const float4 kv = *reinterpret_cast<const float4 *>(s_k + lane * pitch + c);
#pragma unroll
                for (int i = 0; i < kRowsPerWarp; i++) {
                    const float4 qv = *reinterpret_cast<const float4 *>(s_q + (warp * kRowsPerWarp + i) * d4 + c);
                    s[i] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, s[i]));
                    s2[i] = fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s2[i]));
                }
            }
#pragma unroll
            for (int i = 0; i < kRowsPerWarp; i++) s[i] += s2[i];
            bool hidden = false;                         // some pair of this tile is masked
#pragma unroll
            for (int i = 0; i < kRowsPerWarp; i++) {
                const bool seen = there && key <= pos[i] && (!a.window || key > pos[i] - (int)a.window);
                hidden |= there && !seen && warp * kRowsPerWarp + i < pairs;        // keys that are not there are zeros
                const float x = seen ? s[i] * a.scale_log2 : -INFINITY, top = fmaxf(m[i], warp_max(x));
                // a row whose seen scores are all -inf has no weight, like one that sees nothing; NaN stays NaN
                const float w = !seen ? 0.f : x != x ? x : top > -INFINITY ? exp2f(x - top) : 0.f, keep = top > -INFINITY ? exp2f(m[i] - top) : 1.f;
                l[i] = l[i] * keep + warp_sum(w);
                m[i] = top;
                s_p[warp * kRowsPerWarp + i][lane] = w;
                if (lane == 0) s_scale[warp * kRowsPerWarp + i] = keep;
            }
            const bool masked = __syncthreads_or(hidden);
#pragma unroll
            for (int c = 0; c < COLS; c++) {
                const uint32_t col = t + c * kThreads;
                if (col >= d) continue;
#pragma unroll
                for (int r = 0; r < ROWS; r++) acc[c][r] *= s_scale[r];
#pragma unroll 2
                for (int j = 0; j < kKeys; j += 4) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = s_v[(j + e) * pitch + col];
#pragma unroll
                    for (int r = 0; r < ROWS; r++) {
                        const float4 p = *reinterpret_cast<const float4 *>(&s_p[r][j]);
                        if (masked) {                    // what a row does not see stays out, infinities and NaN too
                            acc[c][r] += (p.x != 0.f ? p.x * v[0] : 0.f) + (p.y != 0.f ? p.y * v[1] : 0.f) + (p.z != 0.f ? p.z * v[2] : 0.f) + (p.w != 0.f ? p.w * v[3] : 0.f);
                        } else {
                            acc[c][r] = fmaf(p.x, v[0], fmaf(p.y, v[1], fmaf(p.z, v[2], fmaf(p.w, v[3], acc[c][r]))));
                        }
                    }
                }
            }
            __syncthreads();                             // the tile has been used
        }
        const bool whole = g.first && g.last;
        if (whole) {
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < kRowsPerWarp; i++) s_scale[warp * kRowsPerWarp + i] = l[i] == 0.f ? 0.f : 1.f / l[i];
            __syncthreads();
        }
        float *part = a.parts + (size_t)part_index(blockIdx.x, g) * ROWS * (d + 2);
#pragma unroll
        for (int c = 0; c < COLS; c++) {
            const uint32_t col = t + c * kThreads;
            if (col >= d) continue;
#pragma unroll
            for (uint32_t r = 0; r < ROWS; r++) {
                if (r >= pairs) break;
                const uint32_t token = r / g.heads, head = r - token * g.heads;
                if (whole) static_cast<T *>(a.out)[(size_t)(g.row0 + token) * a.out_pitch + (g.head0 + head) * d + col] = rounded<T>(acc[c][r] * s_scale[r]);
                else       part[r * d + col] = acc[c][r];
            }
        }
        if (!whole) {
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < kRowsPerWarp; i++) {
                    part[ROWS * d + 2 * (warp * kRowsPerWarp + i)] = m[i];
                    part[ROWS * d + 2 * (warp * kRowsPerWarp + i) + 1] = l[i];
                }
            if (t == 0) name_part(a, blockIdx.x, g);
        }
    }
}

bool wide_rows(const AttendArgs &a, int dtype)
{
    return dtype == MGQ_FMT_F32 && a.d % 4 == 0 && reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
}
size_t smem_bytes(uint32_t rows, uint32_t d, bool wide)
{
    const uint32_t d4 = (d + 3) / 4 * 4;
    return ((size_t)rows * d4 + (wide ? 2 : 1) * 2 * kKeys * (d4 + 4)) * sizeof(float);
}
// As many CTAs as their shared memory lets an SM hold, four at most (registers); a form with fewer keys in flight than another one must not need a larger workspace.
uint32_t plain_ctas(uint32_t rows, uint32_t d) { return 148 * min(4u, (uint32_t)(224 * 1024 / (smem_bytes(rows, d, true) + 3584))); }

template <typename T, int ROWS>
int launch_rows(const AttendArgs &a, int dtype, cudaStream_t stream)
{
    const bool wide = wide_rows(a, dtype);
    const uint32_t ctas = plain_ctas(ROWS, a.d);
    const size_t smem = smem_bytes(ROWS, a.d, wide);
    auto *kernel = a.d <= 128 ? attend_kernel<T, ROWS, 1, false> : attend_kernel<T, ROWS, 2, false>;
    if constexpr (sizeof(T) == 4)
        if (wide) kernel = a.d <= 128 ? attend_kernel<T, ROWS, 1, true> : attend_kernel<T, ROWS, 2, true>;
    if (int rc = allow_smem(kernel, smem)) return rc;
    if (int rc = launch(kernel, dim3(ctas), dim3(kThreads), smem, stream, a)) return rc;
    return launch_merge<T, ROWS>(a, ctas, ROWS, stream);
}
template <typename T>
int launch_attend(const AttendArgs &a, int dtype, uint32_t pairs, cudaStream_t stream)
{
    return pairs <= kFewRows ? launch_rows<T, kFewRows>(a, dtype, stream) : launch_rows<T, kRows>(a, dtype, stream);
}

}  // namespace

// Parts of the kernel that serves these arguments (the largest of them where the alignment decides).
size_t paged_attention_workspace(uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_fresh, int dtype)
{
    (void)heads; (void)kv_heads; (void)max_fresh;
    auto bytes = [&](uint32_t ctas, size_t rows) { return ctas * 2 * (sizeof(PartHead) + rows * (head_dim + 2) * sizeof(float)); };
    const size_t plain = max(bytes(plain_ctas(kRows, head_dim), kRows), bytes(plain_ctas(kFewRows, head_dim), kFewRows));
    return dtype == MGQ_FMT_F32 ? plain : max(plain, bytes(decode_ctas(head_dim), kDecodeRows) + bytes(kPrefillCtas, head_dim <= 128 ? kPrefillRows : 0));
}

int launch_paged_attention(const void *q, const void *k_cache, const void *v_cache, int dtype, const uint32_t *table, const uint32_t *starts, const uint32_t *lengths,
                           void *out, uint32_t sequences, uint32_t rows, uint32_t max_fresh, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t page_size,
                           uint32_t pages, uint32_t table_width, uint32_t q_pitch, uint32_t out_pitch, float scale, uint32_t window, void *workspace, void *stream)
{
    AttendArgs a{};
    a.q = q; a.k = k_cache; a.v = v_cache; a.out = out;
    a.starts = starts; a.lengths = lengths; a.table = table;
    a.sequences = sequences; a.rows = rows; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.d = head_dim;
    a.page_shift = page_shift(page_size); a.pages = pages; a.table_width = table_width;
    a.window = window < (1u << 31) ? window : 0u;                      // no sequence is longer
    a.q_pitch = q_pitch; a.out_pitch = out_pitch;
    a.rows_from = 1; a.rows_to = 0xFFFFFFFFu;
    a.scale_log2 = scale * 1.4426950408889634f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto room = [&](uint32_t ctas) {
        a.heads = static_cast<PartHead *>(workspace);
        a.parts = reinterpret_cast<float *>(a.heads + 2 * ctas);
    };
    const uint32_t pairs = (uint32_t)min((unsigned long long)max_fresh * a.group, 0xFFFFFFFFull);
    if (decode_takes(a, dtype)) {
        room(decode_ctas(head_dim));
        if (pairs <= kDecodePairs || !prefill_takes(a, dtype)) return launch_decode(a, dtype, pairs, s);
        // both kinds of sequences may be there
        a.rows_to = kDecodePairs;
        if (int rc = launch_decode(a, dtype, kDecodePairs, s)) return rc;
        a.rows_from = kDecodePairs + 1;
        a.rows_to = 0xFFFFFFFFu;
        a.heads = reinterpret_cast<PartHead *>(a.parts + (size_t)decode_ctas(head_dim) * 2 * kDecodeRows * (head_dim + 2));
        a.parts = reinterpret_cast<float *>(a.heads + 2 * kPrefillCtas);
        return launch_prefill(a, dtype, s);
    }
    room(plain_ctas(pairs <= kFewRows ? kFewRows : kRows, head_dim));
    switch (dtype) {
        case MGQ_FMT_F32: return launch_attend<float>(a, dtype, pairs, s);
        case MGQ_FMT_F16: return launch_attend<__half>(a, dtype, pairs, s);
        default: return launch_attend<__nv_bfloat16>(a, dtype, pairs, s);
    }
}

}  // namespace mgq
