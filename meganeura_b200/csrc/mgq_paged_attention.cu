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
// Up to four pairs take four rows, a warp each: with sixteen a block of keys took 11 us instead of 2.  Four threads fetch a key and its value; with 16-byte
// rows in f32 (WIDE) asynchronously, a tile ahead.  Few rows are bound by these loads, many by the multiply-adds' operands from shared memory.
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
    walk.begin(a, blockIdx.x, gridDim.x, s_walk);
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

// ---------------------------------------------------------------- many new tokens in f32
// 64 pairs of token and head against 64 keys at a time, as two register-tiled products: a thread has four rows and four keys of the scores (eight
// 16-byte loads from shared memory for 64 multiply-adds), then the same rows and eight columns of the sums (twenty for 128), so the multiply-add units bound it.
// Sixteen lanes share a row's maximum and sum by shuffles.  Keys are fetched while values are used and the other way around.
constexpr int kTileThreads = 256, kTileRows = 64, kTileKeys = 64, kTilePitch = kTileKeys + 4;
constexpr uint32_t kTileCtas = 148;
size_t tile_smem(uint32_t d) { return ((size_t)(kTileRows + 2 * kTileKeys) * (d + 4) + kTileRows * kTilePitch) * sizeof(float); }

template <int COLS>                                      // groups of four columns of a thread: heads of up to 64 * COLS
__global__ void __launch_bounds__(kTileThreads, 1) attend_tile_kernel(const AttendArgs a)
{
    extern __shared__ __align__(16) float s_mem[];
    __shared__ unsigned long long s_walk[40];
    const uint32_t t = threadIdx.x, d = a.d, pitch = d + 4, tr = t / 16, tc = t % 16;
    float *s_q = s_mem, *s_k = s_q + kTileRows * pitch, *s_v = s_k + kTileKeys * pitch, *s_p = s_v + kTileKeys * pitch;
    pdl_launch_dependents();
    pdl_wait();
    Walk<kTileRows, kTileKeys, 1> walk;
    walk.begin(a, blockIdx.x, gridDim.x, s_walk);
    if (t == 0) clear_parts(a, blockIdx.x);

    Segment g;
    while (walk.next(a, g)) {
        const uint32_t pairs = g.tokens * g.heads;
        // four threads fetch a key or a value; those that are not there are zeros
        auto fetch = [&](uint32_t kb, const void *from, float *to) {
            const uint32_t j = t / 4, key = kb * kTileKeys + j;
            const uint32_t page = (int)key < g.len ? g.table[key >> a.page_shift] : 0xFFFFFFFFu;
            const bool real = page < a.pages;
            const float *src = static_cast<const float *>(from) + (real ? ((((size_t)page << a.page_shift) + (key & ((1u << a.page_shift) - 1))) * a.kv_heads + g.kv) * d : 0);
            for (uint32_t c = t % 4 * 4; c < d; c += 16) copy16(to + j * pitch + c, src + c, real);
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();                                 // the unit before is done with shared memory
        if (g.begin < g.end) {
            fetch(g.begin, a.k, s_k);
            fetch(g.begin, a.v, s_v);
        }
        for (uint32_t r = t / 32; r < kTileRows; r += kTileThreads / 32) {
            const uint32_t token = r / g.heads, head = r - token * g.heads;
            const float *src = static_cast<const float *>(a.q) + (size_t)(g.row0 + (r < pairs ? token : 0)) * a.q_pitch + (size_t)(g.head0 + head) * d;
            for (uint32_t c = t % 32; c < d; c += 32) s_q[r * pitch + c] = r < pairs ? src[c] * a.scale_log2 : 0.f;
        }
        float m[4], l[4], o[4][COLS][4];
        int pos[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = tr * 4 + i;
            m[i] = -INFINITY;
            l[i] = 0.f;
            pos[i] = r < pairs ? g.pos0 + (int)(r / g.heads) : -1;
#pragma unroll
            for (int c = 0; c < COLS; c++) o[i][c][0] = o[i][c][1] = o[i][c][2] = o[i][c][3] = 0.f;
        }
        const int last_pos = g.pos0 + (int)g.tokens - 1;
        for (uint32_t kb = g.begin; kb < g.end; kb++) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");           // the keys; the values may be on their way
            __syncthreads();
            float s[4][4];
#pragma unroll
            for (int i = 0; i < 4; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll 2
            for (uint32_t c = 0; c < d; c += 4) {
                float4 q[4], k[4];
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = *reinterpret_cast<const float4 *>(s_q + (tr * 4 + i) * pitch + c);
#pragma unroll
                for (int j = 0; j < 4; j++) k[j] = *reinterpret_cast<const float4 *>(s_k + (tc + 16 * j) * pitch + c);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[i][j] = fmaf(q[i].x, k[j].x, fmaf(q[i].y, k[j].y, fmaf(q[i].z, k[j].z, fmaf(q[i].w, k[j].w, s[i][j]))));
            }
            __syncthreads();                             // the keys have been used
            if (kb + 1 < g.end) fetch(kb + 1, a.k, s_k);
            else                asm volatile("cp.async.commit_group;" ::: "memory");
            const int key0 = (int)(kb * kTileKeys);
            bool hidden = false;
            // everything is there and seen: the last key by the first token, the first one by the last
            bool there[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int key = key0 + (int)tc + 16 * j;
                there[j] = key < g.len && g.table[(uint32_t)key >> a.page_shift] < a.pages;
            }
            if (!__syncthreads_and(there[0] && there[1] && there[2] && there[3] && key0 + kTileKeys - 1 <= g.pos0 && (!a.window || key0 > last_pos - (int)a.window))) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = key0 + (int)tc + 16 * j;
                        const bool seen = there[j] && key <= pos[i] && (!a.window || key > pos[i] - (int)a.window);
                        hidden |= there[j] && !seen && tr * 4 + i < pairs;
                        s[i][j] = seen ? s[i][j] : -INFINITY;
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float top = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
                for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                top = fmaxf(m[i], top);
                const float base = top == -INFINITY ? 0.f : top, keep = exp2f(m[i] - base);
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    s[i][j] = exp2f(s[i][j] - base);     // 0 where nothing is seen, NaN stays
                    sum += s[i][j];
                    s_p[(tr * 4 + i) * kTilePitch + tc + 16 * j] = s[i][j];
                }
                l[i] = l[i] * keep + sum;                // of this lane; the sixteen are added at the end
                m[i] = top;
#pragma unroll
                for (int c = 0; c < COLS; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][c][e] *= keep;
            }
            asm volatile("cp.async.wait_group 1;" ::: "memory");           // the values; the next keys may be on their way
            const bool masked = __syncthreads_or(hidden);
            auto sums = [&](auto product) {
#pragma unroll 2
                for (int j = 0; j < kTileKeys; j += 4) {
                    float4 p[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) p[i] = *reinterpret_cast<const float4 *>(s_p + (tr * 4 + i) * kTilePitch + j);
#pragma unroll
                    for (int c = 0; c < COLS; c++) {
                        const uint32_t col = tc * 4 + 64 * c;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float4 v = col < d ? *reinterpret_cast<const float4 *>(s_v + (j + e) * pitch + col) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float w = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
                                product(o[i][c][0], w, v.x);
                                product(o[i][c][1], w, v.y);
                                product(o[i][c][2], w, v.z);
                                product(o[i][c][3], w, v.w);
                            }
                        }
                    }
                }
            };
            // what a row does not see stays out, infinities and NaN too
            if (masked) sums([](float &x, float w, float v) { x += w != 0.f ? w * v : 0.f; });
            else        sums([](float &x, float w, float v) { x = fmaf(w, v, x); });
            __syncthreads();                             // the values have been used
            if (kb + 1 < g.end) fetch(kb + 1, a.v, s_v);
            else                asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const bool whole = g.first && g.last;
        float *part = a.parts + (size_t)part_index(blockIdx.x, g) * kTileRows * (d + 2);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = tr * 4 + i, token = r / g.heads, head = r - token * g.heads;
            float sum = l[i];
#pragma unroll
            for (int x = 1; x < 16; x *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (r < pairs) {
                const float scale = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
                float *dst = whole ? static_cast<float *>(a.out) + (size_t)(g.row0 + token) * a.out_pitch + (size_t)(g.head0 + head) * d : part + r * d;
#pragma unroll
                for (int c = 0; c < COLS; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (tc * 4 + 64 * c < d) dst[tc * 4 + 64 * c + e] = o[i][c][e] * scale;
                if (!whole && tc == 0) *reinterpret_cast<float2 *>(part + kTileRows * d + 2 * r) = make_float2(m[i], sum);
            }
        }
        if (!whole && t == 0) name_part(a, blockIdx.x, g);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// f32 with heads over 128 (smaller ones of this kind are other kernels').
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
        if (wide) kernel = attend_kernel<T, ROWS, 2, true>;      // smaller heads are mgq_paged_few.cu's and the tiles'
    if (int rc = allow_smem(kernel, smem)) return rc;
    if (int rc = launch(kernel, dim3(ctas), dim3(kThreads), smem, stream, a)) return rc;
    return launch_merge<T, ROWS>(a, ctas, ROWS, stream);
}
template <typename T>
int launch_attend(const AttendArgs &a, int dtype, uint32_t pairs, cudaStream_t stream)
{
    return pairs <= kFewRows ? launch_rows<T, kFewRows>(a, dtype, stream) : launch_rows<T, kRows>(a, dtype, stream);
}
int launch_tile(const AttendArgs &a, cudaStream_t stream)
{
    auto *kernel = a.d <= 64 ? attend_tile_kernel<1> : attend_tile_kernel<2>;
    if (int rc = allow_smem(kernel, tile_smem(a.d))) return rc;
    if (int rc = launch(kernel, dim3(kTileCtas), dim3(kTileThreads), tile_smem(a.d), stream, a)) return rc;
    return launch_merge<float, kTileRows>(a, kTileCtas, kTileRows, stream);
}

}  // namespace

// Parts of the kernels that may serve a call: alignment and lengths decide which.
size_t paged_attention_workspace(uint32_t head_dim, int dtype)
{
    auto bytes = [&](uint32_t ctas, size_t rows) { return ctas * 2 * (sizeof(PartHead) + rows * (head_dim + 2) * sizeof(float)); };
    const size_t plain = max(bytes(plain_ctas(kRows, head_dim), kRows), bytes(plain_ctas(kFewRows, head_dim), kFewRows));
    size_t few = 0;
    for (uint32_t rows : {1u, 4u, 8u}) few = max(few, few_ctas(rows) * 2 * (sizeof(PartHead) + few_part_floats(rows, head_dim) * sizeof(float)));
    return dtype == MGQ_FMT_F32 ? max(plain, few + bytes(kTileCtas, head_dim <= 128 ? kTileRows : 0)) : max(plain, bytes(decode_ctas(head_dim), kDecodeRows) + bytes(kPrefillCtas, head_dim <= 128 ? kPrefillRows : 0));
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
    if (few_takes(a, dtype)) {
        // of more than eight pairs units of eight; beside sequences of many tokens most others have one token
        const uint32_t rows = pairs > kFewPairs ? (a.group <= 4 ? 4 : 8) : pairs == 1 ? 1 : pairs <= 4 ? 4 : 8;
        room(few_ctas(rows));
        if (pairs <= kFewPairs) return launch_few(a, rows, s);
        // both kinds of sequences may be there
        a.rows_to = kFewPairs;
        if (int rc = launch_few(a, rows, s)) return rc;
        a.rows_from = kFewPairs + 1;
        a.rows_to = 0xFFFFFFFFu;
        a.heads = reinterpret_cast<PartHead *>(a.parts + few_ctas(rows) * 2 * few_part_floats(rows, head_dim));
        a.parts = reinterpret_cast<float *>(a.heads + 2 * kTileCtas);
        return launch_tile(a, s);
    }
    room(plain_ctas(pairs <= kFewRows ? kFewRows : kRows, head_dim));
    switch (dtype) {
        case MGQ_FMT_F32: return launch_attend<float>(a, dtype, pairs, s);
        case MGQ_FMT_F16: return launch_attend<__half>(a, dtype, pairs, s);
        default: return launch_attend<__nv_bfloat16>(a, dtype, pairs, s);
    }
}

}  // namespace mgq
