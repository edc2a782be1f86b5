// Attention of few new tokens per sequence over a paged cache of f32 (single tokens, drafts): units of up to eight pairs of token and head.
//
// Up to four pairs read every key and value once and HBM bounds them, eight the multiply-adds.  The loads go straight to registers, a step ahead, and no
// warp waits for another one until a unit ends.  L lanes share a key, each with every L-th 16 bytes of it and of its value: a score takes log2(L) shuffles,
// and a lane's sums are those of its own columns.  The 32 / L groups of a warp see different keys and have maxima, weights and sums of their own, joined at the
// unit's end.  A warp's eight keys of a block of 32 lie in one page.  Queries are read from shared memory, a line for all groups.
// Sums are relative to a maximum that may be 2^8 too low: with a maximum that is followed at once, some row of some group had a new one in half of the
// steps (287 us against 239 for 32 single tokens over 1.06 GB).
#include <cfloat>
#include <cstdint>

#include "mgq_paged.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 128, kWarps = 4, kBlock = 32, kWarpKeys = kBlock / kWarps;
constexpr uint32_t kMaxHead = 128;

// Rows of a part in the workspace: four at least, so that parts begin on 16 bytes.
__host__ __device__ constexpr int stored(int rows) { return rows < 4 ? 4 : rows; }
// CTAs of an SM, as their registers allow (eight rows in four: 274 us for 195).
__host__ __device__ constexpr int ctas_per_sm(int rows) { return rows == 8 ? 3 : 4; }

template <int R, int L, int C>                           // rows of a unit, lanes of a key, 16-byte pieces of a lane: heads of up to 4 * L * C
__global__ void __launch_bounds__(kThreads, ctas_per_sm(R)) few_kernel(const AttendArgs a)
{
    constexpr uint32_t G = 32 / L, kSteps = kWarpKeys / G, D = 4 * L * C;        // keys of a step, steps of a block
    __shared__ unsigned long long s_walk[40];
    __shared__ __align__(16) float s_q[R][D], s_o[kWarps][R][D];
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, d = a.d, group = lane / L, part = lane % L;
    pdl_launch_dependents();
    pdl_wait();
    Walk<R, kBlock, R == 1 ? 1 : 2> walk;                // a unit's end takes as long as two blocks (one row: one)
    walk.begin(a, blockIdx.x, gridDim.x, s_walk);
    if (t == 0) clear_parts(a, blockIdx.x);

    Segment g;
    while (walk.next(a, g)) {
        const uint32_t pairs = g.tokens * g.heads;
        __syncthreads();                                 // the unit before has used what is written now
        for (uint32_t i = t; i < R * D; i += kThreads) {
            const uint32_t r = i / D, c = i % D, token = r / g.heads, head = r - token * g.heads;
            s_q[r][c] = r < pairs && c < d ? static_cast<const float *>(a.q)[(size_t)(g.row0 + token) * a.q_pitch + (size_t)(g.head0 + head) * d + c] * a.scale_log2 : 0.f;
        }
        __syncthreads();
        float m[R], l[R], o[R][4 * C];
        int pos[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            m[r] = -FLT_MAX;                             // differences stay numbers; a score of -inf has no weight
            l[r] = 0.f;
            pos[r] = (uint32_t)r < pairs ? g.pos0 + (int)(r / g.heads) : -1;
#pragma unroll
            for (int e = 0; e < 4 * C; e++) o[r][e] = 0.f;
        }
        const uint32_t steps = max(g.end, g.begin) * kSteps - g.begin * kSteps;
        const int last = min(g.len, g.pos0 + (int)g.tokens);                     // keys that some row sees come before
        auto first_key = [&](uint32_t i) { return (int)((g.begin + i / kSteps) * kBlock + warp * kWarpKeys + i % kSteps * G); };
        auto page_of = [&](uint32_t i) {
            const int key = first_key(i);
            return i < steps && key < last ? g.table[(uint32_t)key >> a.page_shift] : 0xFFFFFFFFu;
        };
        float4 k[2][C], v[2][C];
        bool there[2];
        auto load = [&](uint32_t i, uint32_t page, int at) {
            const int key = first_key(i) + (int)group;
            there[at] = page < a.pages && key < last;
            const size_t from = ((((size_t)page << a.page_shift) + (key & ((1u << a.page_shift) - 1))) * a.kv_heads + g.kv) * d + 4 * part;
#pragma unroll
            for (int c = 0; c < C; c++) {
                k[at][c] = v[at][c] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (there[at] && 4 * part + 4 * L * c < d) {
                    k[at][c] = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(a.k) + from + 4 * L * c));
                    v[at][c] = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(a.v) + from + 4 * L * c));
                }
            }
        };
        auto use = [&](uint32_t i, int at) {
            const int key = first_key(i) + (int)group;
            float s[R];
#pragma unroll
            for (int r = 0; r < R; r++) {
                s[r] = 0.f;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const float4 q = *reinterpret_cast<const float4 *>(&s_q[r][4 * part + 4 * L * c]);
                    s[r] = fmaf(q.x, k[at][c].x, fmaf(q.y, k[at][c].y, fmaf(q.z, k[at][c].z, fmaf(q.w, k[at][c].w, s[r]))));
                }
            }
#pragma unroll
            for (int x = 1; x < L; x *= 2)
#pragma unroll
                for (int r = 0; r < R; r++) s[r] += __shfl_xor_sync(0xffffffffu, s[r], x);
            const int key0 = first_key(i);
            bool masked = false;                         // some row does not see a key that is there
            if (!(key0 + (int)G <= last && key0 + (int)G - 1 <= g.pos0 && __all_sync(0xffffffffu, there[at]) && !(a.window && key0 <= last - 1 - (int)a.window))) {
                bool hidden = false;
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const bool seen = there[at] && key <= pos[r] && (!a.window || key > pos[r] - (int)a.window);
                    hidden |= there[at] && !seen && (uint32_t)r < pairs;
                    s[r] = seen ? s[r] : -INFINITY;
                }
                masked = __any_sync(0xffffffffu, hidden);
            }
            bool grows = false;
#pragma unroll
            for (int r = 0; r < R; r++) grows |= s[r] > m[r] + 8.f;
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float top = s[r] > m[r] + 8.f ? s[r] : m[r], keep = exp2_fast(m[r] - top);
                    l[r] *= keep;
                    m[r] = top;
#pragma unroll
                    for (int e = 0; e < 4 * C; e++) o[r][e] *= keep;
                }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float w = exp2_fast(s[r] - m[r]);
                l[r] += w;
                if (masked && w == 0.f) continue;        // what a row does not see stays out, infinities and NaN too
#pragma unroll
                for (int c = 0; c < C; c++) {
                    o[r][4 * c] = fmaf(w, v[at][c].x, o[r][4 * c]);
                    o[r][4 * c + 1] = fmaf(w, v[at][c].y, o[r][4 * c + 1]);
                    o[r][4 * c + 2] = fmaf(w, v[at][c].z, o[r][4 * c + 2]);
                    o[r][4 * c + 3] = fmaf(w, v[at][c].w, o[r][4 * c + 3]);
                }
            }
            __syncwarp();
        };
        if (steps) {                                     // pages are looked up two steps ahead, keys and values one
            uint32_t page = page_of(0);
            load(0, page, 0);
            page = page_of(1);
            for (uint32_t i = 0; i < steps; i += 2) {
                uint32_t next = page_of(i + 2);
                load(i + 1, page, 1);
                use(i, 0);
                page = page_of(i + 3);
                load(i + 2, next, 0);
                use(i + 1, 1);
            }
        }
        // the groups of a warp, then the warps
#pragma unroll
        for (int x = L; x < 32; x *= 2)
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float top = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], x)), keep = l[r] != 0.f ? exp2f(m[r] - top) : 0.f;
                m[r] = top;
                l[r] *= keep;
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
#pragma unroll
                for (int e = 0; e < 4 * C; e++) {
                    const float mine = keep != 0.f ? o[r][e] * keep : 0.f;
                    o[r][e] = mine + __shfl_xor_sync(0xffffffffu, mine, x);
                }
            }
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (lane == 0) {
                s_m[warp][r] = m[r];
                s_l[warp][r] = l[r];
            }
            if (group == 0)
#pragma unroll
                for (int c = 0; c < C; c++)
                    *reinterpret_cast<float4 *>(&s_o[warp][r][4 * part + 4 * L * c]) = make_float4(o[r][4 * c], o[r][4 * c + 1], o[r][4 * c + 2], o[r][4 * c + 3]);
        }
        __syncthreads();
        const bool whole = g.first && g.last;
        float *dst = a.parts + (size_t)part_index(blockIdx.x, g) * stored(R) * (d + 2);
        for (uint32_t i = t; i < pairs * D; i += kThreads) {
            const uint32_t r = i / D, c = i % D, token = r / g.heads, head = r - token * g.heads;
            if (c >= d) continue;
            const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            float sum = 0.f, x = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float keep = s_l[w][r] != 0.f ? exp2f(s_m[w][r] - top) : 0.f;
                sum += keep * s_l[w][r];
                x += keep != 0.f ? keep * s_o[w][r][c] : 0.f;
            }
            if (whole) {
                static_cast<float *>(a.out)[(size_t)(g.row0 + token) * a.out_pitch + (size_t)(g.head0 + head) * d + c] = sum == 0.f ? 0.f : x * (1.f / sum);
            } else {
                dst[r * d + c] = x;
                if (c == 0) {
                    dst[stored(R) * d + 2 * r] = top;
                    dst[stored(R) * d + 2 * r + 1] = sum;
                }
            }
        }
        if (!whole && t == 0) name_part(a, blockIdx.x, g);
    }
}

// Lanes per key for heads of up to 64 and up to 128.
template <int R, int SMALL, int LARGE>
int launch_sized(const AttendArgs &a, cudaStream_t stream)
{
    auto *kernel = a.d <= 64 ? few_kernel<R, SMALL, 16 / SMALL> : few_kernel<R, LARGE, 32 / LARGE>;
    const uint32_t ctas = few_ctas(R);
    if (int rc = launch(kernel, dim3(ctas), dim3(kThreads), 0, stream, a)) return rc;
    return launch_merge<float, stored(R)>(a, ctas, R, stream);
}

}  // namespace

bool few_takes(const AttendArgs &a, int dtype)
{
    auto on = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return dtype == MGQ_FMT_F32 && a.d % 4 == 0 && a.d <= kMaxHead && on(a.k) && on(a.v);
}
size_t few_part_floats(uint32_t rows, uint32_t d) { return (size_t)stored((int)rows) * (d + 2); }
uint32_t few_ctas(uint32_t rows) { return 148u * ctas_per_sm((int)rows); }
// rows: of a unit, 1, 4 or 8.  More lanes per key hold fewer sums each, so that an SM holds more warps, but take more shuffles: 32 single tokens of four
// heads of 128 per key / value head took 239 us with eight lanes (three CTAs per SM) and 221 with sixteen (four), of three heads of 64 53 and 75.  One row takes
// eight: 64 single tokens of 12 heads of 80 (2 GB) 381 us.
int launch_few(const AttendArgs &a, uint32_t rows, cudaStream_t stream)
{
    return rows == 1 ? launch_sized<1, 8, 8>(a, stream) : rows == 4 ? launch_sized<4, 8, 16>(a, stream) : launch_sized<8, 8, 16>(a, stream);
}

}  // namespace mgq
