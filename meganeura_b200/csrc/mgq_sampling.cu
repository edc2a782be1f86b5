// From logits to tokens for rows of many sequences: probabilities with a temperature per row (mgq_token_probs) and the verification
// of drafted tokens against the target's probabilities with given random numbers (mgq_verify_drafts).
//
// Both stream rows of a vocabulary (150000 f32, 0.6 MB) and are bound by HBM when there are many rows, by latency when there are few.
// A row is shared out over a cluster of up to eight CTAs whose sums meet through distributed shared memory.
#include <cfloat>
#include <cstdint>

#include "mgq_launch.cuh"

namespace mgq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kHold = 4;                                 // groups of four values that a thread reads at once
constexpr uint32_t kGroup = 4 * kThreads, kSlice = kHold * kGroup;

// Four values of a row from column c on; `fill` behind its end.  LAST: they are not read again.
template <bool WIDE, bool LAST>
__device__ __forceinline__ void read4(const float *row, uint32_t c, uint32_t end, float fill, float (&v)[4])
{
    if (WIDE) {
        float4 q = make_float4(fill, fill, fill, fill);
        if (c < end) q = LAST ? __ldcs(reinterpret_cast<const float4 *>(row + c)) : *reinterpret_cast<const float4 *>(row + c);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = c + e < end ? row[c + e] : fill;
    }
}

// ---------------------------------------------------------------- probabilities
// p_i = exp((l_i - m) / t) / sum; t <= 0 (or NaN): 1 for the lowest index among the largest logits.  NaN logits count as -inf; where
// the largest is +inf, those that are share the row.  Rows without a finite or +inf logit are all zero.
// A slice of up to 8192 values stays in registers (HELD): few rows over many CTAs, or small vocabularies.  Longer ones are read once for maximum and
// sum, running together as in attention, and again for the result, which finds them in L2 (the rows in flight take 90 of its
// 126 MB).  Keeping 320 rows of 151936 in the registers of clusters of 8 or 16 CTAs took 170 and 210 us: their loads come in bursts between barriers.
template <bool WIDE, bool HELD>
__global__ void __launch_bounds__(kThreads, 3) probs_kernel(const float *logits, uint32_t pitch, const float *temperature, float *out, uint32_t out_pitch, uint32_t vocab)
{
    __shared__ float s_part[2][kWarps], x_max, x_sum;
    __shared__ uint32_t x_at;
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, part = blockIdx.y, parts = gridDim.y;
    const uint32_t each = ((vocab + parts - 1) / parts + 3) / 4 * 4, begin = min(part * each, vocab), end = min(begin + each, vocab);
    if (t == 0) x_at = 0xFFFFFFFFu;
    pdl_launch_dependents();
    pdl_wait();
    const float *row = logits + (size_t)blockIdx.x * pitch;
    float *dst = out + (size_t)blockIdx.x * out_pitch;
    float v[kHold][4];
    auto fetch = [&](uint32_t c0) {                      // NaN becomes -inf
#pragma unroll
        for (int k = 0; k < kHold; k++) {
            read4<WIDE, HELD>(row, c0 + k * kGroup + 4 * t, end, -INFINITY, v[k]);
#pragma unroll
            for (int e = 0; e < 4; e++) v[k][e] = fmaxf(v[k][e], -INFINITY);
        }
    };
    auto largest = [&]() {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kHold; k++) m = fmaxf(m, fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3])));
        return m;
    };
    fetch(begin);
    const float temp = temperature ? temperature[blockIdx.x] : 1.f;
    const bool greedy = !(temp > 0.f);
    // exponents of 2; the difference first, which is exact near the maximum however large that is, and half of it, which no two finite numbers make
    // infinite.  The factor is neither infinite, so that no difference of 0 becomes NaN, nor 0 (a temperature of +inf: the smallest number, with which all
    // finite differences weigh 2^-1e-6 at least), so that -inf stays -inf.
    const float inv = greedy ? 0.f : fmaxf(fminf(2.8853900817779268f / temp, FLT_MAX), 1.4e-45f);
    auto exponent = [&](float x, float m) { return fmaf(x, 0.5f, -0.5f * m) * inv; };
    auto weights = [&](float m) {                        // their sum, relative to a finite maximum
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kHold; k++)
            sum += (exp2_fast(exponent(v[k][0], m)) + exp2_fast(exponent(v[k][1], m))) + (exp2_fast(exponent(v[k][2], m)) + exp2_fast(exponent(v[k][3], m)));
        return sum;
    };
    auto finite = [](float m) { return fabsf(m) <= FLT_MAX ? m : 0.f; };         // sums of rows without a finite maximum are not used

    float m = largest(), sum = 0.f;
    if (!HELD) {
        // a thread's sum is relative to its own maximum, and nothing while that is -inf: the factor would be 2^(the next maximum's size), which can be
        // infinite, and 0 * inf a NaN
        if (!greedy) sum = weights(finite(m));
        for (uint32_t c0 = begin + kSlice; c0 < end; c0 += kSlice) {
            fetch(c0);
            const float top = fmaxf(m, largest());
            if (!greedy) sum = (m > -INFINITY ? sum * exp2_fast(exponent(m, finite(top))) : 0.f) + weights(finite(top));
            m = top;
        }
    }
    const float mine = m;
    m = warp_max(m);
    if (lane == 0) s_part[0][warp] = m;
    __syncthreads();
    m = warp_max(s_part[0][lane % kWarps]);
    if (parts > 1) {
        if (t == 0) x_max = m;
        cluster_sync();
        m = warp_max(cluster_load(&x_max, lane % parts));
    }

    const bool odd = !(fabsf(m) <= FLT_MAX);             // nothing above -inf, or +inf
    uint32_t at = 0xFFFFFFFFu;                           // the greedy choice: of the largest, the lowest
    if (greedy) {                                        // uniform over the cluster
        for (uint32_t c0 = begin; c0 < end; c0 += kSlice) {
            if (!HELD) fetch(c0);
#pragma unroll
            for (int k = kHold - 1; k >= 0; k--)
#pragma unroll
                for (int e = 3; e >= 0; e--) {
                    const uint32_t c = c0 + k * kGroup + 4 * t + e;
                    if (v[k][e] == m && m > -INFINITY && c < at) at = c;
                }
        }
        if (at != 0xFFFFFFFFu) atomicMin(&x_at, at);
        if (parts > 1) cluster_sync();
        else           __syncthreads();
        at = x_at;
        for (uint32_t p = 0; parts > 1 && p < parts; p++) at = min(at, cluster_load(&x_at, p));
    } else {
        if (odd) {                                       // how many are +inf
            sum = 0.f;
            for (uint32_t c0 = begin; c0 < end; c0 += kSlice) {
                if (!HELD) fetch(c0);
#pragma unroll
                for (int k = 0; k < kHold; k++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sum += v[k][e] == INFINITY ? 1.f : 0.f;
            }
        } else {
            sum = HELD ? weights(m) : mine > -INFINITY ? sum * exp2_fast(exponent(mine, m)) : 0.f;
        }
        sum = warp_sum(sum);
        if (lane == 0) s_part[1][warp] = sum;
        __syncthreads();
        sum = warp_sum(lane < kWarps ? s_part[1][lane] : 0.f);
        if (parts > 1) {
            if (t == 0) x_sum = sum;
            cluster_sync();
            sum = warp_sum(lane < parts ? cluster_load(&x_sum, lane) : 0.f);
        }
    }
    const float scale = sum > 0.f ? 1.f / sum : 0.f;
    auto store = [&](uint32_t c0, auto value) {
#pragma unroll
        for (int k = 0; k < kHold; k++) {
            const uint32_t c = c0 + k * kGroup + 4 * t;
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = value(v[k][e], c + e);
            if (WIDE) {
                if (c < end) __stcs(reinterpret_cast<float4 *>(dst + c), make_float4(p[0], p[1], p[2], p[3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c + e < end) __stcs(dst + c + e, p[e]);
            }
        }
    };
    for (uint32_t c0 = begin; c0 < end; c0 += kSlice) {
        if (!HELD && !greedy) fetch(c0);
        if (greedy || odd) store(c0, [&](float x, uint32_t c) { return greedy ? (c == at ? 1.f : 0.f) : x == INFINITY ? scale : 0.f; });
        else               store(c0, [&](float x, uint32_t) { return exp2f(exponent(x, m)) * scale; });
    }
    if (parts > 1) cluster_sync();                       // nobody leaves while its sums are being read
}

// ---------------------------------------------------------------- verification
// Draft i of a sequence (fed as row start + i) is kept while u q(d) < p(d), with p and q from row start + i - 1: the products of
// two f32 are exact in 64 bits.  At the first draft that is not kept the next token is drawn from max(p - q, 0), behind the last
// one from p: the lowest index whose running sum exceeds u times the whole.  Running sums are in 64 bits, because with 150000
// entries an f32 sum is wrong by more than many an entry: per thread and group of four, then warps in order, then CTAs in order.  The warp's
// piece that holds the pick is cut again among all warps: one warp going through it alone, 19 dependent loads one after another, took 23 of 42 us.
struct VerifyArgs {
    const float *target, *draft;
    const uint32_t *tokens, *starts;
    const float *accept, *sample;
    uint32_t *accepted, *next, *out;
    uint32_t target_pitch, draft_pitch, rows, vocab;
};

// What counts of an entry: negative ones, infinities and NaN are nothing.  Positive floats are in order as integers, negative ones behind them all.
__device__ __forceinline__ float mass(float p) { return __float_as_uint(p) <= 0x7F7FFFFFu ? p : 0.f; }

constexpr uint32_t kChunks = 64;                         // of a warp's piece, in the search
constexpr int kBatch = 4;                                // groups of four entries of either row that a thread reads at once
template <bool WIDE>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const VerifyArgs a)
{
    __shared__ double s_sum[kWarps];
    __shared__ double x_sum;
    __shared__ uint32_t s_kept, s_warp;
    __shared__ double s_x, s_chunk[kChunks];
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5, seq = blockIdx.x, part = blockIdx.y, parts = gridDim.y;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t first = min(a.starts[seq], a.rows), last = max(min(a.starts[seq + 1], a.rows), first), n = last - first;
    if (n == 0) {                                        // uniform over the cluster
        if (part == 0 && t == 0) {
            a.accepted[seq] = 0;
            a.next[seq] = MGQ_NO_TOKEN;
        }
        return;
    }
    if (t == 0) s_kept = n - 1;
    __syncthreads();
    for (uint32_t i = t; i + 1 < n; i += kThreads) {
        const uint32_t row = first + i, d = a.tokens[row + 1];
        bool keep = false;
        if (d < a.vocab) {
            const double p = a.target[(size_t)row * a.target_pitch + d], q = a.draft ? (double)a.draft[(size_t)row * a.draft_pitch + d] : 1.0;
            keep = (double)a.accept[row] * q < p;
        }
        if (!keep) {
            atomicMin(&s_kept, i);
            break;
        }
    }
    __syncthreads();
    const uint32_t kept = s_kept, row = first + kept;
    const bool all = kept + 1 == n;
    if (part == 0) {
        if (t == 0) a.accepted[seq] = kept;
        for (uint32_t i = t; i < n; i += kThreads)
            if (i != kept) a.out[first + i] = i < kept ? a.tokens[first + i + 1] : MGQ_NO_TOKEN;
    }
    const uint32_t each = ((a.vocab + parts - 1) / parts + 3) / 4 * 4, begin = min(part * each, a.vocab), end = min(begin + each, a.vocab);
    // a warp takes a contiguous piece of the slice, so that the pieces are in order
    const uint32_t piece = ((end - begin + kWarps - 1) / kWarps + 127) / 128 * 128, w0 = min(begin + warp * piece, end), w1 = min(w0 + piece, end);
    const float *p = a.target + (size_t)row * a.target_pitch, *q = a.draft ? a.draft + (size_t)row * a.draft_pitch : nullptr;
    const uint32_t taboo = !all && !q ? a.tokens[row + 1] : MGQ_NO_TOKEN;
    double total = 0.0, tot[8];
    // first the rest that the draft leaves over; where that is nothing, the target's own row
    for (int pass = all ? 1 : 0; pass < 2; pass++) {
        const bool rest = pass == 0;
        auto read = [&](uint32_t c, uint32_t c1, float (&x)[4], float (&y)[4]) {
            read4<WIDE, false>(p, c, c1, 0.f, x);
            if (rest && q) read4<WIDE, false>(q, c, c1, 0.f, y);
        };
        // x - min(x, y) in 64 bits is exact, and 0 where y is larger
        auto weigh = [&](uint32_t c, const float (&x)[4], const float (&y)[4], double (&w)[4]) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float some = mass(x[e]);
                w[e] = (double)some;
                if (rest) w[e] = q ? w[e] - (double)fminf(some, mass(y[e])) : c + e == taboo ? 0.0 : w[e];
            }
        };
        auto weights = [&](uint32_t c, uint32_t c1, double (&w)[4]) {
            float x[4], y[4] = {0.f, 0.f, 0.f, 0.f};
            read(c, c1, x, y);
            weigh(c, x, y, w);
        };
        double sum = 0.0;
        for (uint32_t c0 = w0 + 4 * lane; c0 < w1; c0 += 128 * kBatch) {
            float x[kBatch][4], y[kBatch][4] = {};
#pragma unroll
            for (int k = 0; k < kBatch; k++) read(c0 + 128 * k, w1, x[k], y[k]);
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                double w[4];
                weigh(c0 + 128 * k, x[k], y[k], w);
                sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        __syncthreads();                                 // the pass before has read these
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        double whole = 0.0;
        for (int w = 0; w < kWarps; w++) whole += s_sum[w];
        if (parts > 1) {
            if (t == 0) x_sum = whole;
            cluster_sync();
        }
        total = 0.0;
        double base = 0.0;
        for (uint32_t i = 0; i < 8; i++) {
            tot[i] = i < parts ? (parts > 1 ? cluster_load(&x_sum, i) : whole) : 0.0;
            if (i == part) base = total;
            total += tot[i];
        }
        if (parts > 1) cluster_sync();                   // read before the next pass writes, and before anybody leaves
        if (!(total > 0.0)) continue;
        // u times the whole lies in exactly one CTA's share; at the whole itself (u = 1) it is the last one with any
        float u = a.sample[seq];
        u = u > 0.f ? fminf(u, 1.f) : 0.f;
        const double x = (double)u * total;
        uint32_t owner = 0;
        double run = 0.0;
        bool found = false;
        for (uint32_t i = 0; i < 8; i++) {
            if (tot[i] > 0.0 && !found) {
                owner = i;
                found = x < run + tot[i];
            }
            run += tot[i];
        }
        if (owner != part) return;
        if (t == 0) {
            double left = x - base;
            uint32_t pick = 0;
            for (int w = 0; w < kWarps; w++)
                if (s_sum[w] > 0.0) pick = w;            // the last with any, should rounding leave `left` at the end
            for (int w = 0; w < kWarps; w++) {
                if (s_sum[w] > 0.0 && left < s_sum[w]) { pick = w; break; }
                if ((uint32_t)w < pick) left -= s_sum[w];
            }
            s_warp = pick;
            s_x = left;
        }
        __syncthreads();
        // chunks of 128 columns or a multiple, 64 at most
        const uint32_t p0 = min(begin + s_warp * piece, end), p1 = min(p0 + piece, end), step = (piece / 128 + kChunks - 1) / kChunks * 128, chunks = (p1 - p0 + step - 1) / step;
        for (uint32_t i = warp; i < chunks; i += kWarps) {
            const uint32_t c1 = min(p0 + (i + 1) * step, p1);
            double own = 0.0;
            for (uint32_t c = p0 + i * step + 4 * lane; c < c1; c += 128) {
                double w[4];
                weights(c, c1, w);
                own += (w[0] + w[1]) + (w[2] + w[3]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
            if (lane == 0) s_chunk[i] = own;
        }
        __syncthreads();
        if (warp != 0) return;
        double left = s_x;
        uint32_t chosen = 0;
        for (uint32_t i = 0; i < chunks; i++)
            if (s_chunk[i] > 0.0) chosen = i;
        for (uint32_t i = 0; i < chunks; i++) {
            if (s_chunk[i] > 0.0 && left < s_chunk[i]) { chosen = i; break; }
            if (i < chosen) left -= s_chunk[i];
        }
        const uint32_t c_end = min(p0 + (chosen + 1) * step, p1);
        uint32_t token = MGQ_NO_TOKEN, highest = MGQ_NO_TOKEN;
        for (uint32_t c0 = p0 + chosen * step; c0 < c_end && token == MGQ_NO_TOKEN; c0 += 128) {
            double w[4];
            weights(c0 + 4 * lane, c_end, w);            // zeros behind the chunk
            const double own = (w[0] + w[1]) + (w[2] + w[3]);
            double upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double below = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += below;
            }
            double at = upto - own;                      // exclusive
            uint32_t mine = MGQ_NO_TOKEN, top = MGQ_NO_TOKEN;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                at += w[e];
                if (w[e] > 0.0) {
                    top = c0 + 4 * lane + e;
                    if (mine == MGQ_NO_TOKEN && at > left) mine = top;
                }
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, mine != MGQ_NO_TOKEN), any = __ballot_sync(0xffffffffu, top != MGQ_NO_TOKEN);
            if (any) highest = __shfl_sync(0xffffffffu, top, 31 - __clz(any));
            if (hit) token = __shfl_sync(0xffffffffu, mine, __ffs(hit) - 1);
            left -= __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) {
            const uint32_t pick = token != MGQ_NO_TOKEN ? token : highest;
            a.next[seq] = pick;
            a.out[row] = pick;
        }
        return;
    }
    if (part == 0 && t == 0) {                           // neither the rest nor the row has any mass
        a.next[seq] = MGQ_NO_TOKEN;
        a.out[row] = MGQ_NO_TOKEN;
    }
}

bool aligned16(const void *p, uint32_t pitch) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch % 4 == 0; }

// CTAs per row: four where there are many, more for few, so that all SMs take part.
uint32_t probs_parts(uint32_t rows, uint32_t vocab)
{
    uint32_t parts = 1;
    while (parts < 8 && vocab > parts * kGroup && (parts < 4 ? vocab > parts * kSlice || rows * parts < 296 : rows * parts < 296)) parts *= 2;
    return parts;
}
// The rows of all sequences at once on the SMs: two CTAs each.
uint32_t verify_parts(uint32_t sequences, uint32_t vocab)
{
    uint32_t parts = 1;
    while (parts < 8 && sequences * parts * 2 <= 296 && vocab > parts * kGroup) parts *= 2;
    return parts;
}

}  // namespace

int launch_token_probs(const float *logits, uint32_t pitch, const float *temperature, float *out, uint32_t out_pitch, uint32_t rows, uint32_t vocab, void *stream)
{
    const uint32_t parts = probs_parts(rows, vocab);
    const bool wide = vocab % 4 == 0 && aligned16(logits, pitch) && aligned16(out, out_pitch), held = vocab <= parts * kSlice;
    auto *kernel = wide ? (held ? probs_kernel<true, true> : probs_kernel<true, false>) : (held ? probs_kernel<false, true> : probs_kernel<false, false>);
    return launch_clustered(kernel, dim3(rows, parts), dim3(kThreads), parts, 0, static_cast<cudaStream_t>(stream), logits, pitch, temperature, out, out_pitch, vocab);
}

int launch_verify_drafts(const float *target, uint32_t target_pitch, const float *draft, uint32_t draft_pitch, const uint32_t *tokens, const uint32_t *starts,
                         const float *accept, const float *sample, uint32_t *accepted, uint32_t *next, uint32_t *out, uint32_t sequences, uint32_t rows,
                         uint32_t vocab, void *stream)
{
    const VerifyArgs a{target, draft, tokens, starts, accept, sample, accepted, next, out, target_pitch, draft_pitch, rows, vocab};
    const uint32_t parts = verify_parts(sequences, vocab);
    const bool wide = vocab % 4 == 0 && aligned16(target, target_pitch) && (!draft || aligned16(draft, draft_pitch));
    return launch_clustered(wide ? verify_kernel<true> : verify_kernel<false>, dim3(sequences, parts), dim3(kThreads), parts, 0, static_cast<cudaStream_t>(stream), a);
}

}  // namespace mgq
