// C ABI of the operators over a paged cache and of what follows them: argument checks, then the launchers.
#include "mgq_internal.h"

using namespace mgq;

namespace {

bool known(int dtype) { return dtype == MGQ_FMT_F32 || dtype == MGQ_FMT_F16 || dtype == MGQ_FMT_BF16; }
uintptr_t element(int dtype) { return dtype == MGQ_FMT_F32 ? 4 : 2; }
bool odd(const void *p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
// Whether one of several words' or floats' arrays does not begin on 4 bytes.
template <typename... P> bool odd_words(const P *...p) { return (odd(p, 4) || ...); }

int check_pages(const char *what, uint32_t page_size, uint32_t pages)
{
    if (page_size < 8 || page_size > 1024 || (page_size & (page_size - 1))) return fail(MGQ_ERR_SHAPE, "%s: page size %u is not a power of two from 8 to 1024", what, page_size);
    if (pages == 0 || (unsigned long long)pages * page_size >= 0xFFFFFFFFull) return fail(MGQ_ERR_SHAPE, "%s: %u pages of %u tokens", what, pages, page_size);
    return MGQ_OK;
}
int check_table(const char *what, uint32_t sequences, uint32_t page_size, uint32_t pages, uint32_t table_width)
{
    if (int rc = check_pages(what, page_size, pages)) return rc;
    if (sequences == 0 || sequences > MGQ_PAGED_MAX_SEQUENCES) return fail(MGQ_ERR_SHAPE, "%s: %u sequences (1 to %d)", what, sequences, MGQ_PAGED_MAX_SEQUENCES);
    if (table_width == 0 || (unsigned long long)table_width * page_size >= (1ull << 30))
        return fail(MGQ_ERR_SHAPE, "%s: a table of %u pages of %u tokens per sequence", what, table_width, page_size);
    return MGQ_OK;
}
int check_heads(const char *what, uint32_t heads, uint32_t kv_heads, uint32_t head_dim)
{
    if (kv_heads == 0 || head_dim == 0 || head_dim > MGQ_PAGED_MAX_HEAD) return fail(MGQ_ERR_SHAPE, "%s: %u key / value heads of %u (at most %d)", what, kv_heads, head_dim, MGQ_PAGED_MAX_HEAD);
    if (heads % kv_heads != 0) return fail(MGQ_ERR_SHAPE, "%s: %u heads over %u key / value heads", what, heads, kv_heads);
    if ((unsigned long long)heads * head_dim >= (1ull << 31)) return fail(MGQ_ERR_SHAPE, "%s: %u heads of %u", what, heads, head_dim);
    return MGQ_OK;
}

}  // namespace

extern "C" {

int mgq_paged_plan(const uint32_t *cached, const uint32_t *fresh, uint32_t sequences, uint32_t page_size, uint32_t *table, uint32_t table_width, uint32_t *held,
                   const uint32_t *free_pages, uint32_t pages, uint32_t *free_count, uint32_t rows, uint32_t *starts, uint32_t *lengths, uint32_t *positions,
                   uint32_t *slots, uint32_t *lacking, void *stream)
{
    if (!cached || !fresh || !table || !held || !free_pages || !free_count || !starts || !lengths || !positions || !slots || !lacking)
        return fail(MGQ_ERR_NULL, "paged_plan: null pointer");
    if (int rc = check_table("paged_plan", sequences, page_size, pages, table_width)) return rc;
    if (rows == 0 || rows >= (1u << 31)) return fail(MGQ_ERR_SHAPE, "paged_plan: %u rows", rows);
    if (odd_words(cached, fresh, table, held, free_pages, free_count, starts, lengths, positions, slots, lacking)) return fail(MGQ_ERR_ALIGN, "paged_plan: misaligned pointer");
    return launch_paged_plan(cached, fresh, sequences, page_size, table, table_width, held, free_pages, pages, free_count, rows, starts, lengths, positions, slots, lacking,
                             stream);
}

int mgq_paged_trim(const uint32_t *lengths, uint32_t sequences, uint32_t page_size, uint32_t *table, uint32_t table_width, uint32_t *held, uint32_t *free_pages,
                   uint32_t pages, uint32_t *free_count, void *stream)
{
    if (!lengths || !table || !held || !free_pages || !free_count) return fail(MGQ_ERR_NULL, "paged_trim: null pointer");
    if (int rc = check_table("paged_trim", sequences, page_size, pages, table_width)) return rc;
    if (odd_words(lengths, table, held, free_pages, free_count)) return fail(MGQ_ERR_ALIGN, "paged_trim: misaligned pointer");
    return launch_paged_trim(lengths, sequences, page_size, table, table_width, held, free_pages, pages, free_count, stream);
}

int mgq_paged_append(const void *q, const void *k, const void *v, int src_dtype, const uint32_t *positions, const uint32_t *slots, void *q_out, void *k_cache,
                     void *v_cache, int cache_dtype, uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t q_pitch, uint32_t k_pitch,
                     uint32_t v_pitch, uint32_t page_size, uint32_t pages, float theta, void *stream)
{
    if (!k || !v || !positions || !slots || !k_cache || !v_cache || (q && !q_out)) return fail(MGQ_ERR_NULL, "paged_append: null pointer");
    if (!known(cache_dtype) || (src_dtype != MGQ_FMT_F32 && src_dtype != cache_dtype))
        return fail(MGQ_ERR_FORMAT, "paged_append: sources of type %d into a cache of type %d (f32, f16, bf16; sources f32 or the cache's type)", src_dtype, cache_dtype);
    if (int rc = check_pages("paged_append", page_size, pages)) return rc;
    if (int rc = check_heads("paged_append", q ? q_heads : kv_heads, kv_heads, head_dim)) return rc;
    if (q && q_heads == 0) return fail(MGQ_ERR_SHAPE, "paged_append: no query heads");
    if (head_dim % 2) return fail(MGQ_ERR_SHAPE, "paged_append: head_dim %u is odd", head_dim);
    if (rows == 0 || rows >= (1u << 31)) return fail(MGQ_ERR_SHAPE, "paged_append: %u rows", rows);
    if ((q && q_pitch < q_heads * head_dim) || k_pitch < kv_heads * head_dim || v_pitch < kv_heads * head_dim)
        return fail(MGQ_ERR_SHAPE, "paged_append: rows of %u, %u and %u elements are shorter than their heads", q_pitch, k_pitch, v_pitch);
    if (!(theta >= 0.f) || theta > 1e30f) return fail(MGQ_ERR_SHAPE, "paged_append: theta %g", (double)theta);
    const uintptr_t src = element(src_dtype), dst = element(cache_dtype);
    if (odd(q, src) || odd(k, src) || odd(v, src) || odd(q_out, dst) || odd(k_cache, dst) || odd(v_cache, dst) || odd_words(positions, slots))
        return fail(MGQ_ERR_ALIGN, "paged_append: misaligned pointer");
    if (q && q == q_out && (src_dtype != cache_dtype || (rows > 1 && q_pitch != q_heads * head_dim)))
        return fail(MGQ_ERR_SHAPE, "paged_append: queries rotated in place must be of the cache's type and dense");
    return launch_paged_append(q, k, v, src_dtype, positions, slots, q_out, k_cache, v_cache, cache_dtype, rows, q_heads, kv_heads, head_dim, q_pitch, k_pitch, v_pitch,
                               (unsigned long long)pages * page_size, theta, stream);
}

size_t mgq_paged_attention_workspace(uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_fresh, int dtype)
{
    if (!known(dtype) || heads == 0 || max_fresh == 0 || check_heads("paged_attention_workspace", heads, kv_heads, head_dim)) return 0;
    return paged_attention_workspace(head_dim, dtype);
}

int mgq_paged_attention(const void *q, const void *k_cache, const void *v_cache, int dtype, const uint32_t *table, const uint32_t *starts, const uint32_t *lengths,
                        void *out, uint32_t sequences, uint32_t rows, uint32_t max_fresh, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t page_size,
                        uint32_t pages, uint32_t table_width, uint32_t q_pitch, uint32_t out_pitch, float scale, uint32_t window, void *workspace, void *stream)
{
    if (!q || !k_cache || !v_cache || !table || !starts || !lengths || !out || !workspace) return fail(MGQ_ERR_NULL, "paged_attention: null pointer");
    if (!known(dtype)) return fail(MGQ_ERR_FORMAT, "paged_attention: type %d is not f32, f16 or bf16", dtype);
    if (int rc = check_table("paged_attention", sequences, page_size, pages, table_width)) return rc;
    if (int rc = check_heads("paged_attention", heads, kv_heads, head_dim)) return rc;
    if (heads == 0) return fail(MGQ_ERR_SHAPE, "paged_attention: no query heads");
    if (rows == 0 || rows >= (1u << 31) || max_fresh == 0) return fail(MGQ_ERR_SHAPE, "paged_attention: %u rows, at most %u of a sequence", rows, max_fresh);
    if (q_pitch < heads * head_dim || out_pitch < heads * head_dim) return fail(MGQ_ERR_SHAPE, "paged_attention: rows of %u and %u elements are shorter than %u heads of %u", q_pitch, out_pitch, heads, head_dim);
    const uintptr_t e = element(dtype);
    if (odd(q, e) || odd(k_cache, e) || odd(v_cache, e) || odd(out, e) || odd(workspace, 16) || odd_words(table, starts, lengths)) return fail(MGQ_ERR_ALIGN, "paged_attention: misaligned pointer");
    return launch_paged_attention(q, k_cache, v_cache, dtype, table, starts, lengths, out, sequences, rows, max_fresh, heads, kv_heads, head_dim, page_size, pages,
                                  table_width, q_pitch, out_pitch, scale, window, workspace, stream);
}

int mgq_token_probs(const float *logits, uint32_t pitch, const float *temperature, float *out, uint32_t out_pitch, uint32_t rows, uint32_t vocab, void *stream)
{
    if (!logits || !out) return fail(MGQ_ERR_NULL, "token_probs: null pointer");
    if (rows == 0 || rows >= (1u << 31) || vocab == 0 || vocab >= (1u << 31)) return fail(MGQ_ERR_SHAPE, "token_probs: %u rows of %u", rows, vocab);
    if (pitch < vocab || out_pitch < vocab) return fail(MGQ_ERR_SHAPE, "token_probs: rows %u and %u apart are shorter than the vocabulary of %u", pitch, out_pitch, vocab);
    if (odd_words(logits, temperature, out)) return fail(MGQ_ERR_ALIGN, "token_probs: misaligned pointer");
    return launch_token_probs(logits, pitch, temperature, out, out_pitch, rows, vocab, stream);
}

int mgq_verify_drafts(const float *target, uint32_t target_pitch, const float *draft, uint32_t draft_pitch, const uint32_t *tokens, const uint32_t *starts,
                      const float *accept, const float *sample, uint32_t *accepted, uint32_t *next, uint32_t *out, uint32_t sequences, uint32_t rows, uint32_t vocab,
                      void *stream)
{
    if (!target || !tokens || !starts || !accept || !sample || !accepted || !next || !out) return fail(MGQ_ERR_NULL, "verify_drafts: null pointer");
    if (sequences == 0 || sequences >= (1u << 31) || rows == 0 || rows >= (1u << 31) || vocab == 0 || vocab >= (1u << 31))
        return fail(MGQ_ERR_SHAPE, "verify_drafts: %u sequences, %u rows of %u", sequences, rows, vocab);
    if (target_pitch < vocab || (draft && draft_pitch < vocab))
        return fail(MGQ_ERR_SHAPE, "verify_drafts: rows %u and %u apart are shorter than the vocabulary of %u", target_pitch, draft_pitch, vocab);
    if (odd_words(target, draft, tokens, starts, accept, sample, accepted, next, out)) return fail(MGQ_ERR_ALIGN, "verify_drafts: misaligned pointer");
    return launch_verify_drafts(target, target_pitch, draft, draft_pitch, tokens, starts, accept, sample, accepted, next, out, sequences, rows, vocab, stream);
}

}  // extern "C"
