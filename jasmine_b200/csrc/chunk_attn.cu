// Attention of new tokens over a paged cache, bf16 or 8-bit: entry points, and which kernel takes which sequence.
#include "chunk_attn.cuh"
#include <math.h>
#include <algorithm>

namespace jsm {

jsm_status cache_view_check(const char* who, CacheView& c, void* pool, void* scales, int n_pages, const int32_t* table, int max_pages, const int32_t* starts,
                            const int32_t* context_lens, int n_seqs, int T, int Hkv, int D);

namespace {
// What runs for a call: chunk_few.cu for sequences of up to few_tokens tokens, the other kernel for the others, if there can be any.
struct Plan {
    int few_tokens;
    bool many;
    FewPlan few;
    size_t bytes;
};
// Up to 64 rows: groups of 16 rows in the kernel of few read the cache once each, the other kernel once for all of them, with tiles of 128 rows that are mostly empty and a start of its own.
// What both take (us), as if every sequence were as long as the bounds: a page takes a run 1.3 (8-bit 1.2, heads of 64 0.65) and a further piece 5; a key tile 2 to 2.4, what is around it 6.
//                                                                              groups   tiles
//   12 sequences of 2 to 9 tokens in a window of 1024, heads of 64, 8-bit         12.2    23.5
//   8 tokens of 8192 positions, 32 / 8 heads of 128                               20.1    28.7
//   the same of 8 sequences of 2000                                               29      51
//   32 sequences of 16 tokens of 300                                              54      36
//   64 sequences of 8 tokens of 4096, 8-bit (bf16)                               276 (338) 312 (260)
//   64 tokens of 4096 positions, 32 / 32 heads                                    41      27.5
float seen(int max_context, int window, int tokens, int unit) {  // pages or key tiles that so many tokens see at most
    const long long all = ((long long)max_context + unit - 1) / unit;  // (a bound may be INT_MAX: none)
    return (float)(window > 0 ? std::min(all, ((long long)window + tokens + unit - 3) / unit + 1) : all);
}
bool groups_win(int n_seqs, int T, int max_new, int max_context, int Hkv, int G, int D, int window, bool q8) {
    auto parts = [&](int tokens) { return (float)std::min((long long)n_seqs * (((long long)max_new + tokens - 1) / tokens), T / tokens + (long long)n_seqs) * Hkv; };
    const int per = 16 / G, tile = 2 * (128 / G), sms = sm_count();
    const float pages = seen(max_context, window, per, JSM_PAGE_SIZE), run = std::max(2.0f, pages * parts(per) / (2 * sms));
    const float groups = 8.0f + (D == 64 ? 0.65f : q8 ? 1.2f : 1.3f) * run + 5.0f * std::max(0.0f, run / pages - 1.0f);
    return groups < 18.0f + parts(tile) * (6.0f + (q8 ? 2.4f : 2.0f) * seen(max_context, window, tile, 128)) / sms;
}
// Sequences of few rows among others: tiles too where all of them together, contexts half of the bound on average, take the chip no longer than the longest sequence does: they run beside it,
// without two more launches behind it (16 sequences of 1 to 256 tokens: 58 us, with the kernel of few 68; 8 in a window of 512: 24, 34).
bool few_beside(int n_seqs, int T, int max_context, int Hkv, int G, int window, bool q8) {
    const int tile = 2 * (128 / G);
    const float key = q8 ? 2.4f : 2.0f, tiles = seen(max_context, window, tile, 128);
    return (T / tile + (float)n_seqs) * Hkv * (6.0f + key * 0.5f * tiles) <= sm_count() * (6.0f + key * tiles);
}
Plan plan_of(int n_seqs, int T, int max_new, int max_context, int Hkv, int G, int D, int window, bool q8) {
    Plan p;
    const long long most = (long long)max_new * G;
    const int rows = most <= 8 ? 8 : most <= 16 || G > 8 ? 16 : 8;
    if (most > 16 && most <= 64 && G <= 16 && groups_win(n_seqs, T, max_new, max_context, Hkv, G, D, window, q8)) {
        p.few_tokens = max_new;
        p.many = false;
        p.few = chunk_few_plan(n_seqs, T, max_new, max_context, Hkv, G, window, 16, max_new, D, q8);
        p.bytes = p.few.bytes;
        return p;
    }
    p.few_tokens = rows / G;
    p.many = most > 16;
    // (sequences that are all as long as they can be: none has few rows; one that has all the same has tiles)
    if (p.many && ((long long)n_seqs * max_new == T || few_beside(n_seqs, T, max_context, Hkv, G, window, q8))) p.few_tokens = 0;
    p.few = p.few_tokens ? chunk_few_plan(n_seqs, T, max_new, max_context, Hkv, G, window, rows, p.few_tokens, D, q8) : FewPlan{};
    p.bytes = p.few.bytes;
    return p;
}
}  // namespace

}  // namespace jsm

using namespace jsm;

extern "C" size_t jsm_attn_chunk_scratch_bytes(int n_seqs, int T, int max_new, int max_context, int Hq, int Hkv, int D, int window) {
    if (n_seqs <= 0 || T <= 0 || max_new <= 0 || max_context < max_new || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 128 || (D != 64 && D != 128) || window < 0) return 0;
    // (the larger of both kinds of cache)
    return std::max(plan_of(n_seqs, T, max_new, max_context, Hkv, Hq / Hkv, D, window, false).bytes, plan_of(n_seqs, T, max_new, max_context, Hkv, Hq / Hkv, D, window, true).bytes);
}

extern "C" jsm_status jsm_attn_chunk(const void* d_q, int64_t q_row_stride, const void* d_pool, const void* d_scales, int n_pages, const int32_t* d_block_table,
                                     int max_pages, const int32_t* d_starts, const int32_t* d_context_lens, int n_seqs, int T, int max_new, int max_context, int Hq,
                                     int Hkv, int D, int window, float scale, void* d_scratch, size_t scratch_bytes, void* d_out, int64_t out_row_stride,
                                     void* stream) {
    ChunkArgs a{};
    const jsm_status s = cache_view_check("jsm_attn_chunk", a.c, const_cast<void*>(d_pool), const_cast<void*>(d_scales), n_pages, d_block_table, max_pages, d_starts,
                                          d_context_lens, n_seqs, T, Hkv, D);
    if (s != JSM_OK) return s;
    if (D != 64 && D != 128) JSM_FAIL(JSM_UNSUPPORTED, "jsm_attn_chunk: head_dim %d (64 or 128)", D);
    if (Hq <= 0 || Hq % Hkv) JSM_FAIL(JSM_SHAPE, "d_model must be divisible by num_heads (Hq %d, Hkv %d)", Hq, Hkv);
    if (Hq > 65535) JSM_FAIL(JSM_UNSUPPORTED, "jsm_attn_chunk: %d query heads", Hq);
    if (Hq / Hkv > 128) JSM_FAIL(JSM_UNSUPPORTED, "jsm_attn_chunk: %d query heads per kv head (up to 128)", Hq / Hkv);
    if (window < 0) JSM_FAIL(JSM_INVALID_ARG, "jsm_attn_chunk: window %d", window);
    if (!(scale > 0.0f) || scale > 1e30f) JSM_FAIL(JSM_UNSUPPORTED, "jsm_attn_chunk: the softmax scale (%g) must be positive", (double)scale);
    if (T == 0 || n_seqs == 0) return JSM_OK;
    if (max_new <= 0 || max_context < max_new) JSM_FAIL(JSM_INVALID_ARG, "jsm_attn_chunk: up to %d new tokens of contexts up to %d", max_new, max_context);
    if (!d_q || !d_out) JSM_FAIL(JSM_INVALID_ARG, "jsm_attn_chunk: null pointer");
    if (q_row_stride < (int64_t)Hq * D || out_row_stride < (int64_t)Hq * D || q_row_stride % 8 || out_row_stride % 8)
        JSM_FAIL(JSM_INVALID_ARG, "jsm_attn_chunk: rows of %lld and %lld elements for %d heads of %d (multiples of 8)", (long long)q_row_stride, (long long)out_row_stride, Hq, D);
    if ((reinterpret_cast<uintptr_t>(d_q) & 15) || (reinterpret_cast<uintptr_t>(d_out) & 15)) JSM_FAIL(JSM_INVALID_ARG, "jsm_attn_chunk: q and out must be 16-byte aligned");
    a.q = static_cast<const __nv_bfloat16*>(d_q);
    a.out = static_cast<__nv_bfloat16*>(d_out);
    a.q_rs = q_row_stride; a.out_rs = out_row_stride;
    a.T = T; a.max_new = max_new; a.max_context = max_context;
    a.Hq = Hq; a.G = Hq / Hkv; a.window = window;
    a.scale_log2 = scale * 1.4426950408889634f;
    const cudaStream_t st = as_stream(stream);
    const Plan p = plan_of(n_seqs, T, max_new, max_context, Hkv, a.G, D, window, d_scales != nullptr);
    if (p.bytes && (!d_scratch || scratch_bytes < p.bytes || (reinterpret_cast<uintptr_t>(d_scratch) & 15)))
        JSM_FAIL(JSM_INVALID_ARG, "jsm_attn_chunk: %zu bytes of scratch (16-byte aligned), %zu are needed", d_scratch ? scratch_bytes : 0, p.bytes);
    if (p.many) {
        const jsm_status m = chunk_flash_launch(a, p.few_tokens, st);
        if (m != JSM_OK) return m;
    }
    return p.few_tokens ? chunk_few_launch(a, p.few, d_scratch, st) : JSM_OK;
}
