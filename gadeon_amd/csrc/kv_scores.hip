// Attention over the paged KV cache with scores that are capped, biased by distance, or
// masked by documents and prefixes: gd_kv_attn's kernels (kv_attn.h) with what a score
// becomes, and a mask that differs row by row, compiled in.
#include "kv_attn.h"

extern "C" int gd_kv_attn_scored(gd_ctx *ctx, const gd_kv *kv, const gd_seqs *s, const void *q, int64_t q_stride,
                                 const void *gate, int64_t gate_stride, void *out, int x_dtype, int n_head, float scale,
                                 const gd_scores *how) {
    const char *fn = "gd_kv_attn_scored";
    GD_REQUIRE(ctx, how, "%s: null scores", fn);
    // (Where the scores' reciprocals and their products stay numbers.)
    GD_REQUIRE(ctx, how->cap == 0.f || (how->cap >= 1e-30f && how->cap <= 1e30f), "%s: cap %g (0, or 1e-30 .. 1e30)", fn,
               (double)how->cap);
    GD_REQUIRE(ctx, ((uintptr_t)how->slope | (uintptr_t)how->first | (uintptr_t)how->prefix) % 4 == 0,
               "%s: slope, first and prefix must be 4-byte aligned", fn);
    const AttnArgs a{kv, s, q, q_stride, gate, gate_stride, out, x_dtype, n_head, scale};
    const int window = how->window, sinks = window ? how->n_sink : 0;
    if (how->cap == 0.f && !how->slope && !how->first && !how->prefix)
        return gd_kv_attn(ctx, kv, s, q, q_stride, gate, gate_stride, out, x_dtype, n_head, scale, window, how->n_sink);
    // tanh(x) / x over x^2 < 1/4: of degree 4 to 2^-26 of itself, and of degree 3 to 2^-20.
    static const float fine[] = {1.f, -0.333331435918808f, 0.13325878977775574f, -0.05304549261927605f, 0.01724149100482464f};
    static const float f16[] = {1.f, -0.33328160643577576f, 0.13205359876155853f, -0.0447506420314312f, 0.f};
    const float cap = how->cap * LOG2E;
    Scores mask{window, sinks, cap, {}, how->slope, how->first, how->prefix};
    for (int i = 0; i < 5; i++) mask.p[i] = cap * (x_dtype == GD_F32 || !s || !s->row_start ? fine : f16)[i];
    return attn(ctx, fn, a, window, how->n_sink, mask, !how->prefix);
}
