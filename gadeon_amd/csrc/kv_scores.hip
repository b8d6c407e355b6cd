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
        return gd_kv_attn_plain(ctx, fn, kv, s, q, q_stride, gate, gate_stride, out, x_dtype, n_head, scale, window, how->n_sink);
    const ScoreArgs args{window, sinks, how->cap * LOG2E, how->slope, how->first, how->prefix};
    if (how->cap > 0.f && how->cap <= (x_dtype == GD_F32 ? EXP_CAP : EXP_CAP_F16))
        return attn(ctx, fn, a, window, how->n_sink, Scores<true>{args}, !how->prefix);
    return attn(ctx, fn, a, window, how->n_sink, Scores<false>{args}, !how->prefix);
}
