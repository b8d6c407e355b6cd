// The paged KV cache of many sequences, what its kernels share (kv_cache.hip, kv_attn.h,
// kv_scores.hip, kv_pages.hip): a gd_kv and a gd_seqs as the kernels see them, places in
// the planes, and the entries' checks of them.
#pragma once

#include "gd_internal.h"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace {

constexpr int BLK = GD_KV_BLOCK;                 // positions of a scale
constexpr int EXP_BIAS = 127;                    // of a stored exponent (an f32's)
constexpr int EXP_MIN = -24, EXP_MAX = 9;        // f16's least step; 127 2^9 < f16's largest
constexpr int EXP_NAN = 255;                     // a block that took a NaN: every value NaN

// n / d for 0 <= n < 2^31 (d > 0) by a high product: q = (mulhi(mul, n) + n) >> shift.
struct FastDiv {
    uint32_t mul, shift;
    explicit FastDiv(uint32_t d) {
        shift = 0;
        while (((uint64_t)1 << shift) < d) shift++;
        mul = (uint32_t)(((((uint64_t)1 << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(mul, n) + n) >> shift; }
};

// What the kernels need of a gd_kv and a gd_seqs.  Page tables, positions and row
// starts are device data: nothing here trusts them with an address.
struct Cache {
    void *k, *v;
    uint8_t *kx, *vx;
    uint32_t n_pages;
    int HKV, P;
    FastDiv by_page;
};
struct Rows {
    const int32_t *row_start, *pos, *shift, *table;
    int n_rows, n_seq, max_pages;
    uint32_t cap;                                // positions that the tables hold
};

// Rows [r0, r1) of sequence b, the first at position pos (r0 = r1 where it is idle).
struct Seq {
    int r0, r1, pos;
};
__device__ __forceinline__ Seq seq_at(const Rows &s, int b) {
    Seq q;
    q.r0 = s.row_start ? min(max(s.row_start[b], 0), s.n_rows) : b;
    q.r1 = s.row_start ? min(max(s.row_start[b + 1], q.r0), s.n_rows) : b + 1;
    q.pos = s.pos[b];
    if (q.pos < 0) q.r1 = q.r0;
    return q;
}

// The sequence of row n, for the whole wave (-1: none).
__device__ __forceinline__ int seq_of_row(const Rows &s, int n) {
    if (!s.row_start) return n < s.n_seq ? n : -1;
    const int lane = threadIdx.x & 63;
    for (int c = 0; c < s.n_seq; c += 64) {
        const int end = c + lane < s.n_seq ? s.row_start[c + lane + 1] : 0x7fffffff;
        const int before = __popcll(__ballot(end <= n));
        if (before < 64) return c + before < s.n_seq && n >= s.row_start[c + before] ? c + before : -1;
    }
    return -1;
}

// Maximum over a wave, every lane getting it, and running sum over its lanes (by lane
// moves within rows of 16, then rows; the whole wave active).
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, gd_dpp<GD_DPP_XOR1>(v));
    v = fmaxf(v, gd_dpp<GD_DPP_XOR2>(v));
    v = fmaxf(v, gd_dpp<GD_DPP_HALF_MIRROR>(v));
    v = fmaxf(v, gd_dpp<GD_DPP_MIRROR>(v));
    auto row = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
    return fmaxf(fmaxf(row(0), row(16)), fmaxf(row(32), row(48)));
}
__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    v = min(v, __float_as_uint(gd_dpp<GD_DPP_XOR1>(__uint_as_float(v))));
    v = min(v, __float_as_uint(gd_dpp<GD_DPP_XOR2>(__uint_as_float(v))));
    v = min(v, __float_as_uint(gd_dpp<GD_DPP_HALF_MIRROR>(__uint_as_float(v))));
    v = min(v, __float_as_uint(gd_dpp<GD_DPP_MIRROR>(__uint_as_float(v))));
    auto row = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    return min(min(row(0), row(16)), min(row(32), row(48)));
}
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // from 1, 2, 4, 8 lanes below in the row
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = r0 + __builtin_amdgcn_readlane(v, 31);
    const int r2 = r1 + __builtin_amdgcn_readlane(v, 47), row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}

// Unit u of the sequences' units, `count` of them each (count(Seq, b) lane by lane), class by
// class (class_of(Seq, b): 0 .. classes - 1; all in one of more than 64 sequences): its sequence
// b, which is sq, and place k in it, for the whole wave.  False: fewer units than that.
//   Each workgroup walks the sequences before its own, 64 at a time, so that a call's time goes
// with their square: one row each behind 100 positions of codes, 40 heads of 128 on 8, attended
// to in 0.10 ms for 512 sequences, 0.75 for 2048, 8.3 for 8192, 122 for 32768 (without row_start
// 0.04, 0.17, 0.63, 2.4).  MAX_RAGGED (check_seqs) keeps such a call under half a second.
template <int classes, class F, class G>
__device__ __forceinline__ bool unit_at(const Rows &s, int u, F count, G class_of, int &b, int &k, Seq &sq) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int c = 0; c < s.n_seq; c += 64) {
        Seq q = {0, 0, 0};
        if (c + lane < s.n_seq) q = seq_at(s, c + lane);
        const int n = c + lane < s.n_seq ? count(q, c + lane) : 0;
        const int mine = classes > 1 && s.n_seq <= 64 && c + lane < s.n_seq ? class_of(q, c + lane) : 0;
#pragma unroll
        for (int x = 0; x < classes; x++) {
            const int nx = mine == x ? n : 0, sum = wave_scan(nx), all = __builtin_amdgcn_readlane(sum, 63);
            if (u - base < all) {
                const int l = __ffsll((unsigned long long)__ballot(sum > u - base)) - 1;
                b = c + l;
                k = u - base - __builtin_amdgcn_readlane(sum - nx, l);
                sq = {__builtin_amdgcn_readlane(q.r0, l), __builtin_amdgcn_readlane(q.r1, l), __builtin_amdgcn_readlane(q.pos, l)};
                return k >= 0 && k < __builtin_amdgcn_readlane(nx, l);   // (sums past 2^31: no row_start)
            }
            base += all;
        }
    }
    return false;
}

// The page of position p of sequence b, -1 where there is none.
__device__ __forceinline__ int page_of(const Cache &c, const Rows &s, int b, uint32_t p) {
    if (p >= s.cap) return -1;
    const int page = s.table[(int64_t)b * s.max_pages + c.by_page(p)];
    return (uint32_t)page < c.n_pages ? page : -1;
}
__device__ __forceinline__ int slot_of(const Cache &c, uint32_t p) { return (int)(p - c.by_page(p) * c.P); }

// Head h's row of (page, slot) in the planes, in rows of head_dim elements (fewer than
// 2^32, check_kv); its exponent is the one of row / 16.
template <bool I8> __device__ __forceinline__ uint32_t row_at(const Cache &c, int page, int slot, int h) {
    return I8 ? ((uint32_t)page * c.HKV + h) * c.P + slot : ((uint32_t)page * c.P + slot) * c.HKV + h;
}
// 2^e of a stored exponent: 0 for a block never written, NaN for one that took a NaN.
__device__ __forceinline__ float step_of(uint8_t x) {
    return x == EXP_NAN ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)x << 23);
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(uint16_t x) { return gd_h2f(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ uint16_t from_f32(float x) { return gd_f2h(x); }
// ---------------------------------------------------------------- checks

int check_kv(gd_ctx *ctx, const char *fn, const gd_kv *kv, bool planes) {
    GD_REQUIRE(ctx, kv, "%s: null cache", fn);
    GD_REQUIRE(ctx, kv->dtype == GD_F16 || kv->dtype == GD_I8, "%s: cache dtype %d (GD_F16 or GD_I8)", fn, kv->dtype);
    GD_REQUIRE(ctx, kv->head_dim == 128 || kv->head_dim == 256, "%s: head_dim %d (takes 128 or 256)", fn, kv->head_dim);
    GD_REQUIRE(ctx, kv->n_head_kv > 0 && kv->n_head_kv <= 4096, "%s: n_head_kv %d", fn, kv->n_head_kv);
    GD_REQUIRE(ctx, kv->page_size > 0 && kv->page_size <= (1 << 24), "%s: page size %d", fn, kv->page_size);
    GD_REQUIRE(ctx, kv->dtype != GD_I8 || kv->page_size % GD_KV_BLOCK == 0,
               "%s: page size %d of an 8-bit cache is not a multiple of %d", fn, kv->page_size, GD_KV_BLOCK);
    // Rows of head_dim are counted in 32 bits: 512 GiB of codes, more than the card has.
    const int64_t page = (int64_t)kv->page_size * kv->n_head_kv;
    GD_REQUIRE(ctx, kv->n_pages > 0 && kv->n_pages < (1LL << 31) && kv->n_pages < (1LL << 32) / page,
               "%s: %lld pages", fn, (long long)kv->n_pages);
    if (!planes) return GD_OK;
    GD_REQUIRE(ctx, kv->k && kv->v && (kv->dtype != GD_I8 || (kv->k_exp && kv->v_exp)), "%s: null cache plane", fn);
    GD_REQUIRE(ctx, ((uintptr_t)kv->k | (uintptr_t)kv->v) % 16 == 0, "%s: cache planes must be 16-byte aligned", fn);
    return GD_OK;
}

constexpr int64_t MAX_WGS = 1 << 24;             // workgroups of a launch: their threads are counted in 32 bits
constexpr int MAX_RAGGED = 1 << 16;              // sequences of a call with row_start (unit_at)
int check_seqs(gd_ctx *ctx, const char *fn, const gd_seqs *s) {
    GD_REQUIRE(ctx, s, "%s: null sequences", fn);
    GD_REQUIRE(ctx, s->n_seq >= 0 && s->n_rows >= 0 && s->n_rows < MAX_WGS, "%s: %d sequences, %lld rows", fn, s->n_seq,
               (long long)s->n_rows);
    GD_REQUIRE(ctx, s->row_start || s->n_rows == s->n_seq,
               "%s: %lld rows of %d sequences need row_start (one row each without)", fn, (long long)s->n_rows, s->n_seq);
    GD_REQUIRE(ctx, !s->row_start || s->n_seq <= MAX_RAGGED, "%s: %d sequences with row_start (%d at most)", fn, s->n_seq,
               MAX_RAGGED);
    GD_REQUIRE(ctx, s->n_rows == 0 || s->n_seq == 0 || (s->pos && s->page_table), "%s: null positions or page table", fn);
    GD_REQUIRE(ctx, s->max_pages > 0 && s->max_len >= 0, "%s: max_pages %d, max_len %d", fn, s->max_pages, s->max_len);
    return GD_OK;
}

// Memory for the partials of ns key splits, `bytes` each: the attention scratch where it
// holds them, else the context's workspace, which may grow to WS_BYTES, by powers of two so
// that batches that grow seldom do it; ns becomes what there is memory for (1: none needed).
// A recording takes the workspace as it is.
constexpr size_t WS_BYTES = 256u << 20;
int split_scratch(gd_ctx *ctx, size_t bytes, int64_t &ns, float **scratch) {
    size_t most = GD_ATTN_SCRATCH_BYTES;
    void *p = nullptr;
    if (ns > 1 && ns * bytes > most && 2 * bytes <= WS_BYTES) {
        const size_t want = std::min<size_t>(ns * bytes, WS_BYTES / bytes * bytes);
        size_t room = 2 * most;
        while (room < want) room *= 2;
        if (ctx->ws_bytes < want) gd_ctx_workspace_grow(ctx, room);
        const size_t have = std::min(want, ctx->ws_bytes);
        if (have / bytes > std::max<size_t>(1, most / bytes)) {
            const int rc = gd_ctx_workspace(ctx, have, &p);
            if (rc) return rc;
            most = have;
        }
    }
    ns = std::max<int64_t>(1, std::min<int64_t>(ns, most / bytes));
    if (ns > 1 && !p) p = gd_attn_scratch(ctx);
    if (!p) ns = 1;
    *scratch = (float *)p;
    return GD_OK;
}

int check_x(gd_ctx *ctx, const char *fn, int dtype) {
    GD_REQUIRE(ctx, dtype == GD_F32 || dtype == GD_F16, "%s: row dtype %d (GD_F32 or GD_F16)", fn, dtype);
    return GD_OK;
}

Cache cache_of(const gd_kv *kv) {
    return Cache{kv->k, kv->v, kv->k_exp, kv->v_exp, (uint32_t)kv->n_pages, kv->n_head_kv, kv->page_size,
                 FastDiv((uint32_t)kv->page_size)};
}
Rows rows_of(const gd_kv *kv, const gd_seqs *s) {
    const int64_t cap = std::min<int64_t>((int64_t)s->max_pages * kv->page_size, 0x7fffffff);
    return Rows{s->row_start, s->pos, s->rope_shift, s->page_table, (int)s->n_rows, s->n_seq, s->max_pages, (uint32_t)cap};
}

}  // namespace

// gd_kv_attn in the name of `fn` (kv_cache.hip, which holds the kernels of plain scores).
int gd_kv_attn_plain(gd_ctx *ctx, const char *fn, const gd_kv *kv, const gd_seqs *s, const void *q, int64_t q_stride,
                     const void *gate, int64_t gate_stride, void *out, int x_dtype, int n_head, float scale, int window,
                     int n_sink);

// The template of head dim, cache type and row type that a call runs.
#define GD_KV_PICK(kv, x_dtype, GO) \
    do { \
        if ((kv)->head_dim == 128) { \
            if ((kv)->dtype == GD_I8) { if ((x_dtype) == GD_F32) { GO(128, true, float); } else { GO(128, true, uint16_t); } } \
            else { if ((x_dtype) == GD_F32) { GO(128, false, float); } else { GO(128, false, uint16_t); } } \
        } else { \
            if ((kv)->dtype == GD_I8) { if ((x_dtype) == GD_F32) { GO(256, true, float); } else { GO(256, true, uint16_t); } } \
            else { if ((x_dtype) == GD_F32) { GO(256, false, float); } else { GO(256, false, uint16_t); } } \
        } \
    } while (0)
