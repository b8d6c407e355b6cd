// The paged KV cache of many sequences: appending rows with the rotation on the
// way, reading rows back, and attention with a sliding window and sinks, over f16
// values or 8-bit codes with a scale for each block of 16 positions and kv head.
//
// The reference serves one conversation at a time (MetalEnc.ropeBatch,
// kvAppendBatch, attnPaged and attnBatch, MetalEnc.swift:560-706, 817-1025) and
// keeps half pages; its attnBatch takes a window for another model family.  Here a
// call serves the rows of many sequences (gd_seqs), each with a page table of its
// own, as the batched GDN step does.
//
// Cache types:
//   GD_F16: [page][slot][n_head_kv][head_dim], what gd_kv_append writes.
//   GD_I8:  codes [page][n_head_kv][slot][head_dim] and, for each 16 slots of a
//           head, one byte e + 127: a code c stands for c 2^e.  e is the least of
//           -24 .. 9 that holds the block's largest value within 127 steps, so the
//           type spans f16's range and every value it holds is an f16 exactly.
#include "kv_attn.h"

namespace {

// A turned value, formed in 64 bits, as the row it would be in 32 (gd_rope's), in T.
// (Opaque: the compiler otherwise rounds the 64 bits to f16 in one step.)
template <typename T> __device__ __forceinline__ T from_f64(double x) {
    float f = (float)x;
    asm("" : "+v"(f));
    return from_f32<T>(f);
}

// ---------------------------------------------------------------- append

// Turns per position of each rotated pair, as fractions of 2^64: the phase of
// position p is p * turn[j] mod 2^64, without rounding whatever p is.
struct Turns {
    uint64_t t[128];
};

// Rotates and appends the rows that fall into one block of 16 positions of a
// sequence (unit blockIdx.x), and turns its query rows: wave w of workgroup y takes
// the heads 4 y + w of the kv heads' keys, then their values, then the query heads (the
// longest work first).
//   A lane holds eight elements of a row as two fours, whose elements make four of the
// rotated pairs (j and j + n_rot / 2, n_rot a multiple of 8) or eight of the dims behind
// them: 64 lanes are four rows of head dim 128 or two of 256, the block's 16 rows that
// many steps, all requested at once (a row at a time 46 us for 2119 rows of 24 / 4 x
// 256, its loads one after the other) and beside them the rows' pages.
//   The cos and sin of the block's positions are formed once a workgroup, and rows turned,
// in 64 bits: from turns in 32 one code in 40 000 came out on the other side of a
// border, and one half in 700 a step off.
//   Bytes bound it, every row read and written once, as far as there are rows enough to
// hide a chain of some 8 us (the unit, its rows, the turns, the block's maximum, codes):
// 2119 f16 rows of 24 / 4 heads of 256 into codes move 65 MB in 19 us, 3.4 TB/s; 1000 f32
// rows of 16 / 8 heads of 128 into halves 29 MB in 11.
//   f32 rows of 128 into codes are held to six waves a SIMD (two registers: 2000 rows of 40 / 8
// heads 31.4 us at five, 30.2 at six).
template <int HD, bool I8, bool VEC, typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 128 && I8 && VEC && sizeof(T) == 4 ? 6 : 1)))
void k_append(Cache c, Rows s, Turns turns, const T *q, int64_t q_stride, T *q_out, int H, const T *kx, int64_t k_stride,
              const T *vx, int64_t v_stride, int n_rot) {
    // Lanes of a row, rows of a step, steps; pairs of a lane are VEC ? 4 : 1 wide.
    constexpr int LPR = HD / 8, RPS = 64 / LPR, ST = BLK / RPS;
    extern __shared__ double2 cs[];              // [BLK][n_rot / 2]
    const int t = threadIdx.x, lane = t & 63, half = n_rot / 2;
    int b, blk;
    Seq sq;
    auto blocks = [](const Seq &q, int) {
        return q.r1 > q.r0 ? (int)(((uint32_t)q.pos % BLK + (uint32_t)(q.r1 - q.r0) + BLK - 1) / BLK) : 0;
    };
    if (!s.row_start) {                          // a row, and a block, each
        b = blockIdx.x;
        blk = 0;
        sq = seq_at(s, b);
        if (sq.pos < 0) return;
    } else if (!unit_at<1>(s, blockIdx.x, blocks, [](const Seq &, int) { return 0; }, b, blk, sq)) {
        return;
    }
    // The block's new rows: n of them from row r on, the first at slot `off` of it.
    const int off = blk ? 0 : sq.pos % BLK;
    const int skip = blk ? blk * BLK - sq.pos % BLK : 0;
    const int r = sq.r0 + skip, n = min(BLK - off, sq.r1 - r);
    const uint32_t p = (uint32_t)sq.pos + (uint32_t)skip;
    const int hs = blockIdx.y * 4 + (t >> 6), H2 = H + 2 * c.HKV;
    const bool is_k = hs < c.HKV, is_q = hs >= 2 * c.HKV;
    const int h = is_q ? hs - 2 * c.HKV : is_k ? hs : hs - c.HKV;
    // This lane's place: row `lr` of a step's, elements d0 .. and d1 .. of it.  Without VEC
    // (any n_rot, any alignment) element e of both is a pair of its own.
    const int lr = lane / LPR, j0 = 4 * (lane % LPR);
    auto dims = [&](int e, int &d0, int &d1) {
        const int j = j0 + e;
        d0 = j < half ? j : n_rot + 2 * (j - half);
        d1 = j < half ? j + half : d0 + 1;
        if (VEC && j0 >= half) {
            d0 = n_rot + 2 * (j0 - half) + e;
            d1 = d0 + 4;
        }
    };
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 x0[ST], x1[ST];
    if (hs < H2) {
        const T *src = (is_q ? q + r * q_stride : is_k ? kx + r * k_stride : vx + r * v_stride) + (int64_t)h * HD;
        const int64_t stride = is_q ? q_stride : is_k ? k_stride : v_stride;
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const T *row = src + min(i * RPS + lr, n - 1) * stride;
            if constexpr (VEC) {
                int d0, d1;
                dims(0, d0, d1);
                x0[i] = *(const T4 *)(row + d0);
                x1[i] = *(const T4 *)(row + d1);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    int d0, d1;
                    dims(e, d0, d1);
                    x0[i][e] = row[d0];
                    x1[i][e] = row[d1];
                }
            }
        }
    }
    // The rows' pages, and the exponent of a block that has rows before these.
    int page[I8 ? 1 : ST], had = 0;
    if (hs < H2 && !is_q) {
#pragma unroll
        for (int i = 0; i < (I8 ? 1 : ST); i++) page[i] = page_of(c, s, b, I8 ? p : p + i * RPS + lr);
        if constexpr (I8)
            if (off && page[0] >= 0) had = (is_k ? c.kx : c.vx)[row_at<true>(c, page[0], slot_of(c, p) - off, h) / BLK];
    }
    const int64_t rp = (int64_t)p + (s.shift ? s.shift[b] : 0);
    for (int i = t; i < n * half; i += 256) {
        const int64_t turn = (int64_t)((uint64_t)(rp + i / half) * turns.t[i % half]);
        double sn, cn;
        sincospi((double)turn * 0x1p-63, &sn, &cn);
        cs[i] = double2{cn, sn};
    }
    __syncthreads();
    if (hs >= H2) return;
    const bool turn = is_q || is_k;
    // Element e of step i, turned where it is one of the rotated.
    auto turned = [&](int i, int e, double &a, double &z) {
        a = to_f32<T>(x0[i][e]), z = to_f32<T>(x1[i][e]);
        const int row = i * RPS + lr, j = j0 + e;
        if (turn && j < half && row < n) {
            const double2 w = cs[row * half + j];
            const double o = a;
            a = o * w.x - z * w.y;
            z = o * w.y + z * w.x;
        }
    };
    // Four results at d0 and four at d1 of a row in memory.
    auto put = [&](auto *y, auto a, auto z) {
        if constexpr (VEC) {
            int d0, d1;
            dims(0, d0, d1);
            *(decltype(a) *)(y + d0) = a;
            *(decltype(z) *)(y + d1) = z;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                int d0, d1;
                dims(e, d0, d1);
                y[d0] = a[e];
                y[d1] = z[e];
            }
        }
    };
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    typedef int8_t i8x4 __attribute__((ext_vector_type(4)));
    if (is_q) {
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const int row = i * RPS + lr;
            if (row >= n) break;
            T4 a4, z4;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                double a, z;
                turned(i, e, a, z);
                a4[e] = from_f64<T>(a);
                z4[e] = from_f64<T>(z);
            }
            put(q_out + ((int64_t)(r + row) * H + h) * HD, a4, z4);
        }
        return;
    }
    void *plane = is_k ? c.k : c.v;
    if constexpr (!I8) {
        // A page may end inside the block.  Values past f16's range are held as its
        // largest.
        auto f16_of = [](double x) { return from_f64<uint16_t>(x > 65504. ? 65504. : x < -65504. ? -65504. : x); };
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const int row = i * RPS + lr;
            if (row >= n) break;
            if (page[i] < 0) continue;
            u16x4 a4, z4;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                double a, z;
                turned(i, e, a, z);
                a4[e] = f16_of(a);
                z4[e] = f16_of(z);
            }
            put((uint16_t *)plane + (uint64_t)row_at<false>(c, page[i], slot_of(c, p + row), h) * HD, a4, z4);
        }
        return;
    } else {
        if (page[0] < 0) return;
        const uint32_t at = row_at<true>(c, page[0], slot_of(c, p) - off, h);
        uint8_t *xp = (is_k ? c.kx : c.vx) + at / BLK;
        int8_t *y = (int8_t *)plane + (uint64_t)at * HD;
        float top = 0.f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < ST; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // (In 32 bits, which holds no 64-bit values till below.)
                const int row = i * RPS + lr, j = j0 + e;
                float a = to_f32<T>(x0[i][e]), z = to_f32<T>(x1[i][e]);
                if (turn && j < half && row < n) {
                    const double2 w = cs[row * half + j];
                    const float cn = (float)w.x, sn = (float)w.y, o = a;
                    a = o * cn - z * sn;
                    z = o * sn + z * cn;
                }
                if (row >= n) a = z = 0.f;
                top = fmaxf(top, fmaxf(fabsf(a), fabsf(z)));
                nan |= a != a || z != z;
            }
        const float mine = top;
        top = wave_max(top);
        // 127 2^ex holds top.  A turned key's is off by three roundings of its pair's larger
        // element, 1.5 times top at most: 5 steps of 32 bits.  So with one of them near the
        // border the lesser exponent is taken here, and looked at again in 64 bits behind the codes.
        const uint32_t bits = __float_as_uint(top), frac = bits & 0x7fffffu;
        const bool near = is_k && frac - (0x7e0000u - 32) <= 64u && __any(j0 < half && __float_as_uint(mine) >= bits - 64);
        int ex = (int)(bits >> 23) - 127 - 6 + (frac > 0x7e0000u && !near);
        ex = min(max(ex, EXP_MIN), EXP_MAX);
        nan = __any(nan);
        int ex0 = EXP_MIN;
        if (off) {
            nan |= had == EXP_NAN;
            ex0 = min(max(had - EXP_BIAS, EXP_MIN), EXP_MAX);
            ex = max(ex, ex0);
        }
        // The exponent, and the rows before these: they keep their codes, or take the greater step.
        auto settle = [&] {
            if (off && ex > ex0) {
                const float f = __uint_as_float((uint32_t)(127 + ex0 - ex) << 23);
                for (int i = lane; i < off * (HD / 4); i += 64) {
                    i8x4 o = ((const i8x4 *)y)[i];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = (int8_t)rintf(o[e] * f);
                    ((i8x4 *)y)[i] = o;
                }
            }
            if (lane == 0) *xp = nan ? EXP_NAN : (uint8_t)(ex + EXP_BIAS);
        };
        if (!near) settle();
        auto code = [](double x, int ex) {
            const double inv = __longlong_as_double((long long)(1023 - ex) << 52);
            return (int8_t)(int)fmin(fmax(rint(x * inv), -127.0), 127.0);
        };
#pragma unroll
        for (int i = 0; i < ST; i++) {
            const int row = i * RPS + lr;
            if (row >= n) break;
            i8x4 a4, z4;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                double a, z;
                turned(i, e, a, z);
                a4[e] = code(a, ex);
                z4[e] = code(z, ex);
            }
            put(y + (off + row) * HD, a4, z4);
        }
        if (!near) return;
        // (The rows read once more: rare, and done without the registers that hold them.)
        auto pairs = [&](auto f) {
#pragma unroll 1
            for (int row = lr; row < n; row += RPS)
#pragma unroll 2
                for (int e = 0; e < 4; e++) {
                    const T *x = kx + (r + row) * k_stride + (int64_t)h * HD;
                    int d0, d1;
                    dims(e, d0, d1);
                    const double o = to_f32<T>(x[d0]), u = to_f32<T>(x[d1]);
                    const double2 w = j0 + e < half ? cs[row * half + j0 + e] : double2{1., 0.};
                    f((off + row) * HD + d0, o * w.x - u * w.y);
                    f((off + row) * HD + d1, o * w.y + u * w.x);
                }
        };
        bool more = false;
        const double most = 127. * __longlong_as_double((long long)(1023 + ex) << 52);
        pairs([&](int, double x) { more |= fabs(x) > most; });
        if (__any(more) && ex < EXP_MAX) {
            ex++;
            pairs([&](int at, double x) { y[at] = code(x, ex); });
        }
        settle();
    }
}

// ---------------------------------------------------------------- read

// Rows of the cache as values, eight dims a thread: thread i over [row][K then V]
// [head][HD / 8].  Rows of pages that are not there come out as zeros.  Its launch bounds it
// up to some hundred rows (3 us), bytes beyond (2300 rows of 4 heads of 256, 14 MB, 5.4 us).
template <int HD, bool I8, typename T>
__global__ __launch_bounds__(256) void k_read(Cache c, Rows s, T *k_out, T *v_out) {
    const int per = 2 * c.HKV * (HD / 8), n = blockIdx.x;
    const int b = seq_of_row(s, n);
    if (b < 0) return;
    const Seq sq = seq_at(s, b);
    if (n < sq.r0 || n >= sq.r1) return;
    const uint32_t p = (uint32_t)sq.pos + (uint32_t)(n - sq.r0);
    const int page = page_of(c, s, b, p), slot = slot_of(c, p);
    for (int i = threadIdx.x; i < per; i += 256) {
        const int d = i % (HD / 8) * 8, hh = i / (HD / 8), h = hh % c.HKV;
        const bool is_k = hh < c.HKV;
        T *y = (is_k ? k_out : v_out) + ((int64_t)n * c.HKV + h) * HD + d;
        float f[8] = {};
        if (page >= 0) {
            const uint32_t row = row_at<I8>(c, page, slot, h);
            if constexpr (I8) {
                const int8_t *x = (const int8_t *)(is_k ? c.k : c.v) + (uint64_t)row * HD + d;
                const float st = step_of((is_k ? c.kx : c.vx)[row / BLK]);
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = (float)x[e] * st;
            } else {
                const uint16_t *x = (const uint16_t *)(is_k ? c.k : c.v) + (uint64_t)row * HD + d;
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = gd_h2f(x[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = from_f32<T>(f[e]);
    }
}

// A positive number modulo 1 as a fraction of 2^64, from its 64 bits and exponent (floorl and
// a conversion a pair took 3 us of a call's 8.3 at 128 rotated dims).
uint64_t fraction(long double x) {
    int up;
    const uint64_t bits = (uint64_t)(frexpl(x, &up) * 0x1p64L);          // x = bits 2^(up - 64)
    return up > 63 || up < -63 ? 0 : up >= 0 ? bits << up : bits >> -up;
}

}  // namespace

// ---------------------------------------------------------------- C ABI
// Arguments are checked before the context is looked at, so that a null one shows
// what is wrong with them too (gd_last_error(NULL)).

static size_t exp_bytes(const gd_kv *kv) {
    return (size_t)kv->n_pages * kv->n_head_kv * (kv->page_size / GD_KV_BLOCK);
}

extern "C" int gd_kv_alloc(gd_ctx *ctx, int dtype, int n_head_kv, int head_dim, int page_size, int64_t n_pages,
                           gd_kv *kv) {
    GD_REQUIRE(ctx, kv, "gd_kv_alloc: null out pointer");
    *kv = gd_kv{nullptr, nullptr, nullptr, nullptr, n_pages, dtype, n_head_kv, head_dim, page_size};
    int rc = check_kv(ctx, "gd_kv_alloc", kv, false);
    if (rc) return rc;
    GD_CHECK_CTX(ctx);
    const size_t plane = (size_t)n_pages * page_size * n_head_kv * head_dim * (dtype == GD_F16 ? 2 : 1);
    void *p[4] = {};
    const int n = dtype == GD_I8 ? 4 : 2;
    for (int i = 0; i < n && !rc; i++) {
        const size_t bytes = ((i < 2 ? plane : exp_bytes(kv)) + 15) / 16 * 16;
        rc = gd_alloc(ctx, bytes, &p[i]);
        if (!rc) rc = gd_fill_u32(ctx, p[i], 0u, bytes / 4);
    }
    kv->k = p[0];
    kv->v = p[1];
    kv->k_exp = (uint8_t *)p[2];
    kv->v_exp = (uint8_t *)p[3];
    if (rc) {
        const std::string why = ctx->err;
        gd_kv_free(ctx, kv);
        ctx->err = why;
    }
    return rc;
}

extern "C" int gd_kv_free(gd_ctx *ctx, gd_kv *kv) {
    GD_CHECK_CTX(ctx);
    if (!kv) return GD_OK;
    int rc = GD_OK;
    for (void *p : {kv->k, kv->v, (void *)kv->k_exp, (void *)kv->v_exp}) {
        const int e = gd_free(ctx, p);
        rc = rc ? rc : e;
    }
    kv->k = kv->v = nullptr;
    kv->k_exp = kv->v_exp = nullptr;
    return rc;
}

extern "C" int gd_kv_append_rope(gd_ctx *ctx, const gd_kv *kv, const gd_seqs *s, const void *q, int64_t q_stride,
                                 void *q_out, int n_head, const void *k, int64_t k_stride, const void *v,
                                 int64_t v_stride, int x_dtype, int n_rot, float base) {
    const char *fn = "gd_kv_append_rope";
    int rc;
    if ((rc = check_kv(ctx, fn, kv, true)) || (rc = check_seqs(ctx, fn, s)) || (rc = check_x(ctx, fn, x_dtype))) return rc;
    const int hd = kv->head_dim;
    GD_REQUIRE(ctx, k && v, "%s: null k or v", fn);
    GD_REQUIRE(ctx, k_stride >= (int64_t)kv->n_head_kv * hd && v_stride >= (int64_t)kv->n_head_kv * hd,
               "%s: k and v rows of %d heads overlap at strides %lld, %lld", fn, kv->n_head_kv, (long long)k_stride,
               (long long)v_stride);
    GD_REQUIRE(ctx, n_rot >= 0 && n_rot % 2 == 0 && n_rot <= hd, "%s: n_rot %d must be even and at most head_dim %d", fn,
               n_rot, hd);
    GD_REQUIRE(ctx, n_rot == 0 || (base > 0.f && std::isfinite(base)), "%s: rotation base %g", fn, (double)base);
    const int64_t widest = std::max({q ? q_stride : 0, k_stride, v_stride});
    GD_REQUIRE(ctx, widest < (1LL << 31), "%s: row stride %lld", fn, (long long)widest);
    if (q) {
        GD_REQUIRE(ctx, q_out && n_head > 0 && n_head <= 65536, "%s: q of %d heads without q_out", fn, n_head);
        GD_REQUIRE(ctx, q_stride >= (int64_t)n_head * hd, "%s: q rows of %d heads overlap at stride %lld", fn, n_head,
                   (long long)q_stride);
        const int64_t size = x_dtype == GD_F32 ? 4 : 2, row = (int64_t)n_head * hd;
        const uintptr_t o = (uintptr_t)q_out, o_end = o + s->n_rows * row * size;
        auto apart = [&](const void *x, int64_t stride, int64_t elems) {
            const uintptr_t a = (uintptr_t)x;
            return !s->n_rows || a + ((s->n_rows - 1) * stride + elems) * size <= o || o_end <= a;
        };
        GD_REQUIRE(ctx, (q == q_out && q_stride == row) || apart(q, q_stride, row),
                   "%s: q turned in place needs q_out = q and rows of n_head * head_dim (stride %lld)", fn,
                   (long long)q_stride);
        const int64_t kv_row = (int64_t)kv->n_head_kv * hd;
        GD_REQUIRE(ctx, apart(k, k_stride, kv_row) && apart(v, v_stride, kv_row), "%s: q_out in the place of k or v", fn);
    }
    GD_CHECK_CTX(ctx);
    if (!s->n_rows || !s->n_seq) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    // base^(-2j / n_rot) / (2 pi) of each pair, by one power and its multiples: off by
    // under 2^-57 of itself, which even position 2^31 turns into less than 2^-28 of a turn.
    Turns turns;
    long double turn = 0.159154943091895335768883763372514362L, by = n_rot ? powl(base, -2.0L / n_rot) : 0.0L;
    for (int j = 0; j < n_rot / 2; j++, turn *= by) turns.t[j] = fraction(turn);
    const int H = q ? n_head : 0;
    // Blocks of 16 positions that the rows can touch: rows / 16 and two ends a sequence.
    const int64_t units = std::min<int64_t>(s->n_rows, s->n_rows / BLK + 2 * std::min<int64_t>(s->n_seq, s->n_rows));
    const dim3 grid((unsigned)units, gd_blocks(H + 2 * kv->n_head_kv, 4));
    const unsigned lds = BLK * (n_rot / 2) * sizeof(double2);
    // Fours of a row in one access: what its place, stride and rotated dims allow.
    const int size = x_dtype == GD_F32 ? 4 : 2;
    const bool vec = n_rot % 8 == 0 && (k_stride | v_stride | (q ? q_stride : 0)) % 4 == 0 &&
                     ((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out) % (4 * size) == 0;
#define GD_GO(HD_, I8_, T_) \
    do { \
        auto kernel = vec ? k_append<HD_, I8_, true, T_> : k_append<HD_, I8_, false, T_>; \
        hipLaunchKernelGGL(kernel, grid, dim3(256), lds, ctx->stream, cache_of(kv), rows_of(kv, s), turns, (const T_ *)q, \
                           q_stride, (T_ *)q_out, H, (const T_ *)k, k_stride, (const T_ *)v, v_stride, n_rot); \
    } while (0)
    GD_KV_PICK(kv, x_dtype, GD_GO);
#undef GD_GO
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}

extern "C" int gd_kv_read(gd_ctx *ctx, const gd_kv *kv, const gd_seqs *s, void *k_out, void *v_out, int dtype) {
    const char *fn = "gd_kv_read";
    int rc;
    if ((rc = check_kv(ctx, fn, kv, true)) || (rc = check_seqs(ctx, fn, s)) || (rc = check_x(ctx, fn, dtype))) return rc;
    GD_REQUIRE(ctx, k_out && v_out, "%s: null output", fn);
    GD_REQUIRE(ctx, ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "%s: outputs must be 16-byte aligned", fn);
    GD_CHECK_CTX(ctx);
    if (!s->n_rows || !s->n_seq) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    const dim3 grid((unsigned)s->n_rows);
#define GD_GO(HD_, I8_, T_) \
    hipLaunchKernelGGL((k_read<HD_, I8_, T_>), grid, dim3(256), 0, ctx->stream, cache_of(kv), rows_of(kv, s), \
                       (T_ *)k_out, (T_ *)v_out)
    GD_KV_PICK(kv, dtype, GD_GO);
#undef GD_GO
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}

int gd_kv_attn_plain(gd_ctx *ctx, const char *fn, const gd_kv *kv, const gd_seqs *s, const void *q, int64_t q_stride,
                     const void *gate, int64_t gate_stride, void *out, int x_dtype, int n_head, float scale, int window,
                     int n_sink) {
    const AttnArgs a{kv, s, q, q_stride, gate, gate_stride, out, x_dtype, n_head, scale};
    return attn(ctx, fn, a, window, n_sink, Mask{window, window ? n_sink : 0}, true);
}

extern "C" int gd_kv_attn(gd_ctx *ctx, const gd_kv *kv, const gd_seqs *s, const void *q, int64_t q_stride,
                          const void *gate, int64_t gate_stride, void *out, int x_dtype, int n_head, float scale,
                          int window, int n_sink) {
    return gd_kv_attn_plain(ctx, "gd_kv_attn", kv, s, q, q_stride, gate, gate_stride, out, x_dtype, n_head, scale, window, n_sink);
}
