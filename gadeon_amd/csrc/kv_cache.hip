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
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // from 1, 2, 4, 8 lanes below in the row
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = r0 + __builtin_amdgcn_readlane(v, 31);
    const int r2 = r1 + __builtin_amdgcn_readlane(v, 47), row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}

// Unit u of the sequences' units, `count` of them each (count(Seq) lane by lane), class by
// class (class_of(Seq): 0 .. classes - 1; all in one of more than 64 sequences): its sequence
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
        const int n = c + lane < s.n_seq ? count(q) : 0;
        const int mine = classes > 1 && s.n_seq <= 64 ? class_of(q) : 0;
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
    auto blocks = [](const Seq &q) {
        return q.r1 > q.r0 ? (int)(((uint32_t)q.pos % BLK + (uint32_t)(q.r1 - q.r0) + BLK - 1) / BLK) : 0;
    };
    if (!s.row_start) {                          // a row, and a block, each
        b = blockIdx.x;
        blk = 0;
        sq = seq_at(s, b);
        if (sq.pos < 0) return;
    } else if (!unit_at<1>(s, blockIdx.x, blocks, [](const Seq &) { return 0; }, b, blk, sq)) {
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

// ---------------------------------------------------------------- attention

struct Mask {
    int window, sinks;                           // window 0: every key up to the query's own
};

// Four codes as two pairs of halves: byte c ^ 0x80 below 0x64 is the half 1152 + c.
__device__ __forceinline__ void halves(uint32_t codes, f16x2 &a, f16x2 &b) {
    const uint32_t x = codes ^ 0x80808080u;
    const f16x2 off = {(f16)1152.f, (f16)1152.f};
    a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - off;
    b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - off;
}
__device__ __forceinline__ f16x8 halves(uint32_t lo, uint32_t hi) {
    f16x2 a, b, c, d;
    halves(lo, a, b);
    halves(hi, c, d);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The visible keys of the query at position p as blocks of W keys that start at a
// multiple of W: first those of the sinks, then those from the window's first key lo on.
// Key t of a block is seen where t <= p and (t >= lo or t < sinks).
template <int W> struct KeyBlocks {
    uint32_t lo, sinks;
    int ns, n;                                   // blocks of sinks, blocks in all
    // Window of the query at `first` and on, keys up to `last`.
    __device__ __forceinline__ KeyBlocks(const Mask &m, uint32_t first, uint32_t last) {
        lo = m.window && first >= (uint32_t)m.window ? first - m.window + 1 : 0;
        sinks = min((uint32_t)m.sinks, lo);
        ns = (int)min((sinks + W - 1) / W, lo / W);
        n = ns + (lo <= last ? (int)(last / W - lo / W + 1) : 0);
    }
    __device__ __forceinline__ uint32_t start(int j) const { return (uint32_t)(j < ns ? j : j - ns + (int)(lo / W)) * W; }
    // Splits that these blocks are worked in: of `least` blocks or more, `most` at most.
    __device__ __forceinline__ int splits(int most, int least) const { return max(1, min(most, (n + least - 1) / least)); }
};

// Partials of the key splits: sums of head h of row n, split z, at acc [n H + h][most][HD]
// and its (maximum, sum of weights) at ml [n H + h][most], maxima in units of log2; how
// many splits there are at used [n H + h] (1: the row is done, and has no partials).
struct Part {
    float *acc;
    float2 *ml;
    int *used;
};

// How finely keys are split, from the sequences' own lengths (the host knows a bound of
// them alone): the fewest blocks of a split, so that all the splits' workgroups, `groups`
// for each, fill the `slots` that the chip holds at once; and no fewer than what a
// workgroup's start, end and merge cost: for tokens 8 blocks of head dim 128 and 4 of 256
// (one token of 600 positions, us at 4 / 8 / 16 blocks: 40 heads of 128 11.5 / 12.3 / 14.8,
// 24 of 256 on codes 14.3 / 16.5 / 21, on halves 16.3 / 18.9 / 26; 32 of up to 3000 behind an
// append, heads of 128, 28.3 / 25.8 / 27.6), for rows 4 (2 rows behind 8191 of codes, at 2 / 4 /
// 8: 17.3 / 17.3 / 24.1, 16 of 8 sequences 29.2 / 30.7 / 35.0; full chips alike).
constexpr int token_fewest(int hd) { return 1024 / hd; }
constexpr int ROWS_FEWEST = 4;
__device__ __forceinline__ KeyBlocks<32> token_blocks(const Rows &s, const Mask &mask, int pos) {
    return KeyBlocks<32>(mask, (uint32_t)pos, min((uint32_t)pos, s.cap - 1));
}
// From an even share of all blocks a slot, to what lets the splits have a slot each, those
// of half as many blocks or fewer a part of one, their start counted as two blocks, as they
// come last and fill the gaps (unit_at; 64 tokens of up to 8192 positions 41 us, a slot for
// each 59; a mixed batch of prompt chunks 115 and 197; the long ones' workgroups first: 37 and
// 115, k_attn_tokens, k_attn_rows);
// blocks(b, n, u): n blocks in each of sequence b's u units.  Over 64 sequences fill the chip
// as they are, and the even share is left (200 tokens of up to 6000 positions, 40 heads of
// 128 on 8: 92 us, fitted 107).
template <class F>
__device__ __forceinline__ int fitting(const Rows &s, int groups, int slots, int fewest, F blocks) {
    const int lane = threadIdx.x & 63;
    float n = 0.f, u = 0.f;                      // of this lane's sequence
    if (lane < s.n_seq) blocks(lane, n, u);
    float sum = n * u;
#pragma unroll 4
    for (int b = lane + 64; b < s.n_seq; b += 64) {
        float nb, ub;
        blocks(b, nb, ub);
        sum += nb * ub;
    }
    const float room = (float)slots / (float)groups;
    float least = fmaxf((float)fewest, ceilf(gd_wave_sum(sum) / room));
    // (At least an even share: so no more than units + slots / groups splits.)
    if (s.n_seq <= 64)
        for (int i = 0; i < 12; i++) {
            if (gd_wave_sum(u * (n <= 0.5f * least ? fminf(n + 2.f, least) / least : ceilf(n / least))) <= room) break;
            least = ceilf(least * 1.125f);
        }
    return (int)least;
}
__device__ __forceinline__ int token_least(const Rows &s, const Mask &mask, int groups, int slots, int fewest) {
    return fitting(s, groups, slots, fewest, [&](int b, float &n, float &u) {
        const int pos = s.pos[b];
        n = pos < 0 ? 0.f : (float)token_blocks(s, mask, pos).n;
        u = pos < 0 ? 0.f : 1.f;
    });
}

// Attention of single tokens: workgroup (row, kv head and eight of its query heads;
// split sp of ns) reads the split's keys once for its heads.  Wave w takes the blocks
// of 32 keys sp + ns (w + TW i): S = K Q^T with K straight from the cache as the A
// operand, and O^T += V^T P^T with V staged in the wave's own LDS rows and read by the
// transposing LDS read (no barrier in the loop).  The 16 columns of an MFMA are the
// heads' q as f16 hi (0..7) and lo (8..15), and P likewise: both halves of a product
// come from one instruction and are added across lanes lr, lr ^ 8.  q is brought to
// 2^14 .. 2^15 by a power of two and weights to 2^8, so that hardly a low half leaves f16's
// normal range; scores are in units of log2.  8-bit keys enter as whole numbers, their
// steps scaling the scores; 8-bit values as the halves they are.  Keys that are not
// seen have the weight 0 and zeros for values.  A block's rows are requested one
// block ahead, its page-table entries two.
//   Memory bounds long rows: 64 tokens of 4096 positions, 40 heads of 128 on 8, 101 us in
// codes (5.3 TB/s), 192 in halves (5.6).  Short ones are a chain of loads (position, page,
// keys: 2.5 us) and the merge of the waves (1.7): one token of 331 positions 8.7 us.  64 of
// up to 8192 (125 MB) take 29: long rows' splits beside many of a few keys.
//   Two waves a SIMD or more, where halves of head dim 256 (32 KiB of them in flight a wave)
// take 380 registers and one: us of two with spills / one, 24 heads on 4: one token of 600
// positions 16.8 / 15.9, 64 of up to 8192 88 / 81, eight 27 / 33.  Codes of 128 at two / three,
// 64 tokens of up to 8192, 40 heads on 8: 41 / 46; codes of 256, up to 4096, 37 / 51.
constexpr int TW = 4;                            // waves
constexpr float LAZY = 7.f;                      // how far (log2) weights may pass the maximum they stand at
                                                 // (0, as ever: 1 to 6% more time)
constexpr int MAX_SPLITS = 64;                   // what the combine weighs in one wave
constexpr float LOG2E = 1.4426950408889634f;

template <int HD, bool I8, bool TILED, typename T>
__global__ __launch_bounds__(64 * TW) __attribute__((amdgpu_waves_per_eu(I8 || HD == 128 ? 2 : 1))) void k_attn_tokens(
        Cache c, Rows s, const T *q, int64_t q_stride, const T *gate, int64_t gate_stride, T *out, Part part, int most,
        int slots, int H, float scale, Mask mask) {
    constexpr int KS = HD / 32, DT = HD / 16, VP = HD + 16;
    constexpr int KL = I8 ? KS / 2 : KS;         // 16-byte loads of a key tile, per lane
    constexpr int CPK = I8 ? HD / 16 : HD / 8;   // 16-byte chunks of a value row
    constexpr int VCH = 32 * CPK / 64;           // of a block's values, per lane
    constexpr int EL = I8 ? 16 : 8;              // elements of 16 bytes
    __shared__ __attribute__((aligned(16))) f16 Vs[TW][32][VP];
    __shared__ f16x8 Qs[KS][64];
    __shared__ float wm[TW][8], wl[TW][8];
    static_assert(sizeof(Vs) >= (size_t)TW * 8 * HD * 4, "the merge reuses Vs");
    const int G = H / c.HKV, groups = c.HKV * ((G + 7) / 8);
    const int gr = blockIdx.x % groups;
    const int kvh = gr / ((G + 7) / 8), g8 = 8 * (gr % ((G + 7) / 8)), h0 = kvh * G + g8, nh = min(8, G - g8);
    int n = blockIdx.x / groups, sp = 0, ns = 1, pos;
    if (most > 1) {
        // The rows' splits one after the other, long rows' first, so that the workgroups that
        // have none come last.  (us in any order / border at 0.25 / 0.5 / 0.75: 64 of up to 8192,
        // codes, 40 heads of 128 on 8, 41 / 37 / 37 / 39, halves 62 / 56 / 57 / 56, 24 of 256 on 4
        // 71 / 64 / 64 / 73; 32 of up to 3000, halves, 19.7 / 19.9 / 18.6 / 18.5.)
        const int least = token_least(s, mask, groups, slots, token_fewest(HD));
        auto splits = [&](const Seq &q) { return q.r1 > q.r0 ? token_blocks(s, mask, q.pos).splits(most, least) : 0; };
        Seq sq;
        auto order = [&](const Seq &q) { return q.r1 > q.r0 && token_blocks(s, mask, q.pos).n > 0.5f * least ? 0 : 1; };
        if (!unit_at<2>(s, n, splits, order, n, sp, sq)) return;
        pos = sq.pos;
        ns = token_blocks(s, mask, pos).splits(most, least);
    } else {
        pos = s.pos[n];
        if (pos < 0) return;
    }
    const KeyBlocks<32> kb = token_blocks(s, mask, pos);
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int lr = lane & 15, g = lane >> 4, col = lr & 7;
    // Key lane % 32 of block j: its page-table entry (a load, used a block later), then its
    // row in the planes (any, where there is none) and whether it is seen.
    struct Entry {
        uint32_t kp;
        int page;
    };
    struct Key {
        uint32_t row;
        bool seen;
    };
    const int32_t *table = s.table + (int64_t)n * s.max_pages;
    auto entry_of = [&](int j) {
        const uint32_t kp = kb.start(min(j, kb.n - 1)) + (lane & 31);
        return Entry{kp, table[c.by_page(min(kp, s.cap - 1))]};
    };
    auto key_of = [&](const Entry &e) {
        const bool there = (uint32_t)e.page < c.n_pages && e.kp < s.cap;
        return Key{there ? row_at<I8>(c, e.page, slot_of(c, e.kp), kvh) : (uint32_t)(I8 ? 0 : kvh),
                   there && e.kp <= (uint32_t)pos && (e.kp >= kb.lo || e.kp < kb.sinks)};
    };
    // Bytes from a row to the next position's, and this lane's place in the 16 keys of a
    // tile (keys) and in those of a load of values: with pages of whole tiles a tile has one
    // page and one step, so that its loads take a uniform base.
    constexpr int ES = I8 ? 1 : 2, KPV = 64 / CPK;
    const uint32_t pitch = HD * ES * (I8 ? 1 : c.HKV);
    const uint32_t kplace = lr * pitch + 16 * g, vplace = lane / CPK * pitch + 16 * (lane % CPK);
    u32x4 kreg[2][KL], vreg[VCH];
    uint8_t kx = 0, vx = 0;
    auto fetch = [&](const Key &k) {
        if constexpr (I8) {
            kx = c.kx[k.row / BLK];
            vx = c.vx[k.row / BLK];
        }
        if constexpr (TILED) {
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const uint64_t row = (uint32_t)__builtin_amdgcn_readlane((int)k.row, 16 * kt);
                const char *kp = (const char *)c.k + row * (HD * ES), *vp = (const char *)c.v + row * (HD * ES);
#pragma unroll
                for (int i = 0; i < KL; i++) kreg[kt][i] = *(const u32x4 *)(kp + kplace + 64 * i);
#pragma unroll
                for (int i = kt * VCH / 2; i < (kt + 1) * VCH / 2; i++)
                    vreg[i] = *(const u32x4 *)(vp + (uint64_t)(i * KPV % 16 * pitch) + vplace);
            }
        } else {
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const uint64_t row = (uint32_t)__shfl((int)k.row, 16 * kt + lr, 64);
#pragma unroll
                for (int i = 0; i < KL; i++) kreg[kt][i] = *(const u32x4 *)((const char *)c.k + row * (HD * ES) + 64 * i + 16 * g);
            }
#pragma unroll
            for (int i = 0; i < VCH; i++) {
                const uint64_t row = (uint32_t)__shfl((int)k.row, i * KPV + lane / CPK, 64);
                vreg[i] = *(const u32x4 *)((const char *)c.v + row * (HD * ES) + 16 * (lane % CPK));
            }
        }
    };
    const int step = ns * TW;
    int j = sp + ns * w;
    Entry en = entry_of(j);
    Key kc = key_of(en);
    en = entry_of(j + step);
    if (kb.n) fetch(kc);
    // The gates of this thread's results, for the end (partials are gated by the merge).
    float gates[8 * HD / (64 * TW)];
#pragma unroll
    for (int x = 0; x < 8 * HD / (64 * TW); x++) {
        const int e = t + 64 * TW * x;
        gates[x] = gate && ns == 1 && e < nh * HD ? to_f32(gate[n * gate_stride + (int64_t)h0 * HD + e]) : 0.f;
    }
    // q's operand, a share of its dims a wave.
    float sf;                                    // score factor of this lane's head
    {
        constexpr int KW = KS / TW;
        const T *qrow = q + n * q_stride + (int64_t)(h0 + min(col, nh - 1)) * HD;
        // Dim of element e of k step ks: as the cache's 16-byte loads give them.
        auto dim = [&](int ks) { return I8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g; };
        f32x4 qv[KW][2];
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < KW; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const T *x = qrow + dim(w * KW + i) + 4 * e;
                if constexpr (sizeof(T) == 4) qv[i][e] = *(const f32x4 *)x;
                else qv[i][e] = __builtin_convertvector(*(const f16x4 *)x, f32x4);
#pragma unroll
                for (int k = 0; k < 4; k++) mx = fmaxf(mx, fabsf(qv[i][e][k]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (lane < 8) wm[w][lane] = mx;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TW; i++) mx = fmaxf(mx, wm[i][col]);
        const int ex = min(max((int)(__float_as_uint(mx) >> 23), 40), 254) - 127;
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        sf = scale * LOG2E * __uint_as_float((uint32_t)(127 - 14 + ex) << 23);
        if (fabsf(sf) < 0x1p-126f) sf = 0x1p-126f;         // weights of 1 alike; times inf not NaN
#pragma unroll
        for (int i = 0; i < KW; i++) {
            f16x8 qf;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f16 hi, lo;
                gd_split_f16(col < nh ? qv[i][e >> 2][e & 3] * up : 0.f, hi, lo);
                qf[e] = lr < 8 ? hi : lo;
            }
            Qs[w * KW + i][lane] = qf;
        }
    }
    const float none = sf < 0.f ? INFINITY : -INFINITY;    // the score of no key
    f32x4 acc[DT];                               // O^T rows 16 dt + 4 g + v
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;                // l: this lane's keys only
    __syncthreads();
    for (; j < kb.n; j += step) {
        // Four chains a key tile: shorter sums round less (and wait less).
        f32x4 st[2][4];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const f16x8 qf = Qs[ks][lane];
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                f16x8 kf;
                if constexpr (I8) kf = halves(kreg[kt][ks / 2][2 * (ks % 2)], kreg[kt][ks / 2][2 * (ks % 2) + 1]);
                else kf = __builtin_bit_cast(f16x8, kreg[kt][ks]);
                st[kt][ks & 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        kf, qf, ks < 4 ? f32x4{0.f, 0.f, 0.f, 0.f} : st[kt][ks & 3], 0, 0, 0);
            }
        }
        const uint32_t seen = (uint32_t)__ballot(kc.seen);
        float kstep[2];
        f16 vstep[2];
#pragma unroll
        for (int kt = 0; kt < (I8 ? 2 : 0); kt++) {
            kstep[kt] = step_of((uint8_t)__builtin_amdgcn_readlane(kx, 16 * kt));
            vstep[kt] = (f16)step_of((uint8_t)__builtin_amdgcn_readlane(vx, 16 * kt));
        }
        f32x4 sc[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++) sc[kt] = (st[kt][0] + st[kt][1]) + (st[kt][2] + st[kt][3]);
        // Values to LDS, then the next block's loads.
#pragma unroll
        for (int i = 0; i < VCH; i++) {
            const int k = i * KPV + lane / CPK;
            f16 *row = &Vs[w][k][EL * (lane % CPK)];
            f16x8 v[I8 ? 2 : 1];
            if constexpr (I8) {
                v[0] = halves(vreg[i][0], vreg[i][1]) * vstep[2 * i / VCH];
                v[1] = halves(vreg[i][2], vreg[i][3]) * vstep[2 * i / VCH];
            } else {
                v[0] = __builtin_bit_cast(f16x8, vreg[i]);
            }
            if (seen != 0xffffffffu) {
                asm volatile("");                // a branch, not selects in every block
#pragma unroll
                for (int x = 0; x < (I8 ? 2 : 1); x++) v[x] = seen >> k & 1 ? v[x] : f16x8{};
            }
#pragma unroll
            for (int x = 0; x < (I8 ? 2 : 1); x++) *(f16x8 *)(row + 8 * x) = v[x];
        }
        kc = key_of(en);
        en = entry_of(j + 2 * step);
        fetch(kc);
        __builtin_amdgcn_sched_barrier(0);
        if (!seen) continue;
        // hi + lo of a head's score; keys 16 kt + 4 g + v of the block.  (Unscaled:
        // a weight's exponent is rounded once.)
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                sc[kt][v] += gd_dpp<GD_DPP_ROR8>(sc[kt][v]);
                if constexpr (I8) sc[kt][v] *= kstep[kt];
            }
        if (seen != 0xffffffffu) {
            asm volatile("");
            const uint32_t mine = seen >> (4 * g);
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int v = 0; v < 4; v++) sc[kt][v] = mine & (1u << (16 * kt + v)) ? sc[kt][v] : none;
        }
        float top = -INFINITY;                   // of this lane's keys
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) top = fmaxf(top, sc[kt][v] * sf);
        // The sums are brought to a new maximum, of all a column's lanes, only where one is
        // over 2^LAZY of the one they stand at.
        if (__any(top > m + LAZY)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) acc[dt] *= alpha;
            m = mn;
        }
        f16x8 pf;                                // weights times 2^8, under 2^15, and so l and the sums
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                float p = __builtin_amdgcn_exp2f(fmaf(sc[kt][v], sf, -m)) * 256.f;
                asm("" : "+v"(p));
                l += p;
                const f16 hi = (f16)p;
                pf[4 * kt + v] = lr < 8 ? hi : (f16)(p - (float)hi);
            }
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const f16 *vr = &Vs[w][4 * g + (lr >> 2)][16 * dt + 4 * (lr & 3)];
            const f16x4 v0 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)vr));
            const f16x4 v1 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vr + 16 * VP)));
            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    f16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]}, pf, acc[dt], 0, 0, 0);
        }
    }
    // Merge the waves: each brings its sums to the common maximum.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < 8) wm[w][lane] = m;
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < TW; i++) M = fmaxf(M, wm[i][col]);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    float *red = (float *)Vs;                    // [TW][8][HD]
    if (lane < 8) wl[w][lane] = l * f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
#pragma unroll
        for (int v = 0; v < 4; v++) acc[dt][v] += gd_dpp<GD_DPP_ROR8>(acc[dt][v]);
        if (lr < 8) *(f32x4 *)&red[(w * 8 + lr) * HD + 16 * dt + 4 * g] = acc[dt] * f;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8 * HD / (64 * TW); x++) {
        const int e = t + 64 * TW * x, hh = e / HD, d = e % HD;
        if (e >= nh * HD) break;
        float A = 0.f, L = 0.f;
#pragma unroll
        for (int i = 0; i < TW; i++) {
            A += red[(i * 8 + hh) * HD + d];
            L += wl[i][hh];
        }
        const int64_t row = (int64_t)n * H + h0 + hh;
        if (ns == 1) {
            float y = L == 0.f ? 0.f : A / L;
            if (gate) y *= gd_sigmoid(gates[x]);
            out[row * HD + d] = from_f32<T>(y);
            if (most > 1 && d == 0) part.used[row] = 1;
        } else {
            part.acc[(row * most + sp) * HD + d] = A;
            if (d == 0) {
                if (sp == 0) part.used[row] = ns;
                float M = wm[0][hh];
#pragma unroll
                for (int i = 1; i < TW; i++) M = fmaxf(M, wm[i][hh]);
                part.ml[row * most + sp] = make_float2(M, L);
            }
        }
    }
}

// Attention of prompt chunks (rows of any length): a unit is PC columns of a sequence
// and kv head, a column being one (row, query head) of the kv head's G heads, row by
// row, so that a tile of keys read once serves all of them; wave w owns columns 32 w ..
// Keys stream through LDS as halves in tiles of AK, requested a tile ahead; per tile a
// wave forms S^T = K Q^T (v_mfma_f32_32x32x16_f16: lane = a column and 16 of each 32 keys),
// its columns' online softmax, and O^T += V^T P^T, the C layout of S^T being the B operand
// of P^T once the MFMA's K index 8 h + e (h = lane / 32) stands for key 4 h + e (e < 4) or
// 8 + 4 h + e - 4 of its 16; V^T is read by the transposing LDS read.  f32 rows enter as
// f16 hi + lo pairs (q brought to 2^14 .. 2^15 by a power of two a column, weights to
// 2^8), f16 rows as they are, with weights rounded to f16 and summed as rounded: 2^-11 of a
// weight at most, as the result's own rounding, and less of a sum of many (errors against 64 bits
// 2.6e-4 of the result's norm, with weights as pairs 2.1e-4, the result's rounding alone; in us
// without / with pairs: the first two below 73 / 87 and 134 / 157, 1024 rows after 3000 of codes
// 144 / 163 and of heads of 256 221 / 243).  k_attn_tokens, which memory bounds, takes them as
// pairs.  The gate of f16 rows is a hardware reciprocal of 1 + 2^x: two roundings of 32 bits.  A
// tile that some column does not see whole goes key by key: a mask, and where V holds a NaN or
// infinity its finite part and, apart, which columns see the others (0 x NaN would reach them all).
//   512 f16 rows behind 3584 positions of codes, 40 heads of 128 on 8: 67 us, 600 TFLOP/s;
// 4096 under a window of 1024 133 us, 570; f32 rows (twice the products) of 24 heads of 256
// on 4 530.  No unit of the CU is full (matrix cores 31% busy, vector ALUs 50%, LDS 31%):
// with the registers of two waves a SIMD a wave's chain of staging, scores, weights and sums
// is what lasts, 2.0 to 2.5 us for two waves' tiles, a lone one 1.7.  (f32 rows of 128 take all
// 256 registers, and 4 of them memory on codes, 2 on halves of odd pages.)  Measured and left out:
// units of twice the columns, eight waves to a tile (codes of 256 219 -> 207 us, but f32 rows
// of chunks 115 -> 122, under a window 133 -> 145); scores formed a tile ahead, beside the
// weights of the last (143 -> 154, of 256 219 -> 261); tiles of 32 keys and three waves a
// SIMD (1024 rows 143 -> 127, 512 75 -> 84).
// Columns of a wave, and of a unit: a wave's sums are head dim x columns, which at head
// dim 256 leave 32 columns no registers (128 of sums, 128 of f32 rows' q).
template <int HD> constexpr int wave_cols() { return HD == 128 ? 32 : 16; }
template <int HD> constexpr int unit_cols() { return 4 * wave_cols<HD>(); }
template <int HD> constexpr int tile_keys() { return HD == 128 ? 64 : 32; }

// A sequence's units: first and last row of unit k, and its blocks of keys.
template <int PC, int AK> struct Units {
    int rows, G;
    uint32_t pos, cap;
    __device__ __forceinline__ Units(const Seq &q, int G_, uint32_t cap_) : rows(q.r1 - q.r0), G(G_), pos(q.pos), cap(cap_) {}
    __device__ __forceinline__ int n() const { return (int)(((int64_t)rows * G + PC - 1) / PC); }
    __device__ __forceinline__ int first(int k) const { return k * PC / G; }
    __device__ __forceinline__ int last(int k) const { return min((k * PC + PC - 1) / G, rows - 1); }
    __device__ __forceinline__ KeyBlocks<AK> blocks(const Mask &mask, int k) const {
        return KeyBlocks<AK>(mask, pos + first(k), min(pos + last(k), cap - 1));
    }
    // Splits of each of the units: as the longest, the last, needs them.
    __device__ __forceinline__ int splits(const Mask &mask, int most, int least) const {
        const int longest = blocks(mask, n() - 1).n;
        return longest <= 1.4f * least ? 1 : min(most, (longest + least - 1) / least);
    }
};
// A unit's n blocks in nz splits or fewer: `per` each, `used` splits.
struct Cut {
    int per, used;
    __device__ __forceinline__ Cut(int n, int nz) : per(max(1, (n + nz - 1) / nz)), used(max(1, (n + per - 1) / per)) {}
};
// How finely the keys are split, as token_least, each of a sequence's units taken for its
// longest.
template <int PC, int AK>
__device__ __forceinline__ int unit_least(const Rows &s, const Mask &mask, int G, int HKV, int slots) {
    return fitting(s, HKV, slots, ROWS_FEWEST, [&](int b, float &n, float &u) {
        const Units<PC, AK> q(seq_at(s, b), G, s.cap);
        u = q.rows > 0 ? (float)q.n() : 0.f;
        n = q.rows > 0 ? (float)q.blocks(mask, q.n() - 1).n : 0.f;
    });
}

template <int HD, bool I8, bool TILED, typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void k_attn_rows(Cache c, Rows s, const T *q, int64_t q_stride, const T *gate, int64_t gate_stride, T *out, Part part,
                 int most, int slots, int H, float scale, Mask mask) {
    constexpr bool HL = sizeof(T) == 4;          // hi + lo
    // A wave keeps its priority over the other of its SIMD through the softmax and the sums
    // too where codes are made halves or rows are pairs, in us with / without it (1024 rows
    // behind 3000, 40 heads of 128 on 8; 24 of 256 on 4): f16 rows on codes 144 / 150 and
    // 221 / 228, f32 rows on codes 194 / 208 and 261 / 261, f32 rows on halves 188 / 194 and
    // 214 / 229; f16 rows on halves 130 / 131 and 189 / 184, under a window of 1024 145 / 133.
    constexpr bool HOLD = I8 || HL;
    constexpr int PC = unit_cols<HD>(), MF = wave_cols<HD>(), NV = MF * MF / 64;   // C values of a lane
    using Acc = std::conditional_t<MF == 32, f32x16, f32x4>;
    // Keys of a tile in key groups of MF; k steps of a score; dims in groups of MF.
    constexpr int AK = tile_keys<HD>(), NT = AK / MF, KS = MF == 32 ? HD / 16 : HD / 32, DT = HD / MF;
    constexpr int ES = I8 ? 1 : 2, CPR = HD * ES / 16;   // 16-byte chunks of a row
    constexpr int CH = AK * CPR / 256, KPP = 256 / CPR;  // chunks a thread stages of K (and of V); keys of a pass
    // V rows padded so that a transposing read's 32 lanes (MF 32: four rows of 32 dims, else
    // eight of 16) lie in 64 different banks.
    constexpr int KP = HD + 8, VP = HD + (MF == 32 ? 32 : 16), FD = 4;
    __shared__ __attribute__((aligned(16))) f16 Ks[2][AK][KP];
    __shared__ __attribute__((aligned(16))) f16 Vs[2][AK][VP];
    __shared__ uint8_t odd[2][AK][HD / 8];       // which values of V are no numbers, a bit each
    __shared__ int any_odd[2];
    const int G = H / c.HKV, kvh = blockIdx.x % c.HKV;
    int b, k, nz = 1;
    // The sequences' units one after the other, each in its splits, so that the workgroups
    // that have none come last; the long sequences first, and of each the units that see the
    // most keys.  Borders of the three classes in blocks of a split, us of one class / 0.7 and
    // 0.3 / 0.5 and 0.2 / 0.35 and 0.1: chunks of up to 200 f16 rows, codes of 24 heads of 256
    // on 4, 16 behind 1500 65 / 57 / 54 / 54, behind 2500 64 / 61 / 70 / 62, behind 5000 91 / 82 /
    // 82 / 82; 32 of them 81 / 76 / 78 / 79, 109 / 95 / 94 / 95, 145 / 124 / 124 / 124; 20 of f32
    // rows behind 5000 115 / 119 / 118 / 115, 32 on halves 156 / 136 / 128 / 126.
    const int least = most > 1 ? unit_least<PC, AK>(s, mask, G, c.HKV, slots) : 0;
    auto units = [&](const Seq &q) {
        const Units<PC, AK> u(q, G, s.cap);
        return u.rows <= 0 ? 0 : u.n() * (most > 1 ? u.splits(mask, most, least) : 1);
    };
    Seq sq;
    auto order = [&](const Seq &q) {
        const Units<PC, AK> u(q, G, s.cap);
        const int n = u.rows > 0 ? u.blocks(mask, u.n() - 1).n : 0;
        return n > 0.35f * least ? 0 : n > 0.1f * least ? 1 : 2;
    };
    if (!unit_at<3>(s, blockIdx.x / c.HKV, units, order, b, k, sq)) return;
    const Units<PC, AK> un(sq, G, s.cap);
    const int rows = un.rows;
    if (most > 1) nz = un.splits(mask, most, least);
    const int z = k % nz;
    k = un.n() - 1 - k / nz;
    const struct { int i0, i1; } tl = {un.first(k), un.last(k)};
    const uint32_t p0 = (uint32_t)sq.pos, cap1 = s.cap - 1;
    const KeyBlocks<AK> kb = un.blocks(mask, k);
    const Cut cut(kb.n, nz);
    if (z >= cut.used) return;
    nz = cut.used;
    const int per = cut.per, jend = min(kb.n, (z + 1) * per);
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int lc = lane % MF, h = lane / MF;
    // This lane's column, and the positions that the wave's columns stand at.
    const int col = k * PC + MF * w + lc, i = min(col / G, rows - 1);
    const bool valid = col < rows * G;
    const int head = kvh * G + (valid ? col % G : G - 1);
    const int64_t n = sq.r0 + i;
    const uint32_t p = p0 + i;
    const bool busy = k * PC + MF * w < rows * G;
    const uint32_t plo = p0 + min((k * PC + MF * w) / G, rows - 1);
    const uint32_t seen_from = mask.window && plo >= (uint32_t)mask.window ? plo - mask.window + 1 : 0;
    const uint32_t phi = p0 + min((k * PC + MF * w + MF - 1) / G, rows - 1);
    // Staging: key lane % AK's page-table entry a tile ahead of its row, that a tile ahead
    // of the halves in LDS, those a tile ahead of use.
    const int32_t *table = s.table + (int64_t)b * s.max_pages;
    struct Entry {
        uint32_t kp;
        int page;
    };
    auto entry_of = [&](int j) {
        const uint32_t kp = kb.start(min(j, kb.n - 1)) + (lane & (AK - 1));
        return Entry{kp, table[c.by_page(min(kp, cap1))]};
    };
    const uint32_t pitch = HD * ES * (I8 ? 1 : c.HKV);   // bytes from a row to the next position's
    u32x4 kr[CH], vr[CH];
    int kx = 0, vx = 0;
    uint64_t here = 0;                           // keys of the tile whose pages are there
    auto fetch = [&](const Entry &e) {
        const bool there = (uint32_t)e.page < c.n_pages && e.kp < s.cap && e.kp <= p0 + tl.i1;
        const uint32_t row = there ? row_at<I8>(c, e.page, slot_of(c, e.kp), kvh) : (uint32_t)(I8 ? 0 : kvh);
        here = __ballot(there);
        if constexpr (I8) {
            kx = c.kx[row / BLK];
            vx = c.vx[row / BLK];
        }
#pragma unroll
        for (int x = 0; x < CH; x++) {
            uint64_t at;
            if constexpr (TILED) {               // 16 keys of a page: those of this wave's pass start at a uniform row
                const int tile = (x * KPP + w * (64 / CPR)) & ~15;
                const uint64_t first = (uint32_t)__builtin_amdgcn_readlane((int)row, tile);
                const bool in = here >> tile & 1;                // (row 0, and that one alone, where there is none)
                at = first * (HD * ES) + (in ? (uint32_t)((x * KPP + t / CPR) & 15) * pitch : 0u);
            } else {
                at = (uint64_t)(uint32_t)__shfl((int)row, x * KPP + t / CPR, 64) * (HD * ES);
            }
            kr[x] = *(const u32x4 *)((const char *)c.k + at + 16 * (t % CPR));
            vr[x] = *(const u32x4 *)((const char *)c.v + at + 16 * (t % CPR));
        }
    };
    constexpr uint64_t ALL = AK == 64 ? ~0ull : 0xffffffffull;
    // The fetched tile (block j) to LDS.  Where some column does not see all of it, what is
    // no number in V goes into bits beside it, and a zero in its place.
    bool whole = true;                           // every column sees all of the tile staged last
    auto stage = [&](int j) {
        const uint32_t k0 = kb.start(j);
        const uint64_t in = here & ALL;
        whole = in == ALL && k0 + AK - 1 <= p0 + tl.i0 &&
                (!mask.window || k0 + mask.window > p0 + tl.i1 || k0 + AK <= (uint32_t)mask.sinks);
        const int s2 = j & 1;
        if (t == 0) any_odd[s2] = 0;             // (set, if at all, after the barrier below)
        bool some = false;
#pragma unroll
        for (int x = 0; x < CH; x++) {
            const int key = x * KPP + t / CPR, d = t % CPR * (16 / ES);
            f16x8 kv[I8 ? 2 : 1], vv[I8 ? 2 : 1];
            if constexpr (I8) {
                const int tile = (x * KPP + w * (64 / CPR)) & ~15;
                const f16 ka = (f16)step_of((uint8_t)__builtin_amdgcn_readlane(kx, tile));
                const f16 va = (f16)step_of((uint8_t)__builtin_amdgcn_readlane(vx, tile));
                kv[0] = halves(kr[x][0], kr[x][1]) * ka;
                kv[1] = halves(kr[x][2], kr[x][3]) * ka;
                vv[0] = halves(vr[x][0], vr[x][1]) * va;
                vv[1] = halves(vr[x][2], vr[x][3]) * va;
            } else {
                kv[0] = __builtin_bit_cast(f16x8, kr[x]);
                vv[0] = __builtin_bit_cast(f16x8, vr[x]);
            }
            if (!whole) {
#pragma unroll
                for (int y = 0; y < (I8 ? 2 : 1); y++) {
                    u32x4 v = __builtin_bit_cast(u32x4, vv[y]);
                    if (!(in >> key & 1)) v = u32x4{0u, 0u, 0u, 0u};
                    uint32_t no = 0;             // a half's top bit: all exponent bits set
#pragma unroll
                    for (int e = 0; e < 4; e++) no |= (v[e] & 0x7c007c00u) + 0x04000400u;
                    uint32_t bits = 0;
                    if (no & 0x80008000u) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t x = (v[e] & 0x7c007c00u) + 0x04000400u;
                            bits |= (x >> 15 & 1u) << 2 * e | (x >> 31) << (2 * e + 1);
                            v[e] &= ((x >> 15 & 1u) ? 0u : 0xffffu) | (x >> 31 ? 0u : 0xffff0000u);
                        }
                        some = true;
                    }
                    odd[s2][key][d / 8 + y] = (uint8_t)bits;
                    vv[y] = __builtin_bit_cast(f16x8, v);
                }
            }
#pragma unroll
            for (int y = 0; y < (I8 ? 2 : 1); y++) {
                *(f16x8 *)&Ks[s2][key][d + 8 * y] = kv[y];
                *(f16x8 *)&Vs[s2][key][d + 8 * y] = vv[y];
            }
        }
        return some;
    };
    auto mfma = [](f16x8 a, f16x8 b, Acc c) {
        if constexpr (MF == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    };
    int j = z * per;
    Entry en = entry_of(j);
    // B operand of S^T: dims 8 (64 / MF) ks + 8 h + e of the lane's column; the sign of the scale
    // goes into it, so that the greatest product is the greatest score.
    f16x8 qh[KS], ql[HL ? KS : 1];
    float sf = fabsf(scale) * LOG2E;
    {
        const T *qrow = q + n * q_stride + (int64_t)head * HD + 8 * h;
        const bool neg = scale < 0.f;
        if constexpr (HL) {
            f32x4 x[KS][2];
            float mx = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    x[ks][y] = *(const f32x4 *)(qrow + 512 / MF * ks + 4 * y);
                }
            if (j < jend) fetch(en);             // (while the rows are on their way)
            en = entry_of(j + 1);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(x[ks][y][e]));
            if constexpr (MF == 16) mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const int ex = min(max((int)(__float_as_uint(mx) >> 23), 40), 254) - 127;
            const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23) * (neg ? -1.f : 1.f);
            sf *= __uint_as_float((uint32_t)(127 - 14 + ex) << 23);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    f16 hi, lo;
                    gd_split_f16(x[ks][e >> 2][e & 3] * up, hi, lo);
                    qh[ks][e] = hi;
                    ql[ks][e] = lo;
                }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) qh[ks] = *(const f16x8 *)(qrow + 512 / MF * ks);
            if (j < jend) fetch(en);
            en = entry_of(j + 1);
            if (neg)
#pragma unroll
                for (int ks = 0; ks < KS; ks++) qh[ks] = -qh[ks];
        }
    }
    if (sf < 0x1p-126f) sf = 0x1p-126f;          // weights of 1 alike; times -inf not NaN
    // Row 8 (v / 4) + 4 h + v % 4 of a C value v (MF 16: 4 h + v).
    Acc acc[DT];                                 // O^T, dims MF dt + row
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = Acc{};
    float m = -INFINITY, l = 0.f;                // l: this lane's keys only
    bool some = j < jend && stage(j);
    uint64_t now = here & ALL;
    if (j + 1 < jend) fetch(en);
    en = entry_of(j + 2);
    __syncthreads();
    for (; j < jend; j++) {
        const uint32_t k0 = kb.start(j);
        const int s2 = j & 1;
        if (some) any_odd[s2] = 1;
        const bool all_see = whole;
        // The next tile to the other half of LDS, the one after it requested.
        const uint64_t next = here & ALL;
        if (j + 1 < jend) {
            some = stage(j + 1);
            fetch(en);
            en = entry_of(j + 3);
        }
        __builtin_amdgcn_sched_barrier(0);
        // The wave's own view of the tile.
        if (busy && k0 <= phi && !(seen_from > k0 + AK - 1 && k0 >= (uint32_t)mask.sinks)) {
            const bool full = now == ALL && k0 + AK - 1 <= plo &&
                              (!mask.window || k0 + mask.window > phi || k0 + AK <= (uint32_t)mask.sinks);
            Acc st[NT];                          // S^T, keys MF kt + row
            __builtin_amdgcn_s_setprio(1);       // over the SIMD's other wave, that may be staging
            {
                // A operands FD reads ahead of their products.
                auto keys = [&](int x) { return *(const f16x8 *)&Ks[s2][x % NT * MF + lc][x / NT * (512 / MF) + 8 * h]; };
                f16x8 ka[FD];
#pragma unroll
                for (int x = 0; x < FD; x++) ka[x] = keys(x);
                __builtin_amdgcn_sched_group_barrier(0x100, FD, 0);
#pragma unroll
                for (int x = 0; x < NT * KS; x++) {
                    const int kt = x % NT, ks = x / NT;
                    st[kt] = mfma(ka[x % FD], qh[ks], ks ? st[kt] : Acc{});
                    if constexpr (HL) st[kt] = mfma(ka[x % FD], ql[ks], st[kt]);
                    __builtin_amdgcn_sched_group_barrier(0x008, HL ? 2 : 1, 0);
                    if (x + FD < NT * KS) {
                        ka[x % FD] = keys(x + FD);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    }
                }
            }
            if constexpr (!HOLD) __builtin_amdgcn_s_setprio(0);
            if (!full) {
                // A bit a key, as this column sees it.
                auto below = [](int64_t x) { return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1; };
                uint64_t see = below((int64_t)p - k0 + 1);
                if (mask.window) see &= ~below((int64_t)p - mask.window + 1 - k0) | below((int64_t)mask.sinks - k0);
                see = (see & now) >> (4 * h);
#pragma unroll
                for (int kt = 0; kt < NT; kt++) {
                    const uint32_t bits = (uint32_t)(see >> (MF * kt));
#pragma unroll
                    for (int v = 0; v < NV; v++)
                        st[kt][v] = bits & (1u << (8 * (v / 4) + v % 4)) ? st[kt][v] : -INFINITY;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < NT; kt++)
#pragma unroll
                for (int v = 0; v < NV; v++) top = fmaxf(top, st[kt][v]);
            // Sums are brought to a new maximum only where a score is over 2^LAZY of the one
            // they stand at (random scores: hardly after the first tiles).
            if (__any(top * sf > m + LAZY)) {
                if constexpr (MF == 16) top = fmaxf(top, __shfl_xor(top, 16, 64));
                const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)) * sf);
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
                l *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) acc[dt] *= alpha;
                m = mn;
            }
            // Weights times 2^8, under 2^15 (f16 rows: in the exponent, where 32-bit rows would
            // lose bits).
            const float off = m == -INFINITY ? 0.f : HL ? -m : 8.f - m;
            // P^T as B operands: keys 16 kk on (MF 32) or 32 kk, element e the row of C value e.
            constexpr int KK = AK / (512 / MF);
            f16x8 ph[KK], pl[HL ? KK : 1];
#pragma unroll
            for (int kt = 0; kt < NT; kt++)
#pragma unroll
                for (int v = 0; v < NV; v += 2) {
                    constexpr auto kk = [](int kt, int v) { return (NV * kt + v) / 8; };
                    float w0 = __builtin_amdgcn_exp2f(fmaf(st[kt][v], sf, off));
                    float w1 = __builtin_amdgcn_exp2f(fmaf(st[kt][v + 1], sf, off));
                    f16x2 hi, lo;
                    if constexpr (HL) {
                        w0 *= 256.f;
                        w1 *= 256.f;
                        gd_split2_f16(w0, w1, hi, lo);
                        pl[kk(kt, v)][(NV * kt + v) % 8] = lo[0];
                        pl[kk(kt, v)][(NV * kt + v) % 8 + 1] = lo[1];
                    } else {
                        typedef float f32x2 __attribute__((ext_vector_type(2)));
                        hi = __builtin_convertvector((f32x2{w0, w1}), f16x2);
                    }
                    if constexpr (HL) {
                        l += w0;
                        l += w1;
                    } else {
                        l = __builtin_amdgcn_fdot2(hi, f16x2{(f16)1.f, (f16)1.f}, l, false);
                    }
                    ph[kk(kt, v)][(NV * kt + v) % 8] = hi[0];
                    ph[kk(kt, v)][(NV * kt + v) % 8 + 1] = hi[1];
                }
            {
                typedef short s16x4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                // V^T of keys (512 / MF) (x / DT) on, dims MF (x % DT) + lane % MF.
                auto values = [&](int x) {
                    const f16 *v = &Vs[s2][x / DT * (512 / MF) + 4 * h + (lane >> 2 & 3)][x % DT * MF + (MF == 32 ? 16 * (lane >> 4 & 1) : 0) + 4 * (lane & 3)];
                    const f16x4 v0 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)v));
                    const f16x4 v1 = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(v + 256 / MF * VP)));
                    return f16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                };
                f16x8 va[FD];
#pragma unroll
                for (int x = 0; x < FD; x++) va[x] = values(x);
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * FD, 1);
#pragma unroll
                for (int x = 0; x < KK * DT; x++) {
                    const int kk = x / DT, dt = x % DT;
                    acc[dt] = mfma(va[x % FD], ph[kk], acc[dt]);
                    if constexpr (HL) acc[dt] = mfma(va[x % FD], pl[kk], acc[dt]);
                    __builtin_amdgcn_sched_group_barrier(0x008, HL ? 2 : 1, 1);
                    if (x + FD < KK * DT) {
                        va[x % FD] = values(x + FD);
                        __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
        if (!all_see && any_odd[s2]) {
            // What is no number reaches the columns that see it.
            for (int key = 0; key < AK; key++)
                if (kb.start(j) + key <= p && (now >> key & 1) &&
                    (!mask.window || k0 + key + mask.window > p || k0 + key < (uint32_t)mask.sinks))
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int v = 0; v < NV; v++)
                            if (odd[s2][key][(MF * dt + 8 * (v / 4) + 4 * h) / 8] >> (4 * h % 8 + v % 4) & 1) acc[dt][v] = __uint_as_float(0x7fc00000u);
            __syncthreads();
        }
        now = next;
    }
    if (!valid) return;
    if constexpr (MF == 16) l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int64_t row = n * H + head;
    if (most > 1 && z == 0 && h == 0) part.used[row] = nz;
    if (nz > 1) {
        float *y = part.acc + (row * most + z) * HD + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int v = 0; v < NV; v += 4)
                *(f32x4 *)(y + MF * dt + 2 * v) = f32x4{acc[dt][v], acc[dt][v + 1], acc[dt][v + 2], acc[dt][v + 3]};
        if (h == 0) part.ml[row * most + z] = make_float2(m, l);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int v = 0; v < NV; v += 4) {
            const int d = MF * dt + 2 * v + 4 * h;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = acc[dt][v + e] * inv;
            if (gate) {
                const T *gr = gate + n * gate_stride + (int64_t)head * HD + d;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    y[e] *= HL ? gd_sigmoid(to_f32(gr[e])) : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * to_f32(gr[e])));
            }
            if constexpr (HL)
                *(f32x4 *)(out + row * HD + d) = f32x4{y[0], y[1], y[2], y[3]};
            else
                *(uint64_t *)(out + row * HD + d) = (uint64_t)gd_f2h(y[0]) | ((uint64_t)gd_f2h(y[1]) << 16) |
                                                    ((uint64_t)gd_f2h(y[2]) << 32) | ((uint64_t)gd_f2h(y[3]) << 48);
        }
}

// Whether row n has a sequence (else nobody has written anything for it).
__device__ __forceinline__ bool has_sequence(const Rows &s, int n) {
    const int b = seq_of_row(s, n);
    if (b < 0) return false;
    const Seq sq = seq_at(s, b);
    return n >= sq.r0 && n < sq.r1;
}

template <typename T> __device__ __forceinline__ float gated(float y, const T *gate) {
    return y * gd_sigmoid(to_f32(*gate));
}

// Merges the partials (up to `most` <= MAX_SPLITS) of head h of row n, few rows: thread
// (d, r) takes the splits r, r + NR, .. of one dim, beside the splits' weights, once a
// workgroup.  A chain of loads: 4.6 us for 64 splits of 24 heads of 256.
template <int HD, typename T>
__global__ __launch_bounds__(512) void k_attn_merge(Part part, int most, Rows s, const T *gate, int64_t gate_stride,
                                                    T *out, int H) {
    constexpr int NR = 512 / HD;
    __shared__ float fs[MAX_SPLITS], sum[NR][HD];
    const int n = blockIdx.x / H, h = blockIdx.x % H, t = threadIdx.x, d = t % HD, r = t / HD;
    const int ns = min(part.used[blockIdx.x], most);
    if (!has_sequence(s, n) || ns <= 1) return;
    const float *p = part.acc + (int64_t)blockIdx.x * most * HD;
    float a[MAX_SPLITS / NR];
#pragma unroll
    for (int i = 0; i < MAX_SPLITS / NR; i++) a[i] = r + NR * i < ns ? p[(r + NR * i) * HD + d] : 0.f;
    float inv;
    {
        const int lane = t & 63;                 // every wave: the weight of split lane
        const float2 ml = lane < ns ? part.ml[(int64_t)blockIdx.x * most + lane] : make_float2(-INFINITY, 0.f);
        const float M = wave_max(ml.x);
        const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
        const float L = gd_wave_sum(ml.y * f);
        inv = L == 0.f ? 0.f : 1.0f / L;
        if (t < MAX_SPLITS) fs[t] = f;
    }
    __syncthreads();
    float A = 0.f;
#pragma unroll
    for (int i = 0; i < MAX_SPLITS / NR; i++) A += a[i] * fs[r + NR * i];
    sum[r][d] = A;
    __syncthreads();
    if (r) return;
#pragma unroll
    for (int i = 1; i < NR; i++) A += sum[i][d];
    float y = A * inv;
    if (gate) y = gated(y, gate + n * gate_stride + (int64_t)h * HD + d);
    out[(int64_t)blockIdx.x * HD + d] = from_f32<T>(y);
}

// The same for many rows: HD / 4 threads a (row, head), four dims each, a split at a time.
// Bytes bound it: 20480 rows and heads of 128 in 3 splits, 37 MB, 11 us.
template <int HD, typename T>
__global__ __launch_bounds__(256) void k_attn_merge_many(Part part, int most, Rows s, const T *gate, int64_t gate_stride,
                                                         T *out, int H) {
    constexpr int TPR = HD / 4, RPW = 256 / TPR;
    const int groups = (H + RPW - 1) / RPW, n = blockIdx.x / groups;
    const int h = (int)(blockIdx.x % groups) * RPW + (int)threadIdx.x / TPR, d = 4 * (threadIdx.x % TPR);
    // (has_sequence takes whole waves.  Threads past the last head leave it alone: out may be
    // gate, which is read where out is written.)
    if (!has_sequence(s, n) || h >= H) return;
    const int64_t row = (int64_t)n * H + h;
    const int ns = min(part.used[row], most);
    if (ns <= 1) return;
    const float2 *ml = part.ml + row * most;
    const float *p = part.acc + row * most * HD + d;
    float M = -INFINITY, L = 0.f;
    for (int z = 0; z < ns; z++) M = fmaxf(M, ml[z].x);
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int z = 0; z < ns; z++) {
        const float2 x = ml[z];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - M);
        L += x.y * f;
        A += *(const f32x4 *)(p + (int64_t)z * HD) * f;
    }
    A *= L == 0.f ? 0.f : 1.0f / L;
    if (gate)
#pragma unroll
        for (int e = 0; e < 4; e++) A[e] = gated(A[e], gate + n * gate_stride + (int64_t)h * HD + d + e);
    T *y = out + row * HD + d;
    if constexpr (sizeof(T) == 4)
        *(f32x4 *)y = A;
    else
        *(uint64_t *)y = (uint64_t)gd_f2h(A[0]) | ((uint64_t)gd_f2h(A[1]) << 16) | ((uint64_t)gd_f2h(A[2]) << 32) |
                         ((uint64_t)gd_f2h(A[3]) << 48);
}

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

// A positive number modulo 1 as a fraction of 2^64, from its 64 bits and exponent (floorl and
// a conversion a pair took 3 us of a call's 8.3 at 128 rotated dims).
uint64_t fraction(long double x) {
    int up;
    const uint64_t bits = (uint64_t)(frexpl(x, &up) * 0x1p64L);          // x = bits 2^(up - 64)
    return up > 63 || up < -63 ? 0 : up >= 0 ? bits << up : bits >> -up;
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

extern "C" int gd_kv_attn(gd_ctx *ctx, const gd_kv *kv, const gd_seqs *s, const void *q, int64_t q_stride,
                          const void *gate, int64_t gate_stride, void *out, int x_dtype, int n_head, float scale,
                          int window, int n_sink) {
    const char *fn = "gd_kv_attn";
    int rc;
    if ((rc = check_kv(ctx, fn, kv, true)) || (rc = check_seqs(ctx, fn, s)) || (rc = check_x(ctx, fn, x_dtype))) return rc;
    const int hd = kv->head_dim, size = x_dtype == GD_F32 ? 4 : 2;
    GD_REQUIRE(ctx, q && out, "%s: null q or out", fn);
    GD_REQUIRE(ctx, n_head > 0 && n_head <= 65536 && n_head % kv->n_head_kv == 0,
               "%s: n_head %d not a multiple of n_head_kv %d", fn, n_head, kv->n_head_kv);
    const int64_t row = (int64_t)n_head * hd;
    GD_REQUIRE(ctx, q_stride >= row && (!gate || gate_stride >= row) && q_stride < (1LL << 31) &&
                        (!gate || gate_stride < (1LL << 31)),
               "%s: rows of %d heads at strides %lld, %lld", fn, n_head, (long long)q_stride, (long long)gate_stride);
    GD_REQUIRE(ctx, ((uintptr_t)q | (uintptr_t)out | (uintptr_t)gate) % 16 == 0 && q_stride * size % 16 == 0 &&
                        (!gate || gate_stride * size % 16 == 0),
               "%s: q, gate and out must be 16-byte aligned, and their rows", fn);
    GD_REQUIRE(ctx, window >= 0 && n_sink >= 0, "%s: window %d, n_sink %d", fn, window, n_sink);
    GD_REQUIRE(ctx, std::isfinite(scale), "%s: scale %g", fn, (double)scale);
    GD_REQUIRE(ctx, s->n_rows * n_head < (1LL << 31) - 256, "%s: %lld rows of %d heads", fn, (long long)s->n_rows, n_head);
    const bool tokens = !s->row_start;
    const int G = n_head / kv->n_head_kv, cols = hd == 128 ? unit_cols<128>() : unit_cols<256>();
    const int64_t groups = tokens ? kv->n_head_kv * ((G + 7) / 8) : kv->n_head_kv;
    const int64_t units = tokens ? s->n_rows : s->n_rows * G / cols + std::min<int64_t>(s->n_seq, s->n_rows);
    // (Splits add no more than the chip's slots and two units.)
    GD_REQUIRE(ctx, units * groups < MAX_WGS - (1 << 16), "%s: %lld rows of %d heads", fn, (long long)s->n_rows, n_head);
    // Workgroups read their q and gate before they write: in place only row on row.
    const size_t span = (size_t)s->n_rows * row * size;
    auto apart = [&](const void *x, int64_t stride) {
        const uintptr_t a = (uintptr_t)x, o = (uintptr_t)out, end = a + ((s->n_rows - 1) * stride + row) * size;
        return !x || !span || (a == o && stride == row) || end <= o || o + span <= a;
    };
    GD_REQUIRE(ctx, apart(q, q_stride) && apart(gate, gate_stride),
               "%s: out in place of q or gate needs their place and rows of n_head * head_dim", fn);
    GD_CHECK_CTX(ctx);
    if (!s->n_rows || !s->n_seq) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    const Mask mask{window, window ? n_sink : 0};
    const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
    const Rows rows = rows_of(kv, s);
    int64_t keys = s->max_len ? std::min<int64_t>(s->max_len, rows.cap) : rows.cap;
    const int width = tokens ? 32 : hd == 128 ? tile_keys<128>() : tile_keys<256>();
    if (window)
        keys = std::min(keys, (int64_t)window + (tokens ? 0 : cols / G) + width - 1 + ((int64_t)n_sink + width - 1) / width * width);
    // Blocks of keys of the longest row, workgroups of a split each, those that the chip
    // holds at once, and the most splits.  The keys are left whole, without a merge's
    // launch, where that is a few rounds of blocks a wave or the workgroups are many; how
    // finely others are split, the kernels know (token_least, unit_least).
    const int64_t blocks = (keys + width - 1) / width;
    const int64_t slots = (tokens && hd == 256 && kv->dtype == GD_F16 ? 1 : 2) * cus, wgs = units * groups;    // (k_attn_tokens' registers)
    // Rows' partials cost a full chip some 15 us, and a split saves what lets the workgroups
    // fill it; but the longest row may be one of a few, which split share the chip.  f16 rows on
    // codes, us whole / split, 40 heads of 128 on 8 (24 of 256 on 4): 10 blocks 28 / 31; 12 of 96
    // workgroups, lengths alike 33 / 32 (29 / 30) and mixed 32 / 22 (28 / 20), of 240 34 / 39 (30 / 38)
    // and 33 / 29 (29 / 25); 19 of 240 47 / 46 (41 / 44) and 45 / 25 (39 / 25), of 288 55 / 61 (48 / 54)
    // and 45 / 27 (39 / 24), of 480 58 / 64 (51 / 59) and 46 / 29 (40 / 27); 24 of 384 67 / 73 (58 / 65)
    // and 54 / 30 (47 / 28); 64 of 360 123 / 89, of 620 127 / 90, of 930 183 / 196.  Under a window
    // lengths count alike: 15 blocks of 156 to 208 workgroups, f32 rows on halves, 39 / 38 to 43,
    // codes 36 / 33 to 39, of 224 and more 39 / 44 to 46 and 36 / 40; 13 of 184 35.5 / 35.2, 17 of 216
    // 41 / 38, of 232 41 / 45.
    bool whole;
    if (tokens)
        // f16 tokens on codes, us whole / split, 40 heads of 128 on 8 (24 of 256 on 4): one of 13
        // blocks 10.2 / 12.0 (15.8 / 14.0), of 18 11.5 / 12.0 (17.8 / 14.0), of 25 14.0 / 11.9.
        // Of 34 blocks under a window, lengths alike / up to 16000, by workgroups: 128 17.7 / 18.3
        // and 17.5 / 15.0; 192 18.3 / 22.6 and 17.7 / 16.8; 248 19.0 / 22.7 and 17.9 / 19.4; 256 19.3 /
        // 22.9 and 17.9 / 18.5; f32 rows on halves of 192 23.4 / 30.9 and 16.5 / 18.1 (heads of 256,
        // codes: 192 31.2 / 35.0 and 28.3 / 25.8; 252 35.9 / 38.7 and 28.5 / 31.3; halves of 192 45.7 /
        // 48.8 and 37.8 / 39.2).  Of 38 and 256 workgroups 19.6 / 23.1 and 18.5 / 15.1.
        //   Tokens of up to 6000 positions: 200 of 8 kv heads (3.1 times the slots) 118 / 99, 500 213 /
        // 250, 1500 456 / 653; 500 of 4 (3.9 times) 248 / 244.  Past 1024 blocks a long one of them
        // would be the call's time.
        whole = blocks <= (hd == 128 ? 5 : 4) * TW || (blocks <= 9 * TW && 8 * wgs >= (hd == 128 ? 6 : 7) * cus) ||
                (blocks <= 256 * TW && wgs >= 4 * slots) || wgs >= 16 * slots;
    else
        whole = blocks <= 10 || (blocks <= 24 && blocks * (slots - wgs) <= (window ? 9 : 8) * slots) ||
                (blocks <= 128 && 2 * wgs >= 3 * slots) || wgs >= 4 * slots;
    const int least = tokens ? token_fewest(hd) : ROWS_FEWEST;
    int64_t ns = whole ? 1 : std::min<int64_t>((blocks + least - 1) / least, MAX_SPLITS);
    float *scratch = nullptr;
    if ((rc = split_scratch(ctx, (size_t)s->n_rows * n_head * (hd + 3) * sizeof(float), ns, &scratch))) return rc;
    const int64_t sums = s->n_rows * n_head * ns;
    const Part part{scratch, (float2 *)(scratch + sums * hd), (int *)(scratch + sums * (hd + 2))};
    // Split, the units take no more workgroups than one each and one a slot (fitting), with
    // two to spare for the kernels' roundings.
    const dim3 grid((unsigned)(groups * (ns > 1 ? std::min(units * ns, units + slots / groups + 2) : units)));
#define GD_GO(HD_, I8_, T_) \
    do { \
        const bool tiled = I8_ || kv->page_size % 16 == 0; \
        auto kernel = tokens ? (tiled ? k_attn_tokens<HD_, I8_, true, T_> : k_attn_tokens<HD_, I8_, I8_, T_>) \
                             : (tiled ? k_attn_rows<HD_, I8_, true, T_> : k_attn_rows<HD_, I8_, I8_, T_>); \
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, cache_of(kv), rows, (const T_ *)q, q_stride, \
                           (const T_ *)gate, gate_stride, (T_ *)out, part, (int)ns, (int)slots, n_head, scale, mask); \
        if (ns > 1) { \
            GD_LAUNCHED(ctx, fn); \
            /* (a workgroup a row and head: one token of 24 heads, 64 splits, 24 us, by the other \
               31.8; 2560 rows and heads 114.8 and 75.2) */ \
            const bool many = s->n_rows * n_head >= 1024; \
            const int per = 1024 / HD_, merges = many ? (n_head + per - 1) / per : n_head; \
            auto merge = many ? k_attn_merge_many<HD_, T_> : k_attn_merge<HD_, T_>; \
            hipLaunchKernelGGL(merge, dim3((unsigned)(s->n_rows * merges)), dim3(many ? 256 : 512), 0, ctx->stream, part, \
                               (int)ns, rows, (const T_ *)gate, gate_stride, (T_ *)out, n_head); \
        } \
    } while (0)
    GD_KV_PICK(kv, x_dtype, GD_GO);
#undef GD_GO
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}
