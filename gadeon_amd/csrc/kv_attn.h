// Attention over the paged KV cache of many sequences: the kernels and their launch, for
// plain scores (kv_cache.hip) and for capped, biased and masked ones (kv_scores.hip).
#pragma once

#include "kv_core.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// How scores are made and which keys are seen.  Plain: every key up to the query's own, or
// those of a window and the first `sinks`.
struct Mask {
    int window, sinks;                           // window 0: every key up to the query's own
    static constexpr bool SCORED = false;
    using Tokens = Mask;                         // what k_attn_tokens is compiled for
};
// Beside that (gd_scores): scores capped at `cap` and -slope[h] times the distance added, both
// in units of log2; no key before first[row], and every key before prefix[b].
struct ScoreArgs {
    int window, sinks;
    float cap;                                   // 0: none
    const float *slope;
    const int32_t *first, *prefix;
};
// BY_EXP: there is a cap, and an exponential makes it (cap_score); prompt chunks are compiled for
// that apart (1021 f32 rows after 3003 of 16 heads, capped and biased, 97 us as it was built, 106 with a branch to the
// other ways in the loop; now 92, not capped 82, by the quotient 102).
template <bool BY_EXP_> struct Scores : ScoreArgs {
    static constexpr bool SCORED = true, BY_EXP = BY_EXP_;
    using Tokens = Scores<false>;
    operator Tokens() const { return {*this}; }
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
        lo = min(lo, last + 1);                  // (a window behind the last key there may be: its block may hold sinks)
        sinks = min((uint32_t)m.sinks, lo);
        ns = (int)min((sinks + W - 1) / W, lo / W);
        n = ns + (int)(last / W + 1 - lo / W);
    }
    __device__ __forceinline__ uint32_t start(int j) const { return (uint32_t)(j < ns ? j : j - ns + (int)(lo / W)) * W; }
    // Splits that these blocks are worked in: of `least` blocks or more, `most` at most.
    __device__ __forceinline__ int splits(int most, int least) const { return max(1, min(most, (n + least - 1) / least)); }
};

// The same of scored rows: a document that starts at `doc`, seen whole up to `prefix`.  The
// keys before the window are those before either bound, and `last` may lie behind the query.
template <int W> struct ScoredBlocks {
    uint32_t lo, sinks, doc;
    int ns, n, from;                             // blocks of sinks, in all; the first of them
    __device__ __forceinline__ ScoredBlocks(const ScoreArgs &m, uint32_t first, uint32_t last, uint32_t prefix, uint32_t doc_) : doc(doc_) {
        lo = m.window && first >= (uint32_t)m.window ? first - m.window + 1 : 0;
        lo = min(lo, last + 1);
        sinks = min(max((uint32_t)m.sinks, prefix), lo);
        from = (int)(doc / W);
        const uint32_t start = max(lo, doc);
        ns = sinks > doc ? (int)min((sinks + W - 1) / W, start / W) - from : 0;
        n = ns + (start <= last + 1 ? (int)(last / W + 1 - start / W) : 0);
        far = (int)(start / W) - ns;
    }
    __device__ __forceinline__ uint32_t start(int j) const { return (uint32_t)(j < ns ? j + from : j + far) * W; }
    __device__ __forceinline__ int splits(int most, int least) const { return max(1, min(most, (n + least - 1) / least)); }

private:
    int far;
};

template <int W, class How> using Blocks = std::conditional_t<How::SCORED, ScoredBlocks<W>, KeyBlocks<W>>;
template <int W> __device__ __forceinline__ KeyBlocks<W> blocks_of(const Mask &m, uint32_t first, uint32_t last, uint32_t, uint32_t) {
    return KeyBlocks<W>(m, first, last);
}
template <int W>
__device__ __forceinline__ ScoredBlocks<W> blocks_of(const ScoreArgs &m, uint32_t first, uint32_t last, uint32_t prefix, uint32_t doc) {
    return ScoredBlocks<W>(m, first, last, prefix, doc);
}
// A sequence's prefix and a row's document's first position (0: none).
template <class How> __device__ __forceinline__ uint32_t prefix_of(const How &m, int b) {
    if constexpr (How::SCORED) return m.prefix ? (uint32_t)max(m.prefix[b], 0) : 0;
    else return 0;
}
template <class How> __device__ __forceinline__ uint32_t doc_of(const How &m, int64_t n) {
    if constexpr (How::SCORED) return m.first ? (uint32_t)max(m.first[n], 0) : 0;
    else return 0;
}

// A head's slope in units of log2, bounded where its products with distances stay numbers (next to a
// score its next key weighs nothing long before; a NaN stays one).
constexpr float STEEPEST = 0x1p96f;
__device__ __forceinline__ float slope_of(const ScoreArgs &m, int head) {
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(m.slope[head] * LOG2E, -STEEPEST), STEEPEST);
}

// Scores s capped: cap tanh(x), x = s to_x.  BY_EXP as cap - 2 cap / (1 + e^2x), off by 2^-22 of
// the cap, by 2^-21.3 where the reciprocal is a step off (x so little that e^2x is lost in 1 leaves six
// half steps of 1): for caps that this is little of, up to EXP_CAP (what the scores' sums of
// products lose; of f16 rows, whose weights are rounded to 2^-11, EXP_CAP_F16).  Else as cap x P(x^2) /
// Q(x^2) over |x| <= TANH_END, from where on tanh is 1 to 2^-25: off by 2^-23.8 of itself in exact
// arithmetic, by 2^-21.4 as formed, 2^-21 with the reciprocal a step off (twelve half steps of 32 bits at most,
// 2^-20.4: one each of u, cap x and the last two products, two of each polynomial's last sums, three of the
// reciprocal, one of the coefficients).  Degrees and coefficients by least squares reweighted to the least
// relative error, all of them positive.  In slots of an instruction at full rate 11 and 18 a score.
//   (Measured and left out: where all scores of a wave are under half the cap, the polynomial of
// tanh alone, 6 or 7: 107 us where one way alone takes 97; and what a row sees made its neighbours' last bits.)
constexpr float TANH_END = 9.02f, EXP_CAP = 64.f, EXP_CAP_F16 = 1024.f;
// to_x of scores in units of sf (bounded: a score of 0 times infinity is not 0).
__device__ __forceinline__ float over_cap(float sf, const ScoreArgs &how) { return __builtin_amdgcn_fmed3f(sf / how.cap, -0x1p120f, 0x1p120f); }
template <bool BY_EXP> __device__ __forceinline__ float cap_score(const ScoreArgs &how, float s, float to_x) {
    if constexpr (!BY_EXP) {
        // (These two keep a NaN, which the median of three would make a bound.)
        const float x = __builtin_elementwise_minimum(__builtin_elementwise_maximum(s * to_x, -TANH_END), TANH_END), u = x * x;
        const float p = fmaf(fmaf(fmaf(fmaf(u, 1.33190953e-08f, 2.05835024e-05f), u, 3.49403605e-03f), u, 1.33797193e-01f), u, 9.99999979e-01f);
        const float q = fmaf(fmaf(fmaf(fmaf(u, 7.76203024e-07f, 3.28309512e-04f), u, 2.58710791e-02f), u, 4.67130345e-01f), u, 1.f);
        return how.cap * x * (p * __builtin_amdgcn_rcpf(q));
    } else {
        return fmaf(-2.f * how.cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * (to_x * (2.f * LOG2E)))), how.cap);
    }
}
template <bool BY_EXP, int N, int V, class Vec> __device__ __forceinline__ void cap_scores(const ScoreArgs &how, float to_x, Vec (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int v = 0; v < V; v++) s[i][v] = cap_score<BY_EXP>(how, s[i][v], to_x);
}

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
// 8: 17.3 / 17.3 / 24.1, 16 of 8 sequences 29.2 / 30.7 / 35.0; full chips alike; fewer where a
// document leaves a unit fewer, Units::splits).
constexpr int token_fewest(int hd) { return 1024 / hd; }
constexpr int ROWS_FEWEST = 4;
template <class How> __device__ __forceinline__ Blocks<32, How> token_blocks(const Rows &s, const How &mask, int b, int pos) {
    return blocks_of<32>(mask, (uint32_t)pos, min((uint32_t)pos, s.cap - 1), prefix_of(mask, b), doc_of(mask, b));
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
template <class How> __device__ __forceinline__ int token_least(const Rows &s, const How &mask, int groups, int slots, int fewest) {
    return fitting(s, groups, slots, fewest, [&](int b, float &n, float &u) {
        const int pos = s.pos[b];
        n = pos < 0 ? 0.f : (float)token_blocks(s, mask, b, pos).n;
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
// 64 tokens of up to 8192, 40 heads on 8: 41 / 46; codes of 256, up to 4096, 37 / 51.  Halves of 128 take 168
// registers, three waves, and scored 173, two: 64 tokens of up to 8191 plain / biased / capped 85.5 / 87.3 / 87.2 us, 32
// of up to 3000 22.1 / 25.2 / 24.6; codes (139 and 144 registers) 37.1 / 38.4 / 38.9 and 19.7 / 21.1 / 21.3.
constexpr int TW = 4;                            // waves
constexpr float LAZY = 7.f;                      // how far (log2) weights may pass the maximum they stand at
                                                 // (0, as ever: 1 to 6% more time)
constexpr int MAX_SPLITS = 64;                   // what the combine weighs in one wave

template <int HD, bool I8, bool TILED, typename T, class How>
__global__ __launch_bounds__(64 * TW) __attribute__((amdgpu_waves_per_eu(I8 || HD == 128 ? 2 : 1))) void k_attn_tokens(
        Cache c, Rows s, const T *q, int64_t q_stride, const T *gate, int64_t gate_stride, T *out, Part part, int most,
        int slots, int H, float scale, How mask) {
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
        auto splits = [&](const Seq &q, int b) { return q.r1 > q.r0 ? token_blocks(s, mask, b, q.pos).splits(most, least) : 0; };
        Seq sq;
        //   A workgroup a CU (ONE): by the splits' lengths in quarters, as a slot's last one is not
        // hidden behind another: 64 of up to 12000, halves, 24 of 256 on 4, 111 us in two classes, 102
        // in four, under a window of 4096 83 and 75.5; codes of 128, two a CU, 34.8 and 35.2.
        constexpr bool ONE = !I8 && HD == 256;
        auto order = [&](const Seq &q, int b) {
            const Blocks<32, How> kb = token_blocks(s, mask, b, q.pos);
            if (!ONE) return q.r1 > q.r0 && kb.n > 0.5f * least ? 0 : 1;
            const float part = q.r1 > q.r0 ? (float)kb.n / (float)(kb.splits(most, least) * least) : 0.f;
            return part > 0.75f ? 0 : part > 0.5f ? 1 : part > 0.25f ? 2 : 3;
        };
        if (!unit_at<ONE ? 4 : 2>(s, n, splits, order, n, sp, sq)) return;
        pos = sq.pos;
        ns = token_blocks(s, mask, n, pos).splits(most, least);
    } else {
        pos = s.pos[n];
        if (pos < 0) return;
    }
    const Blocks<32, How> kb = token_blocks(s, mask, n, pos);
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
        bool seen = there && e.kp <= (uint32_t)pos && (e.kp >= kb.lo || e.kp < kb.sinks);
        if constexpr (How::SCORED) seen &= e.kp >= kb.doc;
        return Key{there ? row_at<I8>(c, e.page, slot_of(c, e.kp), kvh) : (uint32_t)(I8 ? 0 : kvh), seen};
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
    // A score over its cap; the units of scores once they are capped, and once they are biased.
    float slope = 0.f, to_x = 0.f, capped = sf, unit = sf;
    if constexpr (How::SCORED) {
        if (mask.slope) slope = slope_of(mask, h0 + min(col, nh - 1));
        to_x = over_cap(sf, mask);
        if (mask.cap > 0.f) capped = unit = 1.f;
        if (mask.slope) unit = 1.f;
    }
    const float none = unit < 0.f ? INFINITY : -INFINITY;    // the score of no key
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
        const int now = j;
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
        const uint32_t mine = seen >> (4 * g);
        auto unseen = [&](float x) {
            if (seen == 0xffffffffu) return;
            asm volatile("");
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int v = 0; v < 4; v++) sc[kt][v] = mine & (1u << (16 * kt + v)) ? sc[kt][v] : x;
        };
        if constexpr (How::SCORED) {
            if (mask.cap > 0.f) cap_scores<false, 2, 4>(mask, to_x, sc);
            if (mask.slope) {
                // (All seen keys lie before the token.)
                const float b = -slope * (float)(int)((uint32_t)pos - kb.start(now) - 4 * g);
#pragma unroll
                for (int kt = 0; kt < 2; kt++)
#pragma unroll
                    for (int v = 0; v < 4; v++) sc[kt][v] = fmaf(sc[kt][v], capped, fmaf(slope, (float)(16 * kt + v), b));
            }
        }
        unseen(none);
        float top = -INFINITY;                   // of this lane's keys
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int v = 0; v < 4; v++) top = fmaxf(top, sc[kt][v] * unit);
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
                float p = __builtin_amdgcn_exp2f(fmaf(sc[kt][v], unit, -m)) * 256.f;
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
// 4096 under a window of 1024 124 us, 610; f32 rows (twice the products) of 24 heads of 256
// on 4 530.  No unit of the CU is full (matrix cores 31% busy, vector ALUs 50%, LDS 31%):
// with the registers of two waves a SIMD a wave's chain of staging, scores, weights and sums
// is what lasts, 2.0 to 2.5 us for two waves' tiles, a lone one 1.7.  (f32 rows of 128 take all
// 256 registers; capped ones keep 21 more in memory on halves, 18 on those of odd pages, 3 on codes; by the
// quotient or without a cap 5, 7 and none.)  Results leave through LDS, which takes the 16 bytes a lane and line that
// the products' layout gives (calls of 20 mixed f32 chunks 115 -> 106 us, the window's 132 -> 124).  Measured and left out:
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
template <int PC, int AK, class How> struct Units {
    int rows, G;
    FastDiv by_g;                                // (a division by G is some 30 instructions, and there are many)
    uint32_t pos, cap;
    uint32_t prefix;                             // of the sequence's positions
    __device__ __forceinline__ Units(const Seq &q, int G_, const FastDiv &by_g_, uint32_t cap_, const How &mask, int b)
        : rows(q.r1 - q.r0), G(G_), by_g(by_g_), pos(q.pos), cap(cap_), prefix(min(prefix_of(mask, b), pos + rows)) {}
    __device__ __forceinline__ int n() const { return (int)(((int64_t)rows * G + PC - 1) / PC); }
    __device__ __forceinline__ int first(int k) const { return (int)by_g(k * PC); }
    __device__ __forceinline__ int last(int k) const { return min((int)by_g(k * PC + PC - 1), rows - 1); }
    // Position of the last key that some row up to i sees.
    __device__ __forceinline__ uint32_t last_key(int i) const { return How::SCORED ? max(pos + i, prefix - (prefix > 0)) : pos + i; }
    __device__ __forceinline__ Blocks<AK, How> blocks(const How &mask, int k, uint32_t doc = 0) const {
        return blocks_of<AK>(mask, pos + first(k), min(last_key(last(k)), cap - 1), prefix, doc);
    }
    // Splits of each of the units: as the longest, the last, needs them.  Scored: with the
    // documents left out, so that a unit may have fewer blocks than these are made for, down to one a split, its
    // start and its partials (us so / keys left whole: 8 chunks of up to 200 rows behind up to 12000, documents of up to
    // 200, 31.9 / 17.0, 4 of 256 behind 20000, of 300, 30.3 / 23.2; 256 rows behind 20000, of 10000, 87 / 362: a call's
    // max_len says which).
    __device__ __forceinline__ int splits(const How &mask, int most, int least) const {
        const int longest = blocks(mask, n() - 1).n;
        return longest <= 1.4f * least ? 1 : min(most, (longest + least - 1) / least);
    }
    // Unit k from the last one back, with those first that a document gives over half the most
    // keys, then a quarter: a workgroup of 20 tiles that starts last is the call's time.  Long documents gain by it
    // and short ones lose, as every workgroup works the order out, and the documents are not known before (us in the
    // rows' order / so, 40 heads of 128 on 8: 4096 rows, two and a half rounds of workgroups, of documents of up to
    // 1500 109 / 100, 300 61.5 / 64.7, 100 53.4 / 59.7, 30 51.3 / 55.4; 3000 of up to 3000 93.4 / 91.5).
    __device__ __forceinline__ int by_document(const How &mask, int k, int r0) const {
        constexpr int MOST = 8;                  // units a lane
        const int lane = threadIdx.x & 63, last_unit = n() - 1;
        if (last_unit >= 64 * MOST) return k;
        uint32_t keys[MOST], most = 0;
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            const int x = 64 * i + lane;
            keys[i] = 0;
            if (64 * i <= last_unit && x <= last_unit) keys[i] = max((int)(pos + last(x) - doc_of(mask, r0 + first(x))), 0);
            most = max(most, keys[i]);
        }
        most = ~wave_least(~most);
        int at = last_unit - k;
#pragma unroll
        for (int c = 0; c < 3; c++)
#pragma unroll
            for (int i = MOST - 1; i >= 0; i--) {
                if (64 * i > last_unit) continue;
                const int mine = keys[i] > most / 2 ? 0 : keys[i] > most / 4 ? 1 : 2;
                const uint64_t in = __ballot(mine == c && 64 * i + lane <= last_unit);
                if (at < __popcll(in)) {
                    const bool here = (in >> lane & 1) && __popcll(in >> lane >> 1) == at;
                    return 64 * i + __ffsll((unsigned long long)__ballot(here)) - 1;
                }
                at -= __popcll(in);
            }
        return k;                                // (not reached)
    }
};
// A unit's n blocks in nz splits or fewer: `per` each, `used` splits.
struct Cut {
    int per, used;
    __device__ __forceinline__ Cut(int n, int nz) : per(max(1, (n + nz - 1) / nz)), used(max(1, (n + per - 1) / per)) {}
};
// How finely the keys are split, as token_least, each of a sequence's units taken for its
// longest.
template <int PC, int AK, class How>
__device__ __forceinline__ int unit_least(const Rows &s, const How &mask, int G, const FastDiv &by_g, int HKV, int slots) {
    return fitting(s, HKV, slots, ROWS_FEWEST, [&](int b, float &n, float &u) {
        const Units<PC, AK, How> q(seq_at(s, b), G, by_g, s.cap, mask, b);
        u = q.rows > 0 ? (float)q.n() : 0.f;
        n = q.rows > 0 ? (float)q.blocks(mask, q.n() - 1).n : 0.f;
    });
}

template <int HD, bool I8, bool TILED, typename T, class How>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void k_attn_rows(Cache c, Rows s, const T *q, int64_t q_stride, const T *gate, int64_t gate_stride, T *out, Part part,
                 int most, int slots, int H, float scale, How mask, FastDiv by_g) {
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
    constexpr int OP = HD + 4;                   // results' rows, 16 bytes apart in LDS's banks
    static_assert((size_t)PC * OP * 4 <= sizeof(f16) * 2 * AK * (KP + VP), "results take the tiles' place");
    __shared__ union __attribute__((aligned(16))) {
        struct {
            f16 K[2][AK][KP], V[2][AK][VP];
        };
        float O[PC][OP];                         // at the end, the columns' results
    } lds;
    auto &Ks = lds.K;
    auto &Vs = lds.V;
    __shared__ int2 out_row[PC];                 // of a column: its row, and that times H + its head (-1 past the last one)
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
    const int least = most > 1 ? unit_least<PC, AK, How>(s, mask, G, by_g, c.HKV, slots) : 0;
    auto units = [&](const Seq &q, int b) {
        const Units<PC, AK, How> u(q, G, by_g, s.cap, mask, b);
        return u.rows <= 0 ? 0 : u.n() * (most > 1 ? u.splits(mask, most, least) : 1);
    };
    Seq sq;
    auto order = [&](const Seq &q, int b) {
        const Units<PC, AK, How> u(q, G, by_g, s.cap, mask, b);
        const int n = u.rows > 0 ? u.blocks(mask, u.n() - 1).n : 0;
        return n > 0.35f * least ? 0 : n > 0.1f * least ? 1 : 2;
    };
    if (!unit_at<3>(s, blockIdx.x / c.HKV, units, order, b, k, sq)) return;
    const Units<PC, AK, How> un(sq, G, by_g, s.cap, mask, b);
    const int rows = un.rows;
    if (most > 1) nz = un.splits(mask, most, least);
    const int z = k % nz;
    k = un.n() - 1 - k / nz;
    if constexpr (How::SCORED)
        if (mask.first && (int)gridDim.x > slots) k = un.by_document(mask, k, sq.r0);
    const struct { int i0, i1; } tl = {un.first(k), un.last(k)};
    const uint32_t p0 = (uint32_t)sq.pos, cap1 = s.cap - 1;
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int lc = lane % MF, h = lane / MF;
    // This lane's column, and the positions that the wave's columns stand at.
    const int col = k * PC + MF * w + lc, i = min((int)by_g(col), rows - 1);
    const bool valid = col < rows * G;
    const int head = kvh * G + (valid ? col - i * G : G - 1);
    const int64_t n = sq.r0 + i;
    const uint32_t p = p0 + i;
    if (h == 0) out_row[MF * w + lc] = make_int2((int)n, valid ? (int)n * H + head : -1);
    // The column's row of q, and scored rows' documents and slope: all requested at once (what they
    // wait for one after the other is a microsecond each).
    typedef T T8 __attribute__((ext_vector_type(8), aligned(16)));
    T8 qraw[KS];
    {
        const T *qrow = q + n * q_stride + (int64_t)head * HD + 8 * h;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qraw[ks] = *(const T8 *)(qrow + 512 / MF * ks);
    }
    uint32_t doc = 0, doc0 = 0, doc1 = 0, docs0 = 0, docs1 = 0;      // the column's; the unit's and the wave's first and last
    float slope = 0.f;
    if constexpr (How::SCORED) {
        if (mask.slope) slope = slope_of(mask, head);
        if (mask.first) {
            doc = doc_of(mask, n);
            uint32_t a = doc, z = doc;           // (a wave's columns, then all rows of the unit, of which it has some)
            constexpr int RL = PC / 64 + 1;
            uint32_t d[RL];
#pragma unroll
            for (int x = 0; x < RL; x++) d[x] = tl.i0 + lane + 64 * x <= tl.i1 ? doc_of(mask, sq.r0 + tl.i0 + lane + 64 * x) : doc;
#pragma unroll
            for (int x = 0; x < RL; x++) {
                a = min(a, d[x]);
                z = max(z, d[x]);
            }
            doc0 = wave_least(a);
            doc1 = ~wave_least(~z);
        }
    }
    const Blocks<AK, How> kb = un.blocks(mask, k, doc0);
    const Cut cut(kb.n, nz);
    if (z >= cut.used) return;
    nz = cut.used;
    const int per = cut.per, jend = min(kb.n, (z + 1) * per);
    const bool busy = k * PC + MF * w < rows * G;
    const uint32_t plo = p0 + min((int)by_g(k * PC + MF * w), rows - 1);
    const uint32_t seen_from = mask.window && plo >= (uint32_t)mask.window ? plo - mask.window + 1 : 0;
    const uint32_t phi = p0 + min((int)by_g(k * PC + MF * w + MF - 1), rows - 1);
    // Scored: positions that every row sees whole, before the window too, and this column's document.
    const uint32_t sinks = How::SCORED ? max((uint32_t)mask.sinks, un.prefix) : (uint32_t)mask.sinks;
    if constexpr (How::SCORED)
        if (mask.first) {
            docs0 = wave_least(doc);
            docs1 = ~wave_least(~doc);
        }
    auto sees = [&](uint32_t t) {                // whether this column sees position t, if its page is there
        const bool near = t <= p && (!mask.window || t + mask.window > p || t < (uint32_t)mask.sinks);
        if constexpr (How::SCORED) return (near || t < un.prefix) && t >= doc;
        else return near;
    };
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
        const bool there = (uint32_t)e.page < c.n_pages && e.kp < s.cap && e.kp <= un.last_key(tl.i1);
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
        whole = in == ALL && (k0 + AK - 1 <= p0 + tl.i0 || (How::SCORED && k0 + AK <= un.prefix)) &&
                (!mask.window || k0 + mask.window > p0 + tl.i1 || k0 + AK <= sinks) && (!How::SCORED || k0 >= doc1);
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
        const bool neg = scale < 0.f;
        if (j < jend) fetch(en);                 // (while the rows are on their way)
        en = entry_of(j + 1);
        if constexpr (HL) {
            float mx = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(qraw[ks][e]));
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
                    gd_split_f16(qraw[ks][e] * up, hi, lo);
                    qh[ks][e] = hi;
                    ql[ks][e] = lo;
                }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) qh[ks] = __builtin_bit_cast(f16x8, qraw[ks]);
            if (neg)
#pragma unroll
                for (int ks = 0; ks < KS; ks++) qh[ks] = -qh[ks];
        }
    }
    if (sf < 0x1p-126f) sf = 0x1p-126f;          // weights of 1 alike; times -inf not NaN
    // A score over its cap; the units of scores once they are capped, and once they are biased.
    float to_x = 0.f, capped = sf, unit = sf;
    if constexpr (How::SCORED) {
        to_x = over_cap(sf, mask);
        if (How::BY_EXP || mask.cap > 0.f) capped = unit = 1.f;
        if (mask.slope) unit = 1.f;
    }
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
        if (busy && k0 <= un.last_key(phi - p0) && !(seen_from > k0 + AK - 1 && k0 >= sinks) && (!How::SCORED || docs0 < k0 + AK)) {
            const bool full = now == ALL && (k0 + AK - 1 <= plo || (How::SCORED && k0 + AK <= un.prefix)) &&
                              (!mask.window || k0 + mask.window > phi || k0 + AK <= sinks) && (!How::SCORED || k0 >= docs1);
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
            uint64_t see = 0;                    // a bit a key, as this column sees it
            if (!full) {
                auto below = [](int64_t x) { return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1; };
                see = below((int64_t)p - k0 + 1);
                if (mask.window) see &= ~below((int64_t)p - mask.window + 1 - k0) | below((int64_t)mask.sinks - k0);
                if constexpr (How::SCORED) see = (see | below((int64_t)un.prefix - k0)) & ~below((int64_t)doc - k0);
                see = (see & now) >> (4 * h);
            }
            auto unseen = [&](float x) {
                if (full) return;
#pragma unroll
                for (int kt = 0; kt < NT; kt++) {
                    const uint32_t bits = (uint32_t)(see >> (MF * kt));
#pragma unroll
                    for (int v = 0; v < NV; v++) st[kt][v] = bits & (1u << (8 * (v / 4) + v % 4)) ? st[kt][v] : x;
                }
            };
            if constexpr (How::SCORED) {
                if constexpr (How::BY_EXP) cap_scores<true, NT, NV>(mask, to_x, st);
                else if (mask.cap > 0.f) cap_scores<false, NT, NV>(mask, to_x, st);
                if (mask.slope) {
                    const float d = (float)(int)(p - k0 - 4 * h);
#pragma unroll
                    for (int kt = 0; kt < NT; kt++)
#pragma unroll
                        for (int v = 0; v < NV; v++)
                            st[kt][v] = fmaf(-slope, fabsf(d - (float)(MF * kt + 8 * (v / 4) + v % 4)), st[kt][v] * capped);
                }
            }
            unseen(-INFINITY);
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < NT; kt++)
#pragma unroll
                for (int v = 0; v < NV; v++) top = fmaxf(top, st[kt][v]);
            // Sums are brought to a new maximum only where a score is over 2^LAZY of the one
            // they stand at (random scores: hardly after the first tiles).
            if (__any(top * unit > m + LAZY)) {
                if constexpr (MF == 16) top = fmaxf(top, __shfl_xor(top, 16, 64));
                const float mn = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)) * unit);
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
                    float w0 = __builtin_amdgcn_exp2f(fmaf(st[kt][v], unit, off));
                    float w1 = __builtin_amdgcn_exp2f(fmaf(st[kt][v + 1], unit, off));
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
                if (sees(kb.start(j) + key) && (now >> key & 1))
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int v = 0; v < NV; v++)
                            if (odd[s2][key][(MF * dt + 8 * (v / 4) + 4 * h) / 8] >> (4 * h % 8 + v % 4) & 1) acc[dt][v] = __uint_as_float(0x7fc00000u);
            __syncthreads();
        }
        now = next;
    }
    // Through LDS, each wave its own columns, so that a row is written, and its gate read, in whole lines.
    constexpr int TPR = HD / 8, RPP = 64 / TPR, PASS = MF / RPP;     // lanes of a row, eight dims each; rows of a pass
    const int d = 8 * (lane % TPR), r0 = MF * w + lane / TPR;
    T8 gates[PASS];
    if (gate && nz == 1)
#pragma unroll
        for (int x = 0; x < PASS; x++) {
            const int2 row = out_row[r0 + x * RPP];
            if (row.y >= 0) gates[x] = *(const T8 *)(gate + row.x * gate_stride + (row.y - (int64_t)row.x * H) * HD + d);
        }
    if constexpr (MF == 16) l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int64_t mine = out_row[MF * w + lc].y; // (not what it was made of, which would cost registers all along)
    if (mine >= 0 && h == 0) {
        if (most > 1 && z == 0) part.used[mine] = nz;
        if (nz > 1) part.ml[mine * most + z] = make_float2(m, l);
    }
    const float inv = nz > 1 ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int x = 0; x < DT; x++)
#pragma unroll
        for (int v = 0; v < NV; v += 4)
            *(f32x4 *)&lds.O[MF * w + lc][MF * x + 2 * v + 4 * h] =
                    f32x4{acc[x][v] * inv, acc[x][v + 1] * inv, acc[x][v + 2] * inv, acc[x][v + 3] * inv};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int x = 0; x < PASS; x++) {
        const int r = r0 + x * RPP;
        const int64_t row = out_row[r].y;
        if (row < 0) continue;
        f32x4 y[2] = {*(const f32x4 *)&lds.O[r][d], *(const f32x4 *)&lds.O[r][d + 4]};
        if (nz > 1) {
            float *p = part.acc + (row * most + z) * HD + d;
            *(f32x4 *)p = y[0];
            *(f32x4 *)(p + 4) = y[1];
            continue;
        }
        if (gate)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float g = to_f32<T>(gates[x][e]);
                y[e / 4][e % 4] *= HL ? gd_sigmoid(g) : __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * g));
            }
        T8 res;
#pragma unroll
        for (int e = 0; e < 8; e++) res[e] = from_f32<T>(y[e / 4][e % 4]);
        *(T8 *)(out + row * HD + d) = res;
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

// ---------------------------------------------------------------- launch

struct AttnArgs {
    const gd_kv *kv;
    const gd_seqs *s;
    const void *q;
    int64_t q_stride;
    const void *gate;
    int64_t gate_stride;
    void *out;
    int x_dtype, n_head;
    float scale;
};

// Checks a call's arguments, before the context, and launches it.  `bounded`: no key but those
// of the window and the sinks is seen.
template <class How>
int attn(gd_ctx *ctx, const char *fn, const AttnArgs &a, int window, int n_sink, const How &mask, bool bounded) {
    const auto [kv, s, q, q_stride, gate, gate_stride, out, x_dtype, n_head, scale] = a;
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
    auto apart = [&, out = out, s = s](const void *x, int64_t stride) {
        const uintptr_t a = (uintptr_t)x, o = (uintptr_t)out, end = a + ((s->n_rows - 1) * stride + row) * size;
        return !x || !span || (a == o && stride == row) || end <= o || o + span <= a;
    };
    GD_REQUIRE(ctx, apart(q, q_stride) && apart(gate, gate_stride),
               "%s: out in place of q or gate needs their place and rows of n_head * head_dim", fn);
    GD_CHECK_CTX(ctx);
    if (!s->n_rows || !s->n_seq) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    const int cus = ctx->num_cus > 0 ? ctx->num_cus : 256;
    const Rows rows = rows_of(kv, s);
    int64_t keys = s->max_len ? std::min<int64_t>(s->max_len, rows.cap) : rows.cap;
    const int width = tokens ? 32 : hd == 128 ? tile_keys<128>() : tile_keys<256>();
    if (window && bounded)
        keys = std::min(keys, (int64_t)window + (tokens ? 0 : cols / G) + width - 1 + ((int64_t)n_sink + width - 1) / width * width);
    // Blocks of keys of the longest row, workgroups of a split each, those that the chip
    // holds at once, and the most splits.  The keys are left whole, without a merge's
    // launch, where that is a few rounds of blocks a wave or the workgroups are many; how
    // finely others are split, the kernels know (token_least, unit_least).  (Measured below with
    // plain scores, and taken for all.)
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
        if (tokens) { \
            auto kernel = tiled ? k_attn_tokens<HD_, I8_, true, T_, typename How::Tokens> : k_attn_tokens<HD_, I8_, I8_, T_, typename How::Tokens>; \
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, cache_of(kv), rows, (const T_ *)q, q_stride, \
                               (const T_ *)gate, gate_stride, (T_ *)out, part, (int)ns, (int)slots, n_head, scale, \
                               (typename How::Tokens)mask); \
        } else { \
            auto kernel = tiled ? k_attn_rows<HD_, I8_, true, T_, How> : k_attn_rows<HD_, I8_, I8_, T_, How>; \
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, ctx->stream, cache_of(kv), rows, (const T_ *)q, q_stride, \
                               (const T_ *)gate, gate_stride, (T_ *)out, part, (int)ns, (int)slots, n_head, scale, mask, \
                               FastDiv((uint32_t)G)); \
        } \
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

}  // namespace
