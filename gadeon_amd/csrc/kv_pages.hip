// The pages of the paged KV cache: which sequence holds which, on the device, so that a
// serving loop that forks, extends, ends and packs conversations needs no host round trip.
// One table and one count of references serve all layers' caches; copies of pages that a
// call decides on go into a list, which gd_kv_copy_pages carries out for every layer.
//
// The reference keeps one conversation's pages in a pool of the host (MetalKVPool.swift:
// pages allocated one by one, a snapshot shares full ones and copies the last).
#include "kv_core.h"

namespace {

// What the kernels need of a gd_kv_pages.  Its arrays are device data: no entry of them is
// trusted with an address.
struct Pages {
    int32_t *refs, *table;
    uint32_t n_pages;
    int n_seq, max_pages, P;
    __device__ __forceinline__ bool there(int page) const { return (uint32_t)page < n_pages; }
    __device__ __forceinline__ int32_t *row(int b) const { return table + (int64_t)b * max_pages; }
};

__device__ __forceinline__ void count(const Pages &pg, int page, int by) {
    if (pg.there(page)) (void)__hip_atomic_fetch_add(&pg.refs[page], by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------- fork, release

constexpr int EW = 1024;                         // entries that a workgroup works on at once
constexpr int MOST_WGS = 16384;                  // orders times parts of a row, but for a workgroup an order

// Workgroup (order i, EW entries and every gridDim.y-th of them on): row dst[i] takes over src[i]'s entries
// of the first len[i] positions.  No source is the place of another order, so that rows are only read or only
// written; counts are whole numbers, whose order of addition shows nowhere.
//   The counts bound many orders: 400 of 2048 entries add 138 000 of them in random lines in 11 us (with
// the ends of 300 others 22 a pass, without any count 12); few are a launch and three loads, 2.4.  Each
// order looks at all of them, once a workgroup: 8192 rows of 1024 44 us, 65536 2.0 ms.
__global__ __launch_bounds__(256) void k_fork(Pages pg, const int32_t *src, const int32_t *dst, const int32_t *len, int n) {
    const int i = blockIdx.x, s = src[i], d = dst[i], most = len[i];
    if ((uint32_t)s >= (uint32_t)pg.n_seq || (uint32_t)d >= (uint32_t)pg.n_seq) return;
    const int32_t *from = pg.row(s);
    int32_t *to = pg.row(d);
    for (int y = blockIdx.y; y * EW < pg.max_pages; y += gridDim.y) {
        const int e0 = y * EW + threadIdx.x;
        int old[EW / 256], now[EW / 256];
#pragma unroll
        for (int x = 0; x < EW / 256; x++) {
            const int e = e0 + 256 * x;
            old[x] = e < pg.max_pages ? to[e] : -1;
            now[x] = e < pg.max_pages && (int64_t)e * pg.P < most ? from[e] : -1;
        }
        if (y == (int)blockIdx.y) {              // (seen while the rows are on their way)
            bool bad = false;
            for (int j = threadIdx.x; j < n; j += 256) bad |= src[j] == d || (j > i && dst[j] == d);
            if (__syncthreads_or(bad)) return;
        }
#pragma unroll
        for (int x = 0; x < EW / 256; x++) {
            if (!pg.there(now[x])) now[x] = -1;
            if (old[x] == now[x]) continue;
            count(pg, old[x], -1);
            count(pg, now[x], 1);
            to[e0 + 256 * x] = now[x];
        }
    }
}

// Workgroup (order i, EW entries and on, as k_fork): sequence seq[i] drops the pages that hold no position
// of from[i] .. to[i] - 1, nor one of its first keep[seq[i]] before to[i].  Other orders may name the
// sequence too: an entry is counted by the one that exchanges it, and none looks at another (8192 orders of
// one sequence, rows of 1024, 13 us, 65536 42; each walking those before it 13.8 ms for 8192, and with the square of
// their number).
__global__ __launch_bounds__(256) void k_release(Pages pg, const int32_t *keep, const int32_t *seq, const int32_t *from,
                                                 const int32_t *to) {
    const int i = blockIdx.x, b = seq[i];
    if ((uint32_t)b >= (uint32_t)pg.n_seq) return;
    const int kept = keep ? keep[b] : 0;
    const int first = from ? from[i] : 0, end = to[i];
    auto drops = [&](int e) {
        const int64_t p = (int64_t)e * pg.P;
        return !((p + pg.P > first || p < kept) && p < end);
    };
    int32_t *row = pg.row(b);
    for (int y = blockIdx.y; y * EW < pg.max_pages; y += gridDim.y) {
        const int e0 = y * EW + threadIdx.x;
        int old[EW / 256];
#pragma unroll
        for (int x = 0; x < EW / 256; x++) {
            const int e = e0 + 256 * x;
            old[x] = e < pg.max_pages && drops(e) ? row[e] : -1;
        }
#pragma unroll
        for (int x = 0; x < EW / 256; x++)
            if (pg.there(old[x])) {
                int32_t was = old[x];
                if (__hip_atomic_compare_exchange_strong(row + e0 + 256 * x, &was, -1, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                         __HIP_MEMORY_SCOPE_AGENT))
                    count(pg, old[x], -1);
            }
    }
}

// ---------------------------------------------------------------- reserve


// Sum over the threads up to this one; `all` gets the whole sum.  LDS `sums` of two times T / 64
// ints, halves in turn (a barrier a call).  (Held at 2^29, which is over all entries that there
// may be: sequences that share rows could pass 2^31.)
template <int T> __device__ __forceinline__ int block_scan(int v, int *sums, int &turn, int &all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int sum = wave_scan(v);
    int *s = sums + (turn ^= 1) * (T / 64);
    if (lane == 63) s[w] = sum;
    __syncthreads();
    int before = 0;
    all = 0;
    for (int i = 0; i < T / 64; i++) {
        before = min(before + (i < w ? s[i] : 0), 1 << 29);
        all = min(all + s[i], 1 << 29);
    }
    return before + sum;
}

// The counts of pages p .. p + 15 (1 behind the last one), and which are free, a bit each.
struct Counts {
    typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));
    i32x4 r[4];
    __device__ __forceinline__ Counts() {}
    __device__ __forceinline__ Counts(const Pages &pg, uint32_t p) {
        if (p + 16 <= pg.n_pages) {
#pragma unroll
            for (int j = 0; j < 4; j++) r[j] = *(const i32x4 *)(pg.refs + p + 4 * j);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) r[j / 4][j % 4] = p + j < pg.n_pages ? pg.refs[p + j] : 1;
        }
    }
    __device__ __forceinline__ int least() const {
        int m = 1;
#pragma unroll
        for (int j = 0; j < 16; j++) m = min(m, r[j / 4][j % 4]);
        return m;
    }
    __device__ __forceinline__ uint32_t free() const {
        uint32_t f = 0;
#pragma unroll
        for (int j = 0; j < 16; j++) f |= (r[j / 4][j % 4] <= 0) << j;
        return f;
    }
};

// The lowest `needs` free pages, in order, into fresh; how many there are.  `first`: the counts of
// pages 16 t .., on their way since before.  As the lowest free pages are taken first, those before
// them are in use: they are passed 64 a thread (32 of 1024 threads), by a look at the least count. (64 tokens
// behind 131072 pages in use 23 us, of which 9 without them; by 16 a thread, all ranked, 37.)
template <int T>
__device__ __forceinline__ int take_free(const Pages &pg, const Counts &first, int needs, int32_t *fresh, int *sums, int &turn) {
    int found = 0, all;
    auto take = [&](uint32_t free, uint32_t p) {
        const int n = __popc(free);
        int at = found + block_scan<T>(n, sums, turn, all) - n;
        for (; free && at < needs; free &= free - 1) fresh[at++] = (int32_t)p + __ffs(free) - 1;
        found += all;
    };
    if (needs) take(first.free(), 16 * threadIdx.x);
    constexpr int PARTS = T > 256 ? 2 : 4;       // (registers)
    for (uint32_t p0 = 16 * T; p0 < pg.n_pages && found < needs; p0 += 16 * PARTS * T) {
        Counts c[PARTS];
        int least = 1;
#pragma unroll
        for (int i = 0; i < PARTS; i++) c[i] = Counts(pg, p0 + 16 * (i * T + threadIdx.x));
#pragma unroll
        for (int i = 0; i < PARTS; i++) least = min(least, c[i].least());
        if (!__syncthreads_or(least <= 0)) continue;
#pragma unroll
        for (int i = 0; i < PARTS; i++) take(c[i].free(), p0 + 16 * (i * T + threadIdx.x));
    }
    return found;
}

// Per sequence where its entries start among all; per page the entries that share it and the
// last of them; per entry (of the rows of the call, sequence by sequence) what is known of it.
struct Work {
    int32_t *start, *uses, *last, *seq, *entry, *page, *flags, *rank, *fresh;
    int most;                                    // entries that there is room for
    static size_t ints(int64_t n_seq, int64_t n_pages, int64_t most) { return n_seq + 1 + 2 * n_pages + 6 * most; }
};
enum { NEED = 1, KEEP = 2, SHARED = 4, TAIL = 8 };

// One workgroup: the entries of the new rows in order, which of them need a page (none there,
// or one shared with others, of which the last keeps it if no other than these name it), the
// first free pages in order, the k-th need the k-th page.  A sequence gets all or nothing:
// what it needs, if all up to it fits.
//   The chain of its steps bounds it, a dozen of some 0.7 us each.
constexpr int RT = 1024;                         // threads
__global__ __launch_bounds__(RT) void k_reserve(Pages pg, Rows s, FastDiv by_page, Work wk, int32_t *copies, int32_t *n_copies,
                                                int32_t *pos_out) {
    __shared__ int sums[2 * RT / 64];
    const int t = threadIdx.x;
    int turn = 0, all;
    // Entries of each sequence.
    int entries = 0;
    for (int b0 = 0; b0 < s.n_seq; b0 += RT) {
        const int b = b0 + t;
        int n = 0, pos = -1;
        if (b < s.n_seq) {
            pos = s.pos[b];
            const Seq q = seq_at(s, b);
            if (q.r1 > q.r0 && (uint32_t)q.pos < s.cap) {
                const uint32_t last = min((uint32_t)q.pos + (uint32_t)(q.r1 - q.r0 - 1), s.cap - 1);
                n = (int)(by_page(last) - by_page(q.pos)) + 1;
            }
        }
        const int upto = block_scan<RT>(n, sums, turn, all);
        if (b < s.n_seq) {
            wk.start[b] = min(entries + upto - n, wk.most);
            pos_out[b] = pos;
            // (More than there is room for only of rows that sequences share.)
            for (int i = 0, c = entries + upto - n; i < n && c < wk.most; i++, c++) {
                const int e = (int)by_page(pos) + i;
                wk.seq[c] = b;
                wk.entry[c] = e;
                wk.flags[c] = (int64_t)e * pg.P < pos ? TAIL : 0;
            }
        }
        entries = min(entries + all, wk.most);
    }
    if (t == 0) wk.start[s.n_seq] = entries;
    __syncthreads();
    // The pages that they name; those shared are counted.
    bool some = false;
    for (int c = t; c < entries; c += RT) {
        const int page = pg.row(wk.seq[c])[wk.entry[c]];
        const bool there = pg.there(page), shared = there && pg.refs[page] > 1;
        wk.page[c] = there ? page : -1;
        if (shared) {
            wk.flags[c] |= SHARED;
            wk.uses[page] = 0;
            wk.last[page] = -1;
            some = true;
        }
    }
    __threadfence();
    some = __syncthreads_or(some);
    if (some) {
        for (int c = t; c < entries; c += RT)
            if (wk.flags[c] & SHARED) {
                atomicAdd(&wk.uses[wk.page[c]], 1);
                atomicMax(&wk.last[wk.page[c]], c);
            }
        __threadfence();
        __syncthreads();
    }
    auto now = [](const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    int needs = 0;
    for (int c0 = 0; c0 < entries; c0 += RT) {
        const int c = c0 + t;
        int f = 0;
        if (c < entries) {
            const int page = wk.page[c];
            f = wk.flags[c];
            if (page < 0) f |= NEED;
            else if (f & SHARED) f |= now(&wk.uses[page]) == pg.refs[page] && now(&wk.last[page]) == c ? KEEP : NEED;
            wk.flags[c] = f;
        }
        const int upto = block_scan<RT>(f & NEED ? 1 : 0, sums, turn, all);
        if (c < entries) wk.rank[c] = needs + upto;
        needs += all;
    }
    const int found = take_free<RT>(pg, Counts(pg, 16 * t), needs, wk.fresh, sums, turn);
    __syncthreads();
    int copied = 0;
    for (int c0 = 0; c0 < entries; c0 += RT) {
        const int c = c0 + t;
        bool copy = false;
        int old = -1, page = -1;
        if (c < entries) {
            const int f = wk.flags[c], b = wk.seq[c];
            if (f & (NEED | KEEP)) {
                const int whole = wk.rank[min(wk.start[b + 1], entries) - 1];    // needs up to the sequence's end
                if (whole > found) {
                    pos_out[b] = -1;
                } else if (f & NEED) {
                    old = wk.page[c];
                    page = wk.fresh[wk.rank[c] - 1];
                    pg.row(b)[wk.entry[c]] = page;
                    pg.refs[page] = 1;
                    count(pg, old, -1);
                    copy = (f & (SHARED | TAIL)) == (SHARED | TAIL);
                }
            }
        }
        const int upto = block_scan<RT>(copy, sums, turn, all);
        if (copy) {
            copies[2 * (copied + upto - 1)] = old;
            copies[2 * (copied + upto - 1) + 1] = page;
        }
        copied += all;
    }
    if (t == 0) *n_copies = copied;
}

// The same for 4 T sequences and entries at most, in registers and LDS, T of them a round.  Single
// rows' entries are the sequences; others' are found by the sequence that starts last at or before
// each.  Shared pages are counted in a table by a hash of theirs, whose places depend on who comes
// first, but not what stands there.
//   A chain of three loads (row, entry, count) and a dozen short steps bounds it: 6.7 us for 64
// tokens, 8.6 for 200 prompts (k_reserve some 15 and 17; four entries of a thread beside each other
// instead of T apart 9.0 and 9.2).
template <int T> struct FewLds {
    static constexpr int FEW = 4 * T, SLOTS = 2 * FEW;
    int pos[FEW], entry[FEW], start[FEW + 1];    // of a sequence: its position (-1: denied), first entry, and that one's place
    union {                                      // (one after the other)
        int owner[FEW];                          // the sequence that starts at an entry, from 1 on
        struct { int page[SLOTS], uses[SLOTS], last[SLOTS]; };
        struct { int rank[FEW], fresh[FEW]; };   // an entry's needs up to it; free pages
    };
    int sums[2 * T / 64];
};

template <int T>
__global__ __launch_bounds__(T) void k_reserve_few(Pages pg, Rows s, FastDiv by_page, int most, int32_t *copies, int32_t *n_copies,
                                                    int32_t *pos_out) {
    __shared__ FewLds<T> l;
    constexpr int SLOTS = l.SLOTS, R = 4;
    const int t = threadIdx.x;
    const bool single = !s.row_start;
    int turn = 0, all;
    const Counts first(pg, 16 * t);              // on its way
    if (!single)
        for (int i = t; i < most; i += T) l.owner[i] = 0;
    int n[R], entries = 0;
#pragma unroll
    for (int j = 0; j < R; j++) {
        const int b = j * T + t;
        n[j] = 0;
        if (j * T >= s.n_seq) continue;
        if (b < s.n_seq) {
            const Seq q = seq_at(s, b);
            l.pos[b] = q.pos;
            if (q.r1 > q.r0 && (uint32_t)q.pos < s.cap) {
                const uint32_t last = min((uint32_t)q.pos + (uint32_t)(q.r1 - q.r0 - 1), s.cap - 1);
                l.entry[b] = (int)by_page(q.pos);
                n[j] = min((int)by_page(last) - l.entry[b] + 1, (int)l.FEW);
            }
        }
        if (single) continue;
        const int at = entries + block_scan<T>(n[j], l.sums, turn, all) - n[j];
        if (b < s.n_seq) l.start[b] = min(at, most);
        if (n[j] && at < most) l.owner[at] = b + 1;
        entries += all;
    }
    entries = single ? s.n_seq : min(entries, most);
    if (t == 0) l.start[s.n_seq] = entries;
    if (!single) __syncthreads();
    int seq[R], page[R], e[R], f[R], owner = 0;
#pragma unroll
    for (int j = 0; j < R; j++) {
        const int c = j * T + t;
        page[j] = -1;
        f[j] = 0;
        if (j * T >= entries) continue;
        if (single) {
            seq[j] = c;
            if (!n[j]) continue;
            e[j] = l.entry[c];                   // (its own)
        } else {
            int top = c < entries ? l.owner[c] : 0;
            for (int i = 1; i < 64; i *= 2) {
                const int o = __shfl_up(top, i, 64);
                if ((t & 63) >= i) top = max(top, o);
            }
            int *w = l.sums + (turn ^= 1) * (T / 64);
            if ((t & 63) == 63) w[t >> 6] = top;
            __syncthreads();
            int before = owner;                  // of the waves before this one
            for (int i = 0; i < T / 64; i++) {
                before = max(before, i < (t >> 6) ? w[i] : 0);
                owner = max(owner, w[i]);
            }
            if (c >= entries) continue;
            seq[j] = max(top, before) - 1;
            e[j] = l.entry[seq[j]] + c - l.start[seq[j]];
        }
        f[j] = NEED;
        page[j] = pg.row(seq[j])[e[j]];
    }
    int held[R];                                 // counts of the entries' pages
#pragma unroll
    for (int j = 0; j < R; j++) held[j] = f[j] && pg.there(page[j]) ? pg.refs[page[j]] : 0;
    bool some = false;
#pragma unroll
    for (int j = 0; j < R; j++) {
        if (f[j] && pg.there(page[j])) f[j] = held[j] > 1 ? SHARED : 0;
        some |= f[j] == SHARED;
    }
    if (__syncthreads_or(some)) {
        for (int i = t; i < SLOTS; i += T) {
            l.page[i] = -1;
            l.uses[i] = 0;
            l.last[i] = -1;
        }
        __syncthreads();
        auto slot = [&](int page) {              // its place; every probe ends, as half of them are free
            int i = (int)((uint32_t)page * 2654435761u >> 16) % SLOTS;
            for (;; i = (i + 1) % SLOTS) {
                const int there = atomicCAS(&l.page[i], -1, page);
                if (there == -1 || there == page) return i;
            }
        };
        int at[R];
#pragma unroll
        for (int j = 0; j < R; j++)
            if (f[j] & SHARED) {
                at[j] = slot(page[j]);
                atomicAdd(&l.uses[at[j]], 1);
                atomicMax(&l.last[at[j]], j * T + t);
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < R; j++)
            if (f[j] & SHARED) f[j] |= l.uses[at[j]] == held[j] && l.last[at[j]] == j * T + t ? KEEP : NEED;
        __syncthreads();                         // (the ranks take their place)
    }
    int rank[R], needs = 0;
#pragma unroll
    for (int j = 0; j < R; j++) {
        if (j * T >= entries) continue;
        rank[j] = needs + block_scan<T>(f[j] & NEED, l.sums, turn, all);
        if (!single && j * T + t < entries) l.rank[j * T + t] = rank[j];
        needs += all;
    }
    const int found = take_free<T>(pg, first, needs, l.fresh, l.sums, turn);
    __syncthreads();
    // (Nobody reads a count or an entry of the table any more.)
    int copied = 0;
#pragma unroll
    for (int j = 0; j < R; j++) {
        if (j * T >= entries) continue;
        int fresh = -1;
        if (f[j] & (NEED | KEEP)) {
            const int b = seq[j], p = l.pos[b];  // (another thread may set it to -1: then this entry is denied too)
            if ((single ? rank[j] : l.rank[l.start[b + 1] - 1]) > found) {
                l.pos[b] = -1;
            } else if (f[j] & NEED) {
                const int now = l.fresh[rank[j] - 1];
                pg.row(b)[e[j]] = now;
                pg.refs[now] = 1;
                count(pg, page[j], -1);
                if (f[j] & SHARED && (int64_t)e[j] * pg.P < p) fresh = now;
            }
        }
        const int at = copied + block_scan<T>(fresh >= 0, l.sums, turn, all) - 1;
        if (fresh >= 0) {
            copies[2 * at] = page[j];
            copies[2 * at + 1] = fresh;
        }
        copied += all;
    }
#pragma unroll
    for (int j = 0; j < R; j++)
        if (j * T + t < s.n_seq) pos_out[j * T + t] = l.pos[j * T + t];
    if (t == 0) *n_copies = copied;
}

// ---------------------------------------------------------------- compact

constexpr int CT = 256, CP = 4 * CT;             // threads and pages of a workgroup

__device__ __forceinline__ int workgroup_sum(int v, int *red) {
    const int sum = __builtin_amdgcn_readlane(wave_scan(v), 63);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// Pages in use of each CP.
__global__ __launch_bounds__(CT) void k_used(Pages pg, int32_t *counts) {
    __shared__ int red[CT / 64];
    const uint32_t p = blockIdx.x * (uint32_t)CP + threadIdx.x;
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) n += p + j * CT < pg.n_pages && pg.refs[p + j * CT] > 0;
    n = workgroup_sum(n, red);
    if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// With n pages in use: the k-th lowest free page goes into low[k] if it lies below n, the k-th
// highest one in use into high[k] if it does not, which are as many, k into to[page]; to[page] of
// a free one is -1.  Without `counts` every workgroup counts all pages itself.
__global__ __launch_bounds__(CT) void k_rank(Pages pg, const int32_t *counts, int32_t *low, int32_t *high, int32_t *to, int32_t *n_moves) {
    __shared__ int red[CT / 64];
    const uint32_t first = blockIdx.x * (uint32_t)CP;
    // Which of pages p .. p + 3 are in use.
    auto used_at = [&](uint32_t p, int (&used)[4]) {
        typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));
        i32x4 r = {0, 0, 0, 0};
        if (p + 4 <= pg.n_pages) r = *(const i32x4 *)(pg.refs + p);
        else
            for (int j = 0; j < 4; j++) r[j] = p + j < pg.n_pages ? pg.refs[p + j] : 0;
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) n += used[j] = r[j] > 0;
        return n;
    };
    int used[4], before = 0, n = 0;
    const int own = used_at(first + 4 * threadIdx.x, used);
    if (counts) {
        for (int i = threadIdx.x; i < (int)gridDim.x; i += CT) {
            n += counts[i];
            before += i < (int)blockIdx.x ? counts[i] : 0;
        }
    } else {
#pragma unroll 8
        for (uint32_t c = 0; c < gridDim.x; c++) {
            int any[4];
            const int u = used_at(c * CP + 4 * threadIdx.x, any);
            n += u;
            before += c < blockIdx.x ? u : 0;
        }
    }
    n = workgroup_sum(n, red);
    before = workgroup_sum(before, red);
    const int upto = wave_scan(own);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = upto;
    __syncthreads();
    int at = before + upto - own;                // pages in use before this thread's
    for (int i = 0; i < (int)(threadIdx.x >> 6); i++) at += red[i];
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        n_moves[1] = n;
        if (n == 0) n_moves[0] = 0;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t p = first + 4 * threadIdx.x + j;
        if (p >= pg.n_pages) break;
        if (p < (uint32_t)n) {
            if (!used[j]) low[p - at] = (int32_t)p;
            if (p == (uint32_t)n - 1) n_moves[0] = (int)p - at + !used[j];
        } else {
            if (used[j]) high[n - 1 - at] = (int32_t)p;
            to[p] = used[j] ? n - 1 - at : -1;
        }
        at += used[j];
    }
}

// The moves, their counts of references, and the table's entries that name moved pages.
__global__ __launch_bounds__(CT) void k_move(Pages pg, const int32_t *low, const int32_t *high, const int32_t *to, const int32_t *n_moves,
                                             int32_t *moves) {
    const int64_t i0 = blockIdx.x * (int64_t)CT + threadIdx.x, step = (int64_t)gridDim.x * CT;
    const int64_t entries = (int64_t)pg.n_seq * pg.max_pages;
    int page = i0 < entries ? pg.table[i0] : -1;     // (on its way beside the counts)
    const int n = n_moves[1], k = n_moves[0];
    for (int64_t i = i0; i < k; i += step) {
        const int src = high[i], dst = low[i];
        moves[2 * i] = src;
        moves[2 * i + 1] = dst;
        pg.refs[dst] = pg.refs[src];
        pg.refs[src] = 0;
    }
    if (k == 0) return;
    for (int64_t i = i0; i < entries; i += step) {
        if (i != i0) page = pg.table[i];
        if (page < n || !pg.there(page)) continue;
        const int at = to[page];
        if (at >= 0) pg.table[i] = low[at];
    }
}

// All of it in one workgroup, for 4 T pages at most: four pages a thread, what they become in LDS.
template <int T>
__global__ __launch_bounds__(T) void k_compact_few(Pages pg, int entries, int32_t *moves, int32_t *n_moves) {
    __shared__ int low[4 * T], to[4 * T], sums[2 * T / 64];
    const int t = threadIdx.x;
    int turn = 0, n, refs[4], own = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) own += (refs[j] = 4u * t + j < pg.n_pages ? pg.refs[4 * t + j] : 0) > 0;
    int page = t < entries ? pg.table[t] : -1;   // (on its way beside the counts)
    const int before = block_scan<T>(own, sums, turn, n) - own;
    int at = before;                             // pages in use before
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int p = 4 * t + j;
        if (p < n && refs[j] <= 0) low[p - at] = p;
        if (p == n - 1) n_moves[0] = p - at + (refs[j] <= 0);
        at += refs[j] > 0;
    }
    if (t == 0) {
        n_moves[1] = n;
        if (n == 0) n_moves[0] = 0;
    }
    __syncthreads();                             // (all counts are read)
    at = before;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int p = 4 * t + j;
        if (p < n) {
            at += refs[j] > 0;
            continue;
        }
        to[p] = -1;
        if (refs[j] <= 0) continue;
        const int k = n - 1 - at++, dst = low[k];
        to[p] = dst;
        moves[2 * k] = p;
        moves[2 * k + 1] = dst;
        pg.refs[dst] = refs[j];
        pg.refs[p] = 0;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = t; i < entries; i += T) {
        if (i != t) page = pg.table[i];
        if (page >= n && pg.there(page) && to[page] >= 0) pg.table[i] = to[page];
    }
}

// ---------------------------------------------------------------- copy

constexpr int LAYERS = 64;                       // of a launch
struct Layer {
    void *k, *v;
    uint8_t *kx, *vx;
    uint32_t bytes, exps;                        // of a page of a plane, and its exponents
};
struct Layers {
    Layer l[LAYERS];
};

// Workgroup (pairs from x on, plane y of the layers, slice z): SLICE bytes of a page, four
// 16-byte loads a thread in flight.  Bytes bound it: some 950 pages of 32 KiB in 16 planes, 1 GB
// read and written, 180 us, 5.6 TB/s.  What is written goes past the caches (copies of a step in 16
// layers 17.2 -> 16.4 us, large ones 207 -> 202), and so does what is read where it is more than
// they hold for long (-> 196; few pages, which later calls copy again, 16.4 -> 20.5): LARGE.
constexpr uint32_t SLICE = 16384;
constexpr uint64_t LARGE = 96u << 20;            // bytes: 80 MB copied 38 us so, 42 past the caches, 120 MB 60 and 58
__global__ __launch_bounds__(256) void k_copy(Layers layers, uint32_t n_pages, const int32_t *pairs, const int32_t *n_pairs, int most) {
    const Layer l = layers.l[blockIdx.y >> 1];
    const bool is_k = !(blockIdx.y & 1);
    char *plane = (char *)(is_k ? l.k : l.v);
    uint8_t *exps = is_k ? l.kx : l.vx;
    int i = blockIdx.x, src = pairs[2 * i], dst = pairs[2 * i + 1];    // (on their way beside the count)
    const int n = n_pairs ? min(max(*n_pairs, 0), most) : most;
    const bool large = (uint64_t)n * l.bytes * gridDim.y > LARGE;
    for (; i < n; i += gridDim.x) {
        if (i != (int)blockIdx.x) {
            src = pairs[2 * i];
            dst = pairs[2 * i + 1];
        }
        if ((uint32_t)src >= n_pages || (uint32_t)dst >= n_pages || src == dst) continue;
        const char *x = plane + (uint64_t)src * l.bytes;
        char *y = plane + (uint64_t)dst * l.bytes;
        auto slices = [&](auto past) {
            for (uint64_t at = (uint64_t)blockIdx.z * SLICE; at < l.bytes; at += (uint64_t)gridDim.z * SLICE) {
                u32x4 r[SLICE / 4096];
#pragma unroll
                for (uint32_t j = 0; j < SLICE / 4096; j++) {
                    const uint64_t a = at + j * 4096 + threadIdx.x * 16;
                    if (a >= l.bytes) continue;
                    if constexpr (past) r[j] = __builtin_nontemporal_load((const u32x4 *)(x + a));
                    else r[j] = *(const u32x4 *)(x + a);
                }
#pragma unroll
                for (uint32_t j = 0; j < SLICE / 4096; j++) {
                    const uint64_t a = at + j * 4096 + threadIdx.x * 16;
                    if (a < l.bytes) __builtin_nontemporal_store(r[j], (u32x4 *)(y + a));
                }
            }
        };
        if (large) slices(std::true_type());
        else slices(std::false_type());
        if (blockIdx.z == 0)
            for (uint32_t j = threadIdx.x; j < l.exps; j += 256)
                exps[(uint64_t)dst * l.exps + j] = exps[(uint64_t)src * l.exps + j];
    }
}

// ---------------------------------------------------------------- checks

int check_pages(gd_ctx *ctx, const char *fn, const gd_kv_pages *pg) {
    GD_REQUIRE(ctx, pg, "%s: null pages", fn);
    GD_REQUIRE(ctx, pg->n_pages > 0 && pg->n_pages < (1LL << 31) - 2 * CP, "%s: %lld pages", fn, (long long)pg->n_pages);
    GD_REQUIRE(ctx, pg->n_seq >= 0 && pg->n_seq < MAX_WGS && pg->max_pages > 0, "%s: %d sequences of %d pages", fn, pg->n_seq,
               pg->max_pages);
    GD_REQUIRE(ctx, pg->page_size > 0 && pg->page_size <= (1 << 24), "%s: page size %d", fn, pg->page_size);
    GD_REQUIRE(ctx, pg->refs && (pg->table || !pg->n_seq), "%s: null refs or table", fn);
    GD_REQUIRE(ctx, ((uintptr_t)pg->refs | (uintptr_t)pg->table | (uintptr_t)pg->keep) % 4 == 0,
               "%s: refs, table and keep must be 4-byte aligned", fn);
    return GD_OK;
}
Pages pages_of(const gd_kv_pages *pg) {
    return Pages{pg->refs, pg->table, (uint32_t)pg->n_pages, pg->n_seq, pg->max_pages, pg->page_size};
}

// Orders of a call: workgroups walk them all, and are counted as a launch's.
constexpr int MAX_ORDERS = 1 << 16;
int check_orders(gd_ctx *ctx, const char *fn, const gd_kv_pages *pg, int n, const void *a, const void *b, const void *c) {
    GD_REQUIRE(ctx, n >= 0 && n <= MAX_ORDERS, "%s: %d orders (%d at most)", fn, n, MAX_ORDERS);
    GD_REQUIRE(ctx, n == 0 || (a && b), "%s: null orders", fn);
    GD_REQUIRE(ctx, ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % 4 == 0, "%s: orders must be 4-byte aligned", fn);
    const int64_t chunks = ((int64_t)pg->max_pages + EW - 1) / EW;
    GD_REQUIRE(ctx, chunks < 65536 && n * chunks < MAX_WGS, "%s: %d orders over %d pages each", fn, n, pg->max_pages);
    return GD_OK;
}
dim3 order_grid(const gd_kv_pages *pg, int n) {
    return dim3(n, std::min<unsigned>(gd_blocks(pg->max_pages, EW), std::max(1, MOST_WGS / n)));
}

}  // namespace

// ---------------------------------------------------------------- C ABI
// Arguments are checked before the context is looked at (as the other entries of the cache).

extern "C" int gd_kv_fork(gd_ctx *ctx, const gd_kv_pages *pg, const int32_t *src, const int32_t *dst, const int32_t *len, int n) {
    const char *fn = "gd_kv_fork";
    int rc;
    if ((rc = check_pages(ctx, fn, pg)) || (rc = check_orders(ctx, fn, pg, n, src, dst, len))) return rc;
    GD_REQUIRE(ctx, n == 0 || len, "%s: null orders", fn);
    GD_CHECK_CTX(ctx);
    if (!n || !pg->n_seq) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    hipLaunchKernelGGL(k_fork, order_grid(pg, n), dim3(256), 0, ctx->stream, pages_of(pg), src, dst, len, n);
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}

extern "C" int gd_kv_release(gd_ctx *ctx, const gd_kv_pages *pg, const int32_t *seq, const int32_t *from, const int32_t *to, int n) {
    const char *fn = "gd_kv_release";
    int rc;
    if ((rc = check_pages(ctx, fn, pg)) || (rc = check_orders(ctx, fn, pg, n, seq, to, from))) return rc;
    GD_CHECK_CTX(ctx);
    if (!n || !pg->n_seq) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    hipLaunchKernelGGL(k_release, order_grid(pg, n), dim3(256), 0, ctx->stream, pages_of(pg), pg->keep, seq, from, to);
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}

extern "C" int gd_kv_reserve(gd_ctx *ctx, const gd_kv_pages *pg, const gd_seqs *s, int32_t *copies, int32_t *n_copies, int32_t *pos_out) {
    const char *fn = "gd_kv_reserve";
    int rc;
    if ((rc = check_pages(ctx, fn, pg)) || (rc = check_seqs(ctx, fn, s))) return rc;
    GD_REQUIRE(ctx, s->n_seq == pg->n_seq && s->max_pages == pg->max_pages && (s->page_table == pg->table || !s->n_rows),
               "%s: the sequences' table is not the pages' (%d x %d and %d x %d)", fn, s->n_seq, s->max_pages, pg->n_seq, pg->max_pages);
    GD_REQUIRE(ctx, n_copies && (!s->n_seq || (copies && pos_out)), "%s: null copies or positions", fn);
    GD_REQUIRE(ctx, ((uintptr_t)copies | (uintptr_t)n_copies | (uintptr_t)pos_out) % 4 == 0, "%s: outputs must be 4-byte aligned", fn);
    GD_REQUIRE(ctx, !s->n_seq || s->pos, "%s: null positions or page table", fn);
    GD_CHECK_CTX(ctx);
    GD_HIP(ctx, hipSetDevice(ctx->device));
    const int64_t cap = std::min<int64_t>((int64_t)pg->max_pages * pg->page_size, 0x7fffffff);
    const Rows rows{s->row_start, s->pos, nullptr, s->page_table, (int)s->n_rows, s->n_seq, s->max_pages, (uint32_t)cap};
    // Entries of the rows: a page for each page_size of them, and two ends a sequence; one of a single row.
    Work wk;
    wk.most = (int)(s->row_start ? s->n_rows / pg->page_size + 2 * std::min<int64_t>(s->n_seq, s->n_rows) : s->n_rows);
    // us of 256 / 512 / 1024 threads: 200 tokens 6.9 / 7.4 / 9, 400 7.9 / 7.6 / 8.5, 1000 14.6 / 10.0 / 9.7; 200
    // prompts of up to 600 entries 9.2 / 8.6 / 10.1.
    const int widest = std::max(s->n_seq, wk.most), few = widest <= 512 ? 256 : widest <= 2048 ? 512 : 1024;
    if (widest <= 4 * few) {
        auto kernel = few == 256 ? k_reserve_few<256> : few == 512 ? k_reserve_few<512> : k_reserve_few<1024>;
        hipLaunchKernelGGL(kernel, dim3(1), dim3(few), 0, ctx->stream, pages_of(pg), rows, FastDiv((uint32_t)pg->page_size), wk.most, copies,
                           n_copies, pos_out);
        GD_LAUNCHED(ctx, fn);
        return GD_OK;
    }
    void *ws;
    if ((rc = gd_ctx_workspace(ctx, Work::ints(s->n_seq, pg->n_pages, wk.most) * 4, &ws))) return rc;
    int32_t *at = (int32_t *)ws;
    auto take = [&](int64_t n) { int32_t *p = at; at += n; return p; };
    wk.start = take(s->n_seq + 1);
    wk.uses = take(pg->n_pages);
    wk.last = take(pg->n_pages);
    for (int32_t **p : {&wk.seq, &wk.entry, &wk.page, &wk.flags, &wk.rank, &wk.fresh}) *p = take(wk.most);
    hipLaunchKernelGGL(k_reserve, dim3(1), dim3(RT), 0, ctx->stream, pages_of(pg), rows, FastDiv((uint32_t)pg->page_size), wk, copies,
                       n_copies, pos_out);
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}

extern "C" int gd_kv_compact(gd_ctx *ctx, const gd_kv_pages *pg, int32_t *moves, int32_t *n_moves) {
    const char *fn = "gd_kv_compact";
    int rc;
    if ((rc = check_pages(ctx, fn, pg))) return rc;
    GD_REQUIRE(ctx, moves && n_moves, "%s: null moves", fn);
    GD_REQUIRE(ctx, ((uintptr_t)moves | (uintptr_t)n_moves) % 4 == 0, "%s: moves must be 4-byte aligned", fn);
    GD_CHECK_CTX(ctx);
    GD_HIP(ctx, hipSetDevice(ctx->device));
    // One launch or two, us by pages and entries of the table: 100, 150 6.1 / 8.2; 1000, 1000 6.1 / 8.4 (256
    // threads); 2000, 4000 7.2 / 8.8; 4000, 6000 8.2 / 9.1; 4000, 24000 13.6 / 8.8 (1024).
    const int64_t all = (int64_t)pg->n_seq * pg->max_pages;
    if (pg->n_pages <= 4 * 1024 && all <= 6 * 1024) {
        const bool least = pg->n_pages <= 4 * 256 && all <= 8 * 256;
        auto kernel = least ? k_compact_few<256> : k_compact_few<1024>;
        hipLaunchKernelGGL(kernel, dim3(1), dim3(least ? 256 : 1024), 0, ctx->stream, pages_of(pg), (int)all, moves, n_moves);
        GD_LAUNCHED(ctx, fn);
        return GD_OK;
    }
    const int chunks = (int)gd_blocks(pg->n_pages, CP);
    const bool alone = pg->n_pages <= 16 * CP;   // pages that each workgroup of k_rank counts itself (a launch less, 3 us)
    void *ws;
    if ((rc = gd_ctx_workspace(ctx, ((size_t)chunks + 3 * pg->n_pages) * 4, &ws))) return rc;
    int32_t *counts = (int32_t *)ws, *low = counts + chunks, *high = low + pg->n_pages, *to = high + pg->n_pages;
    const Pages p = pages_of(pg);
    if (!alone) {
        hipLaunchKernelGGL(k_used, dim3(chunks), dim3(CT), 0, ctx->stream, p, counts);
        GD_LAUNCHED(ctx, fn);
    }
    hipLaunchKernelGGL(k_rank, dim3(chunks), dim3(CT), 0, ctx->stream, p, alone ? nullptr : counts, low, high, to, n_moves);
    GD_LAUNCHED(ctx, fn);
    const int64_t entries = std::max<int64_t>((int64_t)pg->n_seq * pg->max_pages, pg->n_pages);
    hipLaunchKernelGGL(k_move, dim3(std::min<int64_t>((entries + CT - 1) / CT, 2048)), dim3(CT), 0, ctx->stream, p, low, high, to, n_moves,
                       moves);
    GD_LAUNCHED(ctx, fn);
    return GD_OK;
}

extern "C" int gd_kv_copy_pages(gd_ctx *ctx, const gd_kv *kv, int n_kv, const int32_t *pairs, const int32_t *n_pairs, int64_t max_pairs) {
    const char *fn = "gd_kv_copy_pages";
    int rc;
    GD_REQUIRE(ctx, n_kv >= 0 && (kv || !n_kv), "%s: %d caches", fn, n_kv);
    for (int i = 0; i < n_kv; i++) {
        if ((rc = check_kv(ctx, fn, kv + i, true))) return rc;
        GD_REQUIRE(ctx, kv[i].n_pages == kv[0].n_pages, "%s: caches of %lld and %lld pages", fn, (long long)kv[0].n_pages,
                   (long long)kv[i].n_pages);
        const int64_t bytes = (int64_t)kv[i].page_size * kv[i].n_head_kv * kv[i].head_dim * (kv[i].dtype == GD_F16 ? 2 : 1);
        GD_REQUIRE(ctx, bytes < (1LL << 32), "%s: pages of %lld bytes", fn, (long long)bytes);
    }
    GD_REQUIRE(ctx, max_pairs >= 0 && max_pairs < (1LL << 30), "%s: %lld pairs", fn, (long long)max_pairs);
    GD_REQUIRE(ctx, max_pairs == 0 || pairs, "%s: null pairs", fn);
    GD_REQUIRE(ctx, ((uintptr_t)pairs | (uintptr_t)n_pairs) % 4 == 0, "%s: pairs must be 4-byte aligned", fn);
    GD_CHECK_CTX(ctx);
    if (!max_pairs) return GD_OK;
    GD_HIP(ctx, hipSetDevice(ctx->device));
    for (int i0 = 0; i0 < n_kv; i0 += LAYERS) {
        const int n = std::min(LAYERS, n_kv - i0);
        Layers layers = {};
        uint32_t widest = 0;
        for (int i = 0; i < n; i++) {
            const gd_kv &c = kv[i0 + i];
            const bool i8 = c.dtype == GD_I8;
            const uint32_t rows = (uint32_t)c.page_size * c.n_head_kv;
            layers.l[i] = Layer{c.k, c.v, c.k_exp, c.v_exp, rows * c.head_dim * (i8 ? 1 : 2), i8 ? rows / BLK : 0};
            widest = std::max(widest, layers.l[i].bytes);
        }
        const int64_t slices = std::min<int64_t>(((int64_t)widest + SLICE - 1) / SLICE, 1024);
        const int64_t x = std::min<int64_t>(max_pairs, std::max<int64_t>(1, 16384 / (2 * n * slices)));
        hipLaunchKernelGGL(k_copy, dim3((unsigned)x, 2 * n, (unsigned)slices), dim3(256), 0, ctx->stream, layers, (uint32_t)kv[0].n_pages,
                           pairs, n_pairs, (int)max_pairs);
        GD_LAUNCHED(ctx, fn);
    }
    return GD_OK;
}
