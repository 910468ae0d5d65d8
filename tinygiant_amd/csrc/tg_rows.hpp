/*
 * tg_rows.hpp -- device code that the attention kernels of packed rows share
 * (tg_prompt.hip: dense caches; tg_paged.hip: 8-bit pages): the sequences of a
 * call, its tiles and spans, the operands in registers and LDS, and the merge
 * of two groups of waves.
 */
#ifndef TG_ROWS_HPP
#define TG_ROWS_HPP
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "tg_device.hpp"
#include "tg_prompt.h"
#include "tg_xchg.hpp"

namespace tg {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   /* rows need only 4-byte alignment */
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

/* Sequence s as the kernels use it, from device integers that no host check
 * has seen: everything is brought into range, and a sequence whose slot or
 * length does not fit the cache has no rows (its rows are left as they were). */
struct Seq {
    int r0, n;        /* its packed rows */
    int past;         /* cached before them */
    int slot;
};
__device__ inline Seq seq_at(const PackedSeqs &p, int s) {
    Seq q;
    q.r0 = min(max(p.cu[s], 0), p.rows);
    q.n = min(max(p.cu[s + 1], q.r0), p.rows) - q.r0;
    q.past = p.len ? p.len[s] : 0;
    q.slot = p.slot ? p.slot[s] : s;
    if (q.slot < 0 || q.slot >= p.n_slots || q.past < 0 || q.past > p.kv_max - q.n) q.n = 0;
    return q;
}
/* the last sequence that starts at or before row r (-1: none) */
__device__ inline int seq_of(const PackedSeqs &p, int r) {
    int lo = -1, hi = p.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

/* A run of at most 64 sequences, among which the last is that starts at or
 * before `key`; 64 places of those before are asked at a time.  A start is a
 * row, or with MTILE the place of the sequence's first tile (find_tile). */
struct Run {
    int at, count;   /* 0: none */
};
template <int MTILE>
__device__ inline int start_of(int r0, int s, int ratio) {
    return MTILE ? (int)((unsigned)(r0 * ratio) / (unsigned)(MTILE ? MTILE : 1)) + s : r0;
}
template <int MTILE>
__device__ inline Run wave_narrow(const PackedSeqs &p, int ratio, int key) {
    const int lane = threadIdx.x & 63;
    int at = 0, count = p.n;
    while (count > 64) {
        const int step = (count + 63) / 64, s = at + min(lane * step, count - 1);
        const uint64_t m = __ballot(lane * step < count && start_of<MTILE>(min(max(p.cu[s], 0), p.rows), s, ratio) <= key);
        if (!m) return Run{0, 0};
        const int k = (63 - __builtin_clzll(m)) * step;
        at += k, count = min(step, count - k);
    }
    return Run{at, count};
}

/* lane `at`'s sequence, in the whole wave */
__device__ inline Seq lane_seq(const Seq &q, int at) {
    return Seq{__builtin_amdgcn_readlane(q.r0, at), __builtin_amdgcn_readlane(q.n, at), __builtin_amdgcn_readlane(q.past, at),
               __builtin_amdgcn_readlane(q.slot, at)};
}

/* The sequence of row r, the same r in the whole wave; all that is read of the
 * last 64 in one batch.  False: none. */
__device__ inline bool wave_seq_of(const PackedSeqs &p, int r, Seq &q, int &i) {
    const int lane = threadIdx.x & 63;
    const Run run = wave_narrow<0>(p, 0, r);
    Seq mine = {0, 0, 0, 0};
    if (lane < run.count) mine = seq_at(p, run.at + lane);
    const uint64_t m = __ballot(lane < run.count && mine.r0 <= r);
    if (!m) return false;
    q = lane_seq(mine, 63 - __builtin_clzll(m));   /* the last that starts at or before r */
    i = r - q.r0;
    return i >= 0 && i < q.n;
}

}  // namespace

/* ---- attention ----
 *
 * Row i of a sequence and query head kh * ratio + j, of KV head kh, is "m-row"
 * i * ratio + j: all query heads of a KV head read the same K and V, so they
 * fill the matrix units' columns together, and any ratio and row count packs.
 *
 * A region is a run of cached positions with one base: a sequence's slot, or
 * the shared prefix.  A workgroup takes MT m-rows of one KV head and a span of
 * a region.  Where one workgroup covers all that its rows see, it writes the
 * output; else it writes a record (reference exponent m, sum l, unnormalised
 * o[head_dim]) a row and k_rows_combine merges the records.  Exponents are in
 * base 2: weight 2^(z - m), z = score * log2 e. */
struct RowsPlan {
    int items;              /* upper bound of the own-slot tiles' spans, per KV head */
    int cap;                /* spans a tile has at most */
    int target;             /* spans that the positions of all tiles are cut into, about */
    int unit, pre_unit;     /* a span is a multiple of this; the prefix's */
    int pre_tiles, pre_ns;  /* tiles of the prefix, spans of each */
    bool search;            /* the sequence of a tile is searched for (find_tile), not counted to (find_span) */
    int nrec;               /* room for a row's records: pre_ns + cap; 0: written directly */
    float *ml, *o;          /* [n_rows * n_heads][nrec][4]: m, l, and in the first own span's the count of those;
                               [..][nrec][head_dim] */
};
/* joins the records that the call's workgroups wrote (tg_prompt.hip) */
void launch_rows_combine(const PromptArgs &a, const RowsPlan &p, hipStream_t st);

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KT = 64;    /* positions of a tile */

/* what a workgroup works on, uniform over it */
struct Work {
    int kh, rec;
    int count;       /* own slots' first span: how many spans the tile has; else 0 */
    bool prefix;
    Seq sq;          /* own: the sequence; prefix: all rows of the call as one */
    int m0;          /* the tile's first m-row */
    int i0, j0;      /* its row of the sequence and its query head of the group */
    uint32_t inv;    /* x / ratio = x inv >> 16 for x < 1024 */
    int lo, hi;      /* positions of the region */
    /* row of the sequence and query head of the group of m-row m0 + at */
    __device__ inline void row(int at, int ratio, int &i, int &j) const {
        const int x = j0 + at, d = (int)(((uint32_t)x * inv) >> 16);
        i = i0 + d, j = x - d * ratio;
    }
};

__device__ inline void set_rows(Work &w, int ratio) {
    w.i0 = w.m0 / ratio, w.j0 = w.m0 - w.i0 * ratio;
    w.inv = (65536u + (uint32_t)ratio - 1u) / (uint32_t)ratio;   /* off by less than ratio <= 64: exact below 1024 */
}

__device__ inline int div_up(int a, int b) { return (int)(((unsigned)a + (unsigned)b - 1u) / (unsigned)b); }

/* inclusive sum over the wave's lanes */
__device__ inline int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   /* row_shr:1, 2, 4, 8 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   /* row_bcast:15, :31 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

/* the first position that the rows of w's tile see, and the one behind the last */
__device__ inline int tile_lo(const PromptArgs &a, const Work &w) {
    return a.window > 0 ? max(0, w.sq.past + w.i0 + 1 - a.window) : 0;
}
template <int MTILE>
__device__ inline int tile_hi(const Work &w, int ratio) {
    int i1, j1;
    w.row(MTILE - 1, ratio, i1, j1);
    return w.sq.past + min(w.sq.n - 1, i1) + 1;
}

/* which sequences a part of a call takes: all.  Another type gives a sequence
 * that its part leaves to others no rows. */
struct Everyone {};

/* Tile b of the sequences' tiles of MTILE m-rows, late rows first (they see
 * the most positions).  Sequence s has its tiles from place
 * cu[s] ratio / MTILE + s on, where there is room for them whatever the
 * sequences before it left over: no sum over those is needed. */
template <int MTILE, class Keep = Everyone>
__device__ inline bool find_tile(const PromptArgs &a, const RowsPlan &p, int ratio, int b, Work &w, Keep keep = {}) {
    const PackedSeqs &c = a.s;
    const int lane = threadIdx.x & 63;
    const Run run = wave_narrow<MTILE>(c, ratio, b);
    Seq q = {0, 0, 0, 0};
    if (lane < run.count) q = seq_at(c, run.at + lane);
    if constexpr (!std::is_same_v<Keep, Everyone>) keep(q);
    const uint64_t m = __ballot(lane < run.count && start_of<MTILE>(q.r0, run.at + lane, ratio) <= b);
    if (!m) return false;
    const int at = 63 - __builtin_clzll(m);
    w.sq = lane_seq(q, at);
    const int place = b - start_of<MTILE>(w.sq.r0, run.at + at, ratio), n = div_up(w.sq.n * ratio, MTILE);
    if (place >= n) return false;
    w.m0 = (n - 1 - place) * MTILE;
    set_rows(w, ratio);
    w.rec = p.pre_ns, w.count = 1;
    w.lo = tile_lo(a, w), w.hi = tile_hi<MTILE>(w, ratio);   /* stored last, as in the others: the compiler merges the ends */
    return true;
}

/* Item b of the sequences' spans: tiles as above, in order, each cut into
 * spans of one length for all sequences, so that long and short ones finish
 * together: that length is what cuts the positions of all tiles into about
 * p.target spans (a sequence's tiles count as its longest); with p.cap 1, one
 * span a tile.  A wave counts 64 sequences at a time; sums of positions are
 * floats, the same in every workgroup. */
template <int MTILE, class Keep = Everyone>
__device__ inline bool find_span(const PromptArgs &a, const RowsPlan &p, int ratio, int b, Work &w, Keep keep = {}) {
    const PackedSeqs &c = a.s;
    const int lane = threadIdx.x & 63;
    Seq q = {0, 0, 0, 0};
    auto load = [&](int s0) {
        q.n = 0;
        if (s0 + lane < c.n) q = seq_at(c, s0 + lane);
        if constexpr (!std::is_same_v<Keep, Everyone>) keep(q);
    };
    auto tiles = [&]() { return div_up(q.n * ratio, MTILE); };
    auto sees = [&]() {   /* positions of the sequence's tiles, at most */
        const int n = q.past + q.n;
        return a.window > 0 ? min(n, a.window + (MTILE - 1) / ratio + 1) : n;
    };
    int per = 0x40000000;
    load(0);
    if (p.cap > 1) {
        float sum = 0.f;
        for (int s0 = 0; s0 < c.n; s0 += 64) {
            if (s0) load(s0);
            sum += wave_sum((float)tiles() * (float)sees());
        }
        /* rounded up: a shorter span would make more of them than p.items has room for */
        per = div_up(max(1, (int)fminf(ceilf(sum / (float)p.target), 1e9f)), p.unit) * p.unit;
        if (c.n > 64) load(0);
    }
    for (int s0 = 0; s0 < c.n; s0 += 64) {
        if (s0) load(s0);
        const int nt = tiles(), end = wave_scan(nt * min(div_up(sees(), per), p.cap));
        const uint64_t past = __ballot(end > b);
        if (past) {
            const int at = __builtin_ctzll(past), n = __builtin_amdgcn_readlane(nt, at);
            w.sq = lane_seq(q, at);
            if (at) b -= __builtin_amdgcn_readlane(end, at - 1);
            const int split = b / n;
            w.m0 = (n - 1 - (b - split * n)) * MTILE;
            set_rows(w, ratio);
            const int lo = tile_lo(a, w), hi = tile_hi<MTILE>(w, ratio);
            int count = div_up(hi - lo, per);
            if (count > p.cap) {
                per = div_up(div_up(hi - lo, p.cap), p.unit) * p.unit;
                count = div_up(hi - lo, per);
            }
            if (split >= count) return false;
            w.rec = p.pre_ns + split;
            w.count = split ? 0 : count;
            w.lo = lo + split * per;
            w.hi = min(hi, w.lo + per);
            return true;
        }
        b -= __builtin_amdgcn_readlane(end, 63);
    }
    return false;
}

/* positions of the region that row i of the work's sequence sees: first ..
 * last; false: no row there */
__device__ inline bool row_sees(const PromptArgs &a, const Work &w, int i, int &first, int &last) {
    if (i >= w.sq.n) return false;
    first = 0;
    if (w.prefix) {
        last = a.pre_len - 1;
        if (a.window > 0) {
            const int r = w.sq.r0 + i, s = seq_of(a.s, r);
            if (s < 0) return false;
            const Seq q = seq_at(a.s, s);
            i = r - q.r0;
            if (i < 0 || i >= q.n) return false;
            first = max(0, a.pre_len + q.past + i + 1 - a.window);
        }
    } else {
        last = w.sq.past + i;
        if (a.window > 0) first = max(0, last + 1 - a.window);
    }
    return true;
}

/* This workgroup's work: the prefix's items, then the sequences'; KV heads
 * fastest, so that (8 XCDs, workgroups dealt in turn) those of one head meet
 * in as few L2 caches as possible.  False: none. */
template <int MTILE>
__device__ inline bool find_work(const PromptArgs &a, const RowsPlan &p, int ratio, Work &w) {
    int b = blockIdx.x;
    const int npre = p.pre_tiles * p.pre_ns * a.n_kv;
    w.prefix = b < npre;
    if (!w.prefix) b -= npre;
    const int item = b / a.n_kv;
    w.kh = b - item * a.n_kv;
    if (!w.prefix) return p.search ? find_tile<MTILE>(a, p, ratio, item, w) : find_span<MTILE>(a, p, ratio, item, w);
    const int split = item / p.pre_tiles;
    const int r0 = min(max(a.s.cu[0], 0), a.s.rows), r1 = min(max(a.s.cu[a.s.n], r0), a.s.rows);
    w.rec = split, w.count = 0;
    w.sq = Seq{r0, r1 - r0, 0, 0};
    w.m0 = (item - split * p.pre_tiles) * MTILE;
    if ((unsigned)w.m0 >= (unsigned)w.sq.n * (unsigned)ratio) return false;
    set_rows(w, ratio);
    int lo = 0;
    const int hi = a.pre_len;
    if (a.window > 0) {   /* the first position that any of the rows sees */
        lo = hi;
        for (int at = (int)(threadIdx.x & 63); at < MTILE; at += 64) {
            int f, l, i, j;
            w.row(at, ratio, i, j);
            if (row_sees(a, w, i, f, l)) lo = min(lo, f);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64));
        lo = min(__builtin_amdgcn_readfirstlane(lo), hi);
    }
    const int per = max(1, div_up(div_up(hi - lo, p.pre_ns), p.pre_unit)) * p.pre_unit;
    w.lo = min(hi, lo + split * per);
    w.hi = min(hi, w.lo + per);
    return true;
}

/* a record's statistics */
__device__ inline void write_ml(const RowsPlan &p, const Work &w, size_t rec, float m, float l) {
    *(f4 *)(p.ml + 4 * rec) = f4{m, l, __int_as_float(w.count), 0.f};
}

}  // namespace

/* ---- the f16 matrix units' operands ---- */
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

template <int HD>
__device__ inline constexpr int swz(int key) {
    return HD == 128 ? ((key & 3) << 2) | ((key >> 2) & 3) : (((key >> 1) & 1) << 2) | ((key >> 2) & 3);
}

__device__ inline h8 h8_of(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

/* LDS by pointer, so that constant offsets go into the instructions */
typedef const __attribute__((address_space(3))) uint8_t *Lds;
/* four values of one column of 16-bit values, rows in consecutive lanes' rows */
__device__ inline h4 lds_column(Lds at) {
    typedef __fp16 g4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) g4 *P;
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((P)at));
}
__device__ inline h8 lds_row(Lds at) { return *(const __attribute__((address_space(3))) h8 *)at; }
/* The larger of two, NaN if either is: one instruction, where fmaxf quiets
 * operands that may be signalling first (50 instead of 16 in a tile's
 * softmax).  A NaN makes its row not finite, and such rows are done again. */
__device__ inline float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
/* y = x f = hi + lo in two f16, each to nearest, for two values: one packed
 * conversion and a mixed-precision fma each.  The empty asm keeps the packed
 * pair as it is (the compiler would convert each value once more for lo); a
 * factor that it knows to be 1 would make the fma three instructions. */
__device__ inline void split2(float y0, float y1, float x0, float x1, float f, h2 &hi, h2 &lo) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    hi = __builtin_convertvector((f2{y0, y1}), h2);
    asm("" : "+v"(hi));
    lo = h2{(_Float16)fmaf(x0, f, -(float)hi[0]), (_Float16)fmaf(x1, f, -(float)hi[1])};
}
__device__ inline float opaque_one() {
    float f = 1.f;
    asm("" : "+s"(f));
    return f;
}
__device__ inline float other_half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float other_half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

/* f16 caches: a weight is off by 2^-25 2^-SHIFT beside its own 2^-22.  f32
 * caches, whose groups of positions shift weights by up to SPREAD more, keep
 * 2^-25 with SHIFT = SPREAD. */
constexpr float SHIFT_H = 8.f, LAG_H = 7.f;
constexpr float SHIFT_F = 12.f, LAG_F = 3.f;

/* A lane's m-row (both halves of a wave hold the same 32) and what its wave
 * sees: positions any_lo .. any_hi by some row, all_lo .. all_hi by all. */
struct Lane {
    bool live;       /* false: no row there; its q is zero, nothing is masked, nothing written */
    int first, last;
    int r, h;        /* packed row, query head */
    int any_lo, any_hi, all_lo, all_hi;
};
/* ms: the wave's m-rows, from the tile's from on, of which the lane takes at */
__device__ inline Lane lane_rows(const PromptArgs &a, const Work &w, int from, int at, int ms, int ratio) {
    Lane x;
    int first = 0, last = 0, i, j, i0, i1, u;
    w.row(from + at, ratio, i, j);
    x.live = row_sees(a, w, i, first, last);
    x.r = w.sq.r0 + (x.live ? i : 0), x.h = w.kh * ratio + (x.live ? j : 0);
    x.first = x.live ? first : 0, x.last = x.live ? last : 0x7FFFFFFF;
    w.row(from, ratio, i0, u), w.row(from + ms - 1, ratio, i1, u);   /* uniform */
    i1 = min(w.sq.n - 1, i1);
    if (i0 > i1) {
        x.any_lo = 0x7FFFFFFF, x.any_hi = -1, x.all_lo = 0, x.all_hi = 0x7FFFFFFF;
    } else if (!w.prefix) {   /* later rows see later positions */
        const int l0 = w.sq.past + i0, l1 = w.sq.past + i1;
        x.any_hi = l1, x.all_hi = l0;
        x.any_lo = a.window > 0 ? max(0, l0 + 1 - a.window) : 0;
        x.all_lo = a.window > 0 ? max(0, l1 + 1 - a.window) : 0;
    } else if (a.window <= 0) {
        x.any_lo = x.all_lo = 0, x.any_hi = x.all_hi = a.pre_len - 1;
    } else {   /* rows of sequences of any length */
        int lo = x.live ? first : 0x7FFFFFFF, hi = x.live ? last : -1, alo = x.first, ahi = x.last;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            lo = min(lo, __shfl_xor(lo, o, 64));
            hi = max(hi, __shfl_xor(hi, o, 64));
            alo = max(alo, __shfl_xor(alo, o, 64));
            ahi = min(ahi, __shfl_xor(ahi, o, 64));
        }
        x.any_lo = lo, x.any_hi = hi, x.all_lo = alo, x.all_hi = ahi;
    }
    x.any_lo = __builtin_amdgcn_readfirstlane(x.any_lo), x.any_hi = __builtin_amdgcn_readfirstlane(x.any_hi);
    x.all_lo = __builtin_amdgcn_readfirstlane(x.all_lo), x.all_hi = __builtin_amdgcn_readfirstlane(x.all_hi);
    return x;
}

/* the largest of the wave's words, uniform */
__device__ inline uint32_t wave_umax(uint32_t v) {
    v = max(v, (uint32_t)dpp_i<0xB1>((int)v));
    v = max(v, (uint32_t)dpp_i<0x4E>((int)v));
    v = max(v, (uint32_t)dpp_i<0x141>((int)v));
    v = max(v, (uint32_t)dpp_i<0x140>((int)v));
    const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 15), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 31);
    const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 47), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
    return max(max(a, b), max(c, d));
}

/* the power of two that takes a largest magnitude to 2^14 .. 2^15, as its exponent */
__device__ inline int scale_exp(float big) {
    return big > 0.f && big < INFINITY ? min(15 - __builtin_amdgcn_frexp_expf(big), 100) : 0;
}

/* q of the lane's m-row as the B operands of the first product, two f16
 * planes, from its 16-byte pieces (of which fetch(i) is the i-th, zeros past
 * the row); returns the factor that takes scores of the planes to base 2 */
template <int HD, typename F>
__device__ inline float load_q(int head_dim, int half, const F &fetch, h8 (&qh)[HD / 16], h8 (&ql)[HD / 16]) {
    f4 y[HD / 8];
    float big = 0.f;
#pragma unroll
    for (int s = 0; s < HD / 16; s++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const f4 u = y[2 * s + e] = fetch(4 * s + 2 * half + e);
            big = max_nan(big, max_nan(max_nan(fabsf(u[0]), fabsf(u[1])), max_nan(fabsf(u[2]), fabsf(u[3]))));
        }
    const int ex = scale_exp(other_half_max(big));
    const float f = __builtin_amdgcn_ldexpf(1.f, ex);
#pragma unroll
    for (int s = 0; s < HD / 16; s++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float y0 = y[2 * s + (e >> 2)][e & 3], y1 = y[2 * s + (e >> 2)][(e & 3) + 1];
            h2 hi, lo;
            split2(y0 * f, y1 * f, y0, y1, f, hi, lo);
            qh[s][e] = hi[0], qh[s][e + 1] = hi[1], ql[s][e] = lo[0], ql[s][e + 1] = lo[1];
        }
    return __builtin_amdgcn_ldexpf(LOG2E / sqrtf((float)head_dim), -ex);
}

/* ... straight from memory */
__device__ inline auto memory_q(const PromptArgs &a, const Lane &x) {
    const float *src = a.q + (size_t)x.r * a.q_stride + (size_t)x.h * a.head_dim;
    const int n = x.live ? a.head_dim / 4 : 0;
    return [=](int i) { return i < n ? (f4)*(const f4u *)(src + 4 * i) : f4{0.f, 0.f, 0.f, 0.f}; };
}

/* With two groups, the m-rows' q and outputs go through LDS, row by row: a lane
 * holds one m-row's values, and 64 rows in an access of 16 bytes a lane are
 * many lines for the address unit (loading q took 2.2 - 3.6 us of a
 * workgroup's prologue that way, writing o 2.4).  512 tokens 22.5 -> 21.0 us;
 * with one group, whose q would have to come before its first tile, 16 tokens
 * took 10.0 instead of 8.8.  Rows of HD floats, 16-byte piece i of row r at
 * place i ^ (r mod HD / 4), where neither order of access meets itself in a
 * bank. */
template <int HD>
__device__ inline uint32_t row_piece(int row, int piece) {
    return (uint32_t)((piece ^ (row & (HD / 4 - 1))) << 4);
}
/* q of the tile's ROWS m-rows by direct copies, `waves` of them from `wave`
 * on: the first half of the rows to lo, the second to hi */
template <int HD, int ROWS>
__device__ inline void copy_q(const PromptArgs &a, const Work &w, int ratio, int wave, int waves, uint8_t *lo, uint8_t *hi) {
    constexpr int R = 256 / HD, N = ROWS / R;   /* rows of a copy, copies */
    const int lane = threadIdx.x & 63, place = lane % (HD / 4);
    const u32x4 d = buf_desc(a.q + (size_t)(w.sq.r0 + w.i0) * a.q_stride + (size_t)w.kh * ratio * a.head_dim, 0x7FFFFF00u);
    for (int n = wave; n < N; n += waves) {
        const int row = R * n + lane / (HD / 4), piece = place ^ (row & (HD / 4 - 1));
        int i, j;
        w.row(row, ratio, i, j);
        const uint32_t off = ((uint32_t)(i - w.i0) * (uint32_t)a.q_stride + (uint32_t)(j * a.head_dim + 4 * piece)) * 4u;
        copy_lanes(d, i < w.sq.n && 4 * piece < a.head_dim ? off : 0x7FFFFF00u,
                   lds_addr(n < N / 2 ? lo : hi) + 1024u * (uint32_t)(n % (N / 2)));
    }
}
/* the staged outputs, rows of wave v at lds + v * stride, to where they go */
template <int HD, int ROWS>
__device__ inline void store_rows(int head_dim, const uint8_t *lds, int stride, const long long *where, float *base, int wave,
                                  int waves) {
    constexpr int R = 256 / HD;
    const int lane = threadIdx.x & 63, piece = lane % (HD / 4);
    for (int n = wave; n < ROWS / R; n += waves) {
        const int row = R * n + lane / (HD / 4);
        const long long at = where[row];
        const f4 y = *(const f4 *)(lds + (row >> 5) * stride + (row & 31) * (HD * 4) + row_piece<HD>(row, piece));
        if (at >= 0 && 4 * piece < head_dim) *(f4u *)(base + at + 4 * piece) = y;
    }
}

/* Byte offset in a tile of 16-bit rows of the lane's operand of the first
 * product (step s: XOR s << 5, positions + 32: + 32 rows), and of the columns
 * of the second (dims 32 d ..; e: the chunk's positions 8 e ..; 16 positions
 * on: + 16 rows). */
template <int HD>
__device__ inline uint32_t k_operand(int lane) {
    return (uint32_t)((lane & 31) * (HD * 2) + (((lane >> 5) ^ swz<HD>(lane & 31)) << 4));
}
template <int HD>
__device__ inline uint32_t v_operand(int lane, int d, int e) {
    const int key = 8 * e + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    return (uint32_t)(key * (HD * 2) + ((piece ^ swz<HD>(key)) << 4) + 8 * (lane & 1));
}

/* scores of 32 positions, register v at position at + 8 (v / 4) + v % 4: -inf
 * for those that the row does not see (most tiles: none, by uniform tests) */
__device__ inline void mask_scores(f16v &s, int at, const Lane &x) {
    const int t = __builtin_amdgcn_readfirstlane(at);   /* lane 0: the first position */
    if (t + 31 > x.all_hi) {
        const int n = x.last - at;
#pragma unroll
        for (int v = 0; v < 16; v++) s[v] = 8 * (v >> 2) + (v & 3) <= n ? s[v] : -INFINITY;
    }
    if (t < x.all_lo) {
        const int n = x.first - at;
#pragma unroll
        for (int v = 0; v < 16; v++) s[v] = 8 * (v >> 2) + (v & 3) >= n ? s[v] : -INFINITY;
    }
}

/* Group 1's sums of a workgroup whose two groups of MW waves took the tiles
 * in turn, through LDS (room: MW * 64 * (HD / 2 + 3) floats), into group 0's.
 * oexp as in write_rows. */
template <int HD, int MW>
__device__ inline void merge_groups(float *lds, int wave, int lane, float &mx, float &l, int &oexp, f16v (&o)[HD / 32]) {
    constexpr int N = HD / 2;   /* o values a lane */
    float *at = lds + (wave % MW) * 64 * (N + 3);
    __syncthreads();
    if (wave >= MW) {
#pragma unroll
        for (int d = 0; d < HD / 32; d++)
#pragma unroll
            for (int v = 0; v < 16; v += 4)
                *(f4 *)&at[((16 * d + v) / 4 * 64 + lane) * 4] = f4{o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
        at[64 * N + lane] = mx, at[64 * (N + 1) + lane] = l, at[64 * (N + 2) + lane] = __int_as_float(oexp);
    }
    __syncthreads();
    if (wave >= MW) return;
    const float m1 = at[64 * N + lane], M = max_nan(mx, m1), base = M == -INFINITY ? 0.f : M;
    const int e1 = __float_as_int(at[64 * (N + 2) + lane]), e = min(oexp, e1);
    const float a0 = __builtin_amdgcn_exp2f(mx - base), a1 = __builtin_amdgcn_exp2f(m1 - base);
    const float f0 = __builtin_amdgcn_ldexpf(a0, e - oexp), f1 = __builtin_amdgcn_ldexpf(a1, e - e1);
    l = fmaf(l, a0, at[64 * (N + 1) + lane] * a1);
    mx = M, oexp = e;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
            const f4 y = *(const f4 *)&at[((16 * d + v) / 4 * 64 + lane) * 4];
#pragma unroll
            for (int q = 0; q < 4; q++) o[d][v + q] = fmaf(o[d][v + q], f0, y[q] * f1);
        }
}

#define MFMA_H(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0)

}  // namespace tg
#endif
