/*
 * tg_prompt.hip -- packed rows of several sequences: their K and V rows into
 * the caches, and their attention over them.
 *
 * The reference runs attention one row at a time (tg_attention_v2,
 * csrc/libtinygiant.c:939-983, called row by row at tinygiant/engine.py:
 * 232-275); these are the same formulas for many rows a call:
 *
 *   append     K and V of each row, normed and rotated, into its slot; q normed
 *              and rotated (k_kv_append)
 *   attention  o = sum_j p_j v_j / (sum_j p_j + p_sink),
 *              p_j = exp(q k_j / sqrt(head_dim) - m), over the positions that
 *              the row sees, in one pass with running m and sums
 *
 * Kernels of the attention, chosen by sizes alone (rows_cut):
 *   k_rows_h        f16 caches, 128 query rows of a KV head a workgroup
 *   k_rows_f        f32 caches, 128 or 256
 *   k_rows_n        either, 16: few rows
 *   k_rows_combine  joins what several workgroups made of a row's positions
 * A row that does not come out finite is computed again from the formulas
 * with plain loads (slow_row).
 */
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
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

/* ---- append ----
 * One workgroup a row; a segment of G lanes (16, or 8 for heads of up to 64
 * values) takes a head: lane i the pairs (4 i + e, head_dim / 2 + 4 i + e),
 * so the loads are 16 bytes and RoPE needs no exchange.  The norm is
 * tg_rms_norm's (csrc/libtinygiant.c:680-698), the rotation
 * apply_rope_inplace's (:702-719); an f16 cache gets K and V rounded once, to
 * nearest.  Bound: the bytes.  4,001 rows of 64 + 2 x 8 heads of 64 into an f32
 * cache: 165 MB in 32.9 us, 5.0 TB/s, a large copy's rate; 8 rows 6 us, the
 * launch and two dependent reads. */
template <bool HALF, int G>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
    const int r = blockIdx.x;
    Seq sq;
    int i;
    if (!wave_seq_of(a.s, r, sq, i)) return;
    const int at = sq.past + i, pos = a.base_pos + at;
    const bool turn = a.rope_cos != nullptr;
    if (turn && pos >= a.rope_len) return;
    const int seg = threadIdx.x / G, l = threadIdx.x % G;
    const int half = a.head_dim / 2, hd = a.head_dim;
    const bool on = 4 * l < half;
    f4 c = {1.f, 1.f, 1.f, 1.f}, sn = {0.f, 0.f, 0.f, 0.f};
    if (turn && on) {
        c = *(const f4u *)(a.rope_cos + (size_t)pos * half + 4 * l);
        sn = *(const f4u *)(a.rope_sin + (size_t)pos * half + 4 * l);
    }
    const int heads = a.n_heads + 2 * a.n_kv;
    for (int h0 = a.q_out ? 0 : a.n_heads; h0 < heads; h0 += 256 / G) {
        const int h = h0 + seg;
        const bool live = h < heads && on;
        const int kh = h - a.n_heads;   /* K heads from 0, V heads from n_kv */
        const bool isq = h < a.n_heads, isv = kh >= a.n_kv;
        const float *src = isq ? a.q + (size_t)r * a.q_stride + (size_t)h * hd
                               : (isv ? a.v + (size_t)(kh - a.n_kv) * hd : a.k + (size_t)kh * hd) + (size_t)r * a.kv_stride;
        f4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
        if (live) {
            x = *(const f4u *)(src + 4 * l);
            y = *(const f4u *)(src + half + 4 * l);
        }
        const float *nw = isq ? a.q_norm : isv ? nullptr : a.k_norm;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        if (!live) continue;
        if (nw) {
            const float scale = 1.f / sqrtf(ss / (float)hd + a.eps);
            x = x * scale * (f4)*(const f4u *)(nw + 4 * l);
            y = y * scale * (f4)*(const f4u *)(nw + half + 4 * l);
        }
        if (turn && !isv) {
            const f4 t = x * c - y * sn;
            y = y * c + x * sn;
            x = t;
        }
        if (isq) {
            float *dst = a.q_out + (size_t)r * a.q_out_stride + (size_t)h * hd;
            *(f4u *)(dst + 4 * l) = x;
            *(f4u *)(dst + half + 4 * l) = y;
            continue;
        }
        const size_t row = (((size_t)sq.slot * a.n_kv + (isv ? kh - a.n_kv : kh)) * a.s.kv_max + at) * hd;
        void *base = isv ? a.kv_v : a.kv_k;
        if constexpr (HALF) {
            _Float16 *dst = (_Float16 *)base + row;
            *(h4 *)(dst + 4 * l) = __builtin_convertvector(x, h4);
            *(h4 *)(dst + half + 4 * l) = __builtin_convertvector(y, h4);
        } else {
            float *dst = (float *)base + row;
            *(f4 *)(dst + 4 * l) = x;
            *(f4 *)(dst + half + 4 * l) = y;
        }
    }
}

void launch_kv_append(const AppendArgs &a, bool half, hipStream_t st) {
    const dim3 grid(a.s.rows), block(256);
    const bool narrow = a.head_dim <= 64;
    if (half) {
        if (narrow) hipLaunchKernelGGL((k_kv_append<true, 8>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_kv_append<true, 16>), grid, block, 0, st, a);
    } else {
        if (narrow) hipLaunchKernelGGL((k_kv_append<false, 8>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_kv_append<false, 16>), grid, block, 0, st, a);
    }
}

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

/* Tile b of the sequences' tiles of MTILE m-rows, late rows first (they see
 * the most positions).  Sequence s has its tiles from place
 * cu[s] ratio / MTILE + s on, where there is room for them whatever the
 * sequences before it left over: no sum over those is needed. */
template <int MTILE>
__device__ inline bool find_tile(const PromptArgs &a, const RowsPlan &p, int ratio, int b, Work &w) {
    const PackedSeqs &c = a.s;
    const int lane = threadIdx.x & 63;
    const Run run = wave_narrow<MTILE>(c, ratio, b);
    Seq q = {0, 0, 0, 0};
    if (lane < run.count) q = seq_at(c, run.at + lane);
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
template <int MTILE>
__device__ inline bool find_span(const PromptArgs &a, const RowsPlan &p, int ratio, int b, Work &w) {
    const PackedSeqs &c = a.s;
    const int lane = threadIdx.x & 63;
    Seq q = {0, 0, 0, 0};
    auto load = [&](int s0) {
        q.n = 0;
        if (s0 + lane < c.n) q = seq_at(c, s0 + lane);
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

template <typename T>
__device__ inline const T *region(const PromptArgs &a, const Work &w, const void *own, const void *pre) {
    return w.prefix ? (const T *)pre + (size_t)w.kh * a.pre_max * a.head_dim
                    : (const T *)own + ((size_t)w.sq.slot * a.n_kv + w.kh) * a.s.kv_max * a.head_dim;
}

/* One m-row over the work's span by 256 threads of the workgroup, from the formulas
 * with plain loads: only positions that the row sees are read.  It is how
 * rows are computed that came out of the matrix units not finite, which
 * multiply every value of a tile: 0 * inf there is not a row's own result.
 * lds: PROMPT_MAX_HEAD_DIM + 260 floats. */
template <typename T>
__device__ void slow_row(const PromptArgs &a, const RowsPlan &p, const Work &w, int at, int ratio, float *lds) {
    float *qs = lds, *sc = lds + PROMPT_MAX_HEAD_DIM, *red = sc + 256;
    const int tid = threadIdx.x, hd = a.head_dim;
    const bool on = tid < 256;   /* further threads only keep the barriers */
    int i, j, first = 0, last = -1;
    w.row(at, ratio, i, j);
    const int h = w.kh * ratio + j, r = w.sq.r0 + i;
    (void)row_sees(a, w, i, first, last);
    first = max(first, w.lo), last = min(last, w.hi - 1);
    const T *k = region<T>(a, w, a.kv_k, a.pre_k), *v = region<T>(a, w, a.kv_v, a.pre_v);
    const float scale = LOG2E / sqrtf((float)hd);
    __syncthreads();
    if (tid < hd) qs[tid] = a.q[(size_t)r * a.q_stride + (size_t)h * hd + tid];
    float mx = -INFINITY, l = 0.f, o = 0.f;
    __syncthreads();
    for (int t0 = first; t0 <= last; t0 += 256) {
        const int pz = t0 + tid;
        float z = -INFINITY;
        if (on && pz <= last) {
            const T *row = k + (size_t)pz * hd;
            float acc = 0.f;
            for (int d = 0; d < hd; d++) acc = fmaf(qs[d], (float)row[d], acc);
            z = acc * scale;
        }
        float t = wave_max(z);
        if (on && (tid & 63) == 0) red[tid >> 6] = t;
        __syncthreads();
        t = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(mx, t), base = mn == -INFINITY ? 0.f : mn, alpha = exp2f(mx - base);
        const float e = on && pz <= last ? exp2f(z - base) : 0.f;
        if (on) sc[tid] = e;
        const float s = wave_sum(e);
        __syncthreads();
        if (on && (tid & 63) == 0) red[tid >> 6] = s;
        __syncthreads();
        l = l * alpha + ((red[0] + red[1]) + (red[2] + red[3]));
        mx = mn;
        if (tid < hd) {
            o *= alpha;
            const int n = min(256, last + 1 - t0);
            for (int n1 = 0; n1 < n; n1++) o = fmaf(sc[n1], (float)v[(size_t)(t0 + n1) * hd + tid], o);
        }
        __syncthreads();
    }
    if (p.nrec) {
        const size_t rec = ((size_t)r * a.n_heads + h) * p.nrec + w.rec;
        /* scores that are all NaN leave mx at -inf, which is the record of no position */
        if (tid == 0) write_ml(p, w, rec, l != l ? l : mx, l);
        if (tid < hd) p.o[rec * hd + tid] = o;
    } else if (tid < hd) {
        if (a.sinks) {
            const float sk = a.sinks[h] * LOG2E, mn = fmaxf(mx, sk), base = mn == -INFINITY ? 0.f : mn, f = exp2f(mx - base);
            l = l * f + exp2f(sk - base);
            o *= f;
        }
        a.out[(size_t)r * a.out_stride + (size_t)h * hd + tid] = o / l;
    }
}

}  // namespace

/* ---- float16 caches on the matrix units ----
 *
 * S^T[position][m-row] = K Q^T and O^T[dim][m-row] += V^T P^T, both as
 * v_mfma_f32_32x32x16_f16.  D of the first has m-row lane % 32, positions
 * 8 (v / 4) + 4 (lane / 32) + v % 4 in register v: a lane holds one m-row's
 * scores, so the softmax needs one exchange between the two halves of the
 * wave, and its own registers are the B operand of the second product, whose
 * k index is a permutation of the positions that V^T's fragments follow
 * (ds_read_b64_tr_b16: four positions of one dim a lane).  O^T too has the
 * m-row in the lane: rescaling needs no exchange.
 *
 * K and V are f16 as they are.  q and the weights are f32: each is the sum of
 * two f16 (hi the nearest, lo the nearest to the rest: 22 bits), so each
 * product is two MFMAs, and the result is as good as f32 sums.  What keeps
 * lo out of f16's underflow: q is scaled by a power of two a row (its largest
 * value to 2^14 .. 2^15), undone in the factor that takes scores to base 2;
 * weights are taken times 2^SHIFT.
 *
 * The reference exponent m follows a row's largest score only when that is
 * more than LAG above it, so most tiles rescale nothing (8,192 tokens: 883 us,
 * with m the largest score 910).  SHIFT + LAG stays below f16's largest, 2^16.
 *
 * K and V tiles of 64 positions go to LDS by direct copies, two buffers; the
 * 16-byte pieces of a row are permuted by its position (swz) so that neither
 * the K fragments (16 positions, one piece) nor the transposing reads (8
 * positions, four pieces) meet in the same banks.  Rows past the region's end
 * and dims past head_dim arrive as zeros. */
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

/* The wave's rows finished: weights were summed times 2^SHIFT
 * relative to 2^mx, values (SCALED) besides in units of 2^-oexp.  They go to
 * `stage` (LDS, the wave's 32 rows), where[] saying where in p.o or a.out each
 * belongs (-1: nowhere), or without stage to memory.  Returns the m-rows that
 * came out not finite, which are not written. */
template <int HD, bool SCALED>
__device__ inline uint32_t write_rows(const PromptArgs &a, const RowsPlan &p, const Work &w, const Lane &x, int lane, float mx,
                                      float l, int oexp, const f16v (&o)[HD / 32], uint8_t *stage, long long *where) {
    constexpr float SHIFT = SCALED ? SHIFT_F : SHIFT_H;
    float big = fabsf(l);   /* NaN where anything is */
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) big = max_nan(big, fabsf(o[d][v]));
    const uint64_t mask = __ballot(x.live && !(big < INFINITY));
    const uint32_t bad = (uint32_t)mask | (uint32_t)(mask >> 32);
    const int half = lane >> 5, row = lane & 31, hd = a.head_dim;
    bool write = x.live && !((bad >> row) & 1u);
    long long at;
    float f = 1.f;
    if (p.nrec) {
        const size_t rec = ((size_t)x.r * a.n_heads + x.h) * p.nrec + w.rec;
        constexpr float one = 1.f / (float)(1 << (int)SHIFT);
        if (write && half == 0) write_ml(p, w, rec, mx, l * one);
        write = write && mx > -INFINITY;      /* a record of no position has no sums */
        at = (long long)(rec * hd);
        f = one;
    } else {
        if (a.sinks && write) {
            const float ref = mx - SHIFT, sk = a.sinks[x.h] * LOG2E, M = fmaxf(ref, sk), base = M == -INFINITY ? 0.f : M;
            f = exp2f(ref - base);
            l = l * f + exp2f(sk - base);
        }
        f /= l;
        at = (long long)x.r * a.out_stride + (long long)x.h * hd;
    }
    if (stage && half == 0) where[row] = write ? at : -1;
    float *dst = (p.nrec ? p.o : a.out) + at;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int dim = 32 * d + 8 * v + 4 * half;
            f4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = SCALED ? __builtin_amdgcn_ldexpf(o[d][4 * v + e] * f, -oexp) : o[d][4 * v + e] * f;
            if (stage) *(f4 *)(stage + row * (HD * 4) + row_piece<HD>(row, 8 * d + 2 * v + half)) = y;
            else if (write && dim < hd) *(f4u *)(dst + dim) = y;
        }
    return bad;
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

/* MW waves of 32 m-rows; with KG = 2, two groups of them take the tiles in
 * turn.  J blocks of 32 positions are computed together: two overlap their
 * latencies (8,192 tokens: 883 us, one at a time 911), one is half the code
 * and skips what a window hides (4,096 tokens, window 128: 42.9, 45.4).
 *
 * Bound for long prompts: the matrix units at the power limit.  8,192 tokens of
 * 32 heads of 128: 883 us (923 on another card), 1.25 PFLOP/s counting both
 * products (a large f16 product runs at 1.23), the clock at 1.45 - 1.6 GHz.  4,096 tokens of 64 heads of
 * 64 with a window of 128: 42.9 us, 142 MB; two rounds of workgroups that load
 * (5 us), compute (8: a block's softmax takes more issue slots than its
 * products) and store (2) with little overlap between those of a CU. */
template <int HD, int MW, int KG>
struct SharedH {
    __attribute__((aligned(1024))) uint8_t bufs[KG][2][2][KT * HD * 2];
    uint32_t bad_rows[MW];
    long long where[KG == 2 ? 32 * MW : 1];
};
template <int HD, int MW, int KG, int J>
__device__ inline __attribute__((always_inline)) void rows_h(const PromptArgs &a, const RowsPlan &p, SharedH<HD, MW, KG> &sh) {
    constexpr int RB = HD * 2, TILE = KT * RB;       /* bytes of a row in LDS, of a tile of K or V */
    constexpr int NC = TILE / 1024 / MW;             /* copies of 1 KiB a wave, matrix and tile */
    constexpr int DB = HD / 32, STEPS = HD / 16;
    auto &bufs = sh.bufs;
    auto &bad_rows = sh.bad_rows;
    auto &where = sh.where;
    const int ratio = a.n_heads / a.n_kv, hd = a.head_dim;
    Work w;
    if (!find_work<32 * MW>(a, p, ratio, w)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, group = wave / MW, mwave = wave % MW;
    static_assert(KG == 1 || sizeof bufs >= MW * 256 * (HD / 2 + 3), "merge_groups");
    uint8_t(*buf)[2][TILE] = bufs[group];

    /* copies: LDS byte 1024 n + 16 l of a tile is piece c' of row key; n = mwave + MW k */
    const uint32_t rb = (uint32_t)hd * 2u;
    const u32x4 kd = buf_desc(region<_Float16>(a, w, a.kv_k, a.pre_k), (uint32_t)w.hi * rb);
    const u32x4 vd = buf_desc(region<_Float16>(a, w, a.kv_v, a.pre_v), (uint32_t)w.hi * rb);
    const int ckey = (1024 * mwave + 16 * lane) / RB, cpiece = (lane % (RB / 16)) ^ swz<HD>(ckey);
    const uint32_t coff = 8 * cpiece < hd ? (uint32_t)ckey * rb + 16u * (uint32_t)cpiece : 0x7FFFFF00u;
    auto copy_tile = [&](int t0, int b) __attribute__((always_inline)) {
        const uint32_t at = coff + (uint32_t)t0 * rb;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const uint32_t src = at + (uint32_t)k * (MW * 1024u / RB) * rb, dst = 1024u * (uint32_t)(mwave + MW * k);
            copy_lanes(kd, src, lds_addr(buf[b][0]) + dst);
            copy_lanes(vd, src, lds_addr(buf[b][1]) + dst);
        }
    };
    static_assert(MW * 1024 / RB % 16 == 0, "swz of a copy's rows is that of the first");
    if (w.lo + group * KT < w.hi) copy_tile(w.lo + group * KT, 0);
    /* two groups: q comes by way of their second buffers, with the first tiles
     * (one group would have to fetch one after the other) */
    static_assert(KG == 1 || 32 * MW * HD * 4 == sizeof bufs / 2, "q fits");
    if constexpr (KG == 2) copy_q<HD, 32 * MW>(a, w, ratio, wave, MW * KG, bufs[0][1][0], bufs[1][1][0]);
    const Lane x = lane_rows(a, w, 32 * mwave, lane & 31, 32, ratio);

    h8 qh[STEPS], ql[STEPS];
    float c;
    if constexpr (KG == 2) {
        wait_copies();
        bar_lds();
        const uint8_t *mine = bufs[mwave / (MW / 2)][1][0] + (mwave % (MW / 2) * 32 + (lane & 31)) * (HD * 4);
        c = load_q<HD>(hd, half, [&](int i) { return *(const f4 *)(mine + row_piece<HD>(lane & 31, i)); }, qh, ql);
    } else {
        c = load_q<HD>(hd, half, memory_q(a, x), qh, ql);
    }
    f16v o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[d][v] = 0.f;
    float mx = -INFINITY, l = 0.f;
    const uint32_t kaddr = k_operand<HD>(lane);
    uint32_t vaddr[DB][2];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 2; e++) vaddr[d][e] = TILE + v_operand<HD>(lane, d, e);

    const float one = opaque_one();
    int b = 0;
    for (int t0 = w.lo; t0 < w.hi; t0 += KG * KT, b ^= 1) {
        const int t = t0 + group * KT;
        wait_copies();
        bar_lds();   /* every wave's copies of this tile are there, and every wave is done with the other buffer */
        if (t + KG * KT < w.hi) copy_tile(t + KG * KT, b ^ 1);
        if (t > x.any_hi || t + KT <= x.any_lo || t >= w.hi) continue;   /* uniform in the wave */
#pragma unroll 1
        for (int n = 0; n < KT; n += 32 * J) {
            const int at = t + n;
            if (J == 1 && (at > x.any_hi || at + 32 <= x.any_lo)) continue;
            const Lds tile = (Lds)buf[b][0] + n * RB;
            f16v s[J];
            h8 k0[J], k1[J];
#pragma unroll
            for (int j = 0; j < J; j++) {
#pragma unroll
                for (int v = 0; v < 16; v++) s[j][v] = 0.f;
                k0[j] = lds_row(tile + kaddr + j * 32 * RB);
            }
#pragma unroll
            for (int st = 0; st < STEPS; st++) {   /* the next step's operands are read a step ahead */
                const Lds next = tile + (kaddr ^ (uint32_t)((st + 1) << 5));
#pragma unroll
                for (int j = 0; j < J; j++) k1[j] = st + 1 < STEPS ? lds_row(next + j * 32 * RB) : k0[j];
#pragma unroll
                for (int j = 0; j < J; j++) s[j] = MFMA_H(k0[j], ql[st], s[j]);
#pragma unroll
                for (int j = 0; j < J; j++) s[j] = MFMA_H(k0[j], qh[st], s[j]);
#pragma unroll
                for (int j = 0; j < J; j++) k0[j] = k1[j];
            }
            auto column = [&](int i) __attribute__((always_inline)) {
                const int q = i / DB, d = i % DB;
                return h8_of(lds_column(tile + vaddr[d][0] + q * 16 * RB), lds_column(tile + vaddr[d][1] + q * 16 * RB));
            };
            h8 v0 = column(0), v1 = column(1);
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < J; j++) {
                mask_scores(s[j], at + 32 * j + 4 * half, x);
#pragma unroll
                for (int v = 0; v < 16; v++) top = max_nan(top, s[j][v]);
            }
            top = other_half_max(top) * c;
            if (__any(top > mx + LAG_H)) {
                const float mn = max_nan(mx, top);
                const float alpha = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
                mx = mn;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[d][v] *= alpha;
            }
            const float sh = mx == -INFINITY ? 0.f : SHIFT_H - mx;
            /* the scheduler's order of MFMAs and exponentials: 8,192 tokens 896 us without, 883 */
            __builtin_amdgcn_iglp_opt(2);
            h8 ph[2 * J], pl[2 * J];
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int v = 0; v < 16; v += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(s[j][v], c, sh));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(s[j][v + 1], c, sh));
                    sum[v & 3] += e0, sum[(v & 3) + 1] += e1;
                    h2 hi, lo;
                    split2(e0, e1, e0, e1, one, hi, lo);
                    const int q = 2 * j + (v >> 3), e = v & 7;
                    ph[q][e] = hi[0], ph[q][e + 1] = hi[1], pl[q][e] = lo[0], pl[q][e + 1] = lo[1];
                }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
            for (int i = 0; i < 2 * J * DB; i += 2) {
                const bool more = i + 2 < 2 * J * DB;
                const h8 n0 = more ? column(i + 2) : v0, n1 = more ? column(i + 3) : v1;
                const int q = i / DB, d = i % DB;
                o[d] = MFMA_H(v0, pl[q], o[d]);
                o[d + 1] = MFMA_H(v1, pl[q], o[d + 1]);
                o[d] = MFMA_H(v0, ph[q], o[d]);
                o[d + 1] = MFMA_H(v1, ph[q], o[d + 1]);
                v0 = n0, v1 = n1;
            }
        }
    }
    l = other_half_sum(l);
    int oexp = 0;
    if (KG == 2 && w.hi - w.lo > KT) merge_groups<HD, MW>((float *)bufs, wave, lane, mx, l, oexp, o);
    else __syncthreads();   /* one group, or the second had no tile: all are done with the tiles */
    constexpr int STRIDE = 64 * (HD / 2 + 3) * 4;   /* a wave's share of merge_groups' room */
    if (group == 0) {
        const uint32_t bad = write_rows<HD, false>(a, p, w, x, lane, mx, l, oexp, o, KG == 2 ? (uint8_t *)bufs + wave * STRIDE : nullptr,
                                                   where + (KG == 2 ? 32 * wave : 0));
        if (lane == 0) bad_rows[wave] = bad;
    }
    __syncthreads();
    if constexpr (KG == 2) {
        store_rows<HD, 32 * MW>(hd, (const uint8_t *)bufs, STRIDE, where, p.nrec ? p.o : a.out, wave, MW * KG);
        __syncthreads();
    }
    for (int wv = 0; wv < MW; wv++)
        for (uint32_t y = bad_rows[wv]; y; y &= y - 1)
            slow_row<_Float16>(a, p, w, 32 * wv + __builtin_ctz(y), ratio, (float *)bufs);
}

template <int HD, int MW, int KG, int J>
__global__ __launch_bounds__(64 * MW * KG, HD == 64 && J == 1 ? 4 : 2) void k_rows_h(PromptArgs a, RowsPlan p) {
    __shared__ SharedH<HD, MW, KG> sh;
    rows_h<HD, MW, KG, J>(a, p, sh);
}

/* ---- few rows: positions over the waves ----
 *
 * A workgroup of four waves takes 16 m-rows; a wave walks tiles of 16
 * positions (every fourth) with K and V straight from the cache into the
 * operands, no LDS and no barrier until the end, where the four waves' sums
 * meet.  S^T[position][m-row] on 16x16 MFMAs: D lane l holds m-row l % 16,
 * positions 4 (l / 16) + v, which is B of the second product over positions
 * 4 (l / 16) + i as it lies.  The second product is f32 (16x16x4) for both
 * cache types: V converts exactly, the weights are not rounded, and the rate
 * is above what the cache's bytes allow.  The first is f32 for an f32 cache
 * and two f16 products (q in two planes) for an f16 one.
 *
 * Bound: the cache's bytes.  One row of each of 32 sequences of 2,091 positions
 * on average, 4 KV heads of 128, f16: 137 MB in 32 us, 4.3 TB/s; at 1,500
 * positions and less the chain of a workgroup (find its work 1 us, q and the
 * first tile 3, merge and write 3). */
typedef float v4f __attribute__((ext_vector_type(4)));
constexpr int MN = 16;

template <typename T, int HD>
struct NarrowK {   /* float: K pieces of 4 dims, dims 16 j + 4 kq + e in MFMA (j, e) */
    static constexpr int J = HD / 16;
    v4f q[J];
    u32x4 k[J];
    __device__ inline float load_q(const PromptArgs &a, const Lane &x, int kq) {
        const float *src = a.q + (size_t)x.r * a.q_stride + (size_t)x.h * a.head_dim;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int d = 16 * j + 4 * kq;
            q[j] = x.live && d < a.head_dim ? (v4f)*(const f4u *)(src + d) : v4f{0.f, 0.f, 0.f, 0.f};
        }
        return LOG2E / sqrtf((float)a.head_dim);
    }
    __device__ inline void load_k(Buf kd, uint32_t row, int kq, int hd) {
#pragma unroll
        for (int j = 0; j < J; j++) k[j] = ld16(kd, 16 * j + 4 * kq < hd ? row + 64u * j + 16u * (uint32_t)kq : 0x7FFFFF00u);
    }
    __device__ inline v4f scores() const {
        v4f s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;   /* two chains */
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = __uint_as_float(k[j][e]);
                if (e & 1) s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(y, q[j][e], s1, 0, 0, 0);
                else s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(y, q[j][e], s0, 0, 0, 0);
            }
        return s0 + s1;
    }
};
template <int HD>
struct NarrowK<_Float16, HD> {   /* K pieces of 8 dims, dims 32 j + 8 kq + e in MFMA j */
    static constexpr int J = HD / 32;
    h8 qh[J], ql[J];
    u32x4 k[J];
    __device__ inline float load_q(const PromptArgs &a, const Lane &x, int kq) {
        const float *src = a.q + (size_t)x.r * a.q_stride + (size_t)x.h * a.head_dim;
        f4 u[J], v[J];
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int d = 32 * j + 8 * kq;
            const bool on = x.live && d < a.head_dim;
            u[j] = on ? (f4)*(const f4u *)(src + d) : f4{0.f, 0.f, 0.f, 0.f};
            v[j] = on ? (f4)*(const f4u *)(src + d + 4) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) big = fmaxf(big, fmaxf(fabsf(u[j][e]), fabsf(v[j][e])));
        }
        big = fmaxf(big, __shfl_xor(big, 16, 64));
        const int ex = scale_exp(fmaxf(big, __shfl_xor(big, 32, 64)));
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float z = __builtin_amdgcn_ldexpf(e < 4 ? u[j][e & 3] : v[j][e & 3], ex);
                const _Float16 hi = (_Float16)z;
                qh[j][e] = hi;
                ql[j][e] = (_Float16)(z - (float)hi);
            }
        return __builtin_amdgcn_ldexpf(LOG2E / sqrtf((float)a.head_dim), -ex);
    }
    __device__ inline void load_k(Buf kd, uint32_t row, int kq, int hd) {
#pragma unroll
        for (int j = 0; j < J; j++) k[j] = ld16(kd, 32 * j + 8 * kq < hd ? row + 64u * j + 16u * (uint32_t)kq : 0x7FFFFF00u);
    }
    __device__ inline v4f scores() const {
        v4f s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const h8 y = __builtin_bit_cast(h8, k[j]);
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qh[j], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ql[j], s1, 0, 0, 0);
        }
        return s0 + s1;
    }
};

/* V of a lane's position: HD / 16 dims; dim(i, t) is the t-th of lane i % 16 */
template <typename T, int HD>
struct NarrowV {
    static constexpr int N = HD / 16;
    u32x4 v[N / 4];
    static __device__ inline int dim(int i, int t) { return 64 * (t >> 2) + 4 * i + (t & 3); }
    __device__ inline void load(Buf vd, uint32_t row, int i, int hd) {
#pragma unroll
        for (int n = 0; n < N / 4; n++) v[n] = ld16(vd, 64 * n + 4 * i < hd ? row + 256u * n + 16u * (uint32_t)i : 0x7FFFFF00u);
    }
    __device__ inline float at(int t) const { return __uint_as_float(v[t >> 2][t & 3]); }
};
template <int HD>
struct NarrowV<_Float16, HD> {
    static constexpr int N = HD / 16;
    typedef _Float16 H __attribute__((ext_vector_type(N)));
    H v;
    static __device__ inline int dim(int i, int t) { return N * i + t; }
    __device__ inline void load(Buf vd, uint32_t row, int i, int hd) {
        const uint32_t at = N * i < hd ? row + 2u * N * (uint32_t)i : 0x7FFFFF00u;
        if constexpr (N == 8) v = __builtin_bit_cast(H, ld16(vd, at));
        else v = __builtin_bit_cast(H, ld8(vd, at));
    }
    __device__ inline float at(int t) const { return (float)v[t]; }
};

template <int HD, int NW>
struct SharedN {
    __attribute__((aligned(16))) float mo[NW][MN][HD];
    float mm[NW][MN], ml[NW][MN];
    uint32_t bad_rows;
};
/* m-rows `from` .. from + 15 of the work's tile, by all NW waves of the workgroup */
template <typename T, int HD, int NW>
__device__ inline __attribute__((always_inline)) void rows_n(const PromptArgs &a, const RowsPlan &p, const Work &w, int from,
                                                             SharedN<HD, NW> &sh) {
    constexpr int N = HD / 16;
    auto &mo = sh.mo;
    auto &mm = sh.mm;
    auto &ml = sh.ml;
    auto &bad_rows = sh.bad_rows;
    const int ratio = a.n_heads / a.n_kv, hd = a.head_dim;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, kq = lane >> 4;
    const Lane x = lane_rows(a, w, from, c16, 16, ratio);
    if (tid == 0) bad_rows = 0;

    const uint32_t rb = (uint32_t)hd * (uint32_t)sizeof(T);
    const Buf kd = make_buf_uniform(region<T>(a, w, a.kv_k, a.pre_k), (uint32_t)w.hi * rb);
    const Buf vd = make_buf_uniform(region<T>(a, w, a.kv_v, a.pre_v), (uint32_t)w.hi * rb);
    NarrowK<T, HD> K;
    NarrowV<T, HD> V[4];
    auto load_v = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) V[i].load(vd, (uint32_t)(t0 + 4 * kq + i) * rb, c16, hd);
    };
    int t = w.lo + 16 * wave;
    K.load_k(kd, (uint32_t)(t + c16) * rb, kq, hd);   /* past the span: zeros, no memory access */
    load_v(t);
    const float c = K.load_q(a, x, kq);
    float mx = -INFINITY, l = 0.f;
    v4f o[N];
#pragma unroll
    for (int n = 0; n < N; n++) o[n] = v4f{0.f, 0.f, 0.f, 0.f};
    for (; t < w.hi; t += 16 * NW) {
        v4f s = K.scores();
        K.load_k(kd, (uint32_t)(t + 16 * NW + c16) * rb, kq, hd);
        const bool masked = t + 15 > x.all_hi || t < x.all_lo;   /* uniform */
        float top = -INFINITY;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int pos = t + 4 * kq + v;
            if (masked) s[v] = pos <= x.last && pos >= x.first ? s[v] : -INFINITY;
            top = fmaxf(top, s[v]);
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64)) * c;
        const float mn = fmaxf(mx, top), base = mn == -INFINITY ? 0.f : mn;
        if (__any(mn > mx)) {
            const float alpha = __builtin_amdgcn_exp2f(mx - base);
            l *= alpha;
#pragma unroll
            for (int n = 0; n < N; n++) o[n] *= alpha;
        }
        mx = mn;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], c, -base));
            l += s[v];
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < N; n++) o[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(V[i].at(n), s[i], o[n], 0, 0, 0);
        load_v(t + 16 * NW);
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
        for (int n = 0; n < N; n += 4) {
            const int d = NarrowV<T, HD>::dim(4 * kq + v, n);   /* the next three follow */
            *(f4 *)&mo[wave][c16][d] = f4{o[n][v], o[n + 1][v], o[n + 2][v], o[n + 3][v]};
        }
    if (kq == 0) mm[wave][c16] = mx, ml[wave][c16] = l;
    __syncthreads();
    /* the waves' sums as one, in wave order: 16 threads a row, HD / 16 dims each */
    const bool on = tid < 16 * MN;
    const int row = (tid >> 4) & (MN - 1), d0 = (tid & 15) * N;
    const Lane y = lane_rows(a, w, from, row, 16, ratio);
    float M = mm[0][row];
#pragma unroll
    for (int q = 1; q < NW; q++) M = fmaxf(M, mm[q][row]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, r[N];
#pragma unroll
    for (int n = 0; n < N; n++) r[n] = 0.f;
#pragma unroll
    for (int q = 0; q < NW; q++) {
        const float e = __builtin_amdgcn_exp2f(mm[q][row] - base);
        L = fmaf(ml[q][row], e, L);
#pragma unroll
        for (int n = 0; n < N; n++) r[n] = fmaf(mo[q][row][d0 + n], e, r[n]);
    }
    float nan = L * 0.f;
#pragma unroll
    for (int n = 0; n < N; n++) nan = fmaf(r[n], 0.f, nan);
    if (on && y.live && !(nan == 0.f)) atomicOr(&bad_rows, 1u << row);
    __syncthreads();
    const uint32_t bad = bad_rows;
    if (on && y.live && !((bad >> row) & 1u) && d0 < hd) {
        float *dst, f = 1.f;
        if (p.nrec) {
            const size_t rec = ((size_t)y.r * a.n_heads + y.h) * p.nrec + w.rec;
            if (d0 == 0) write_ml(p, w, rec, M, L);
            dst = p.o + rec * hd + d0;
        } else {
            if (a.sinks) {
                const float sk = a.sinks[y.h] * LOG2E, mn = fmaxf(M, sk), b2 = mn == -INFINITY ? 0.f : mn;
                f = exp2f(M - b2);
                L = L * f + exp2f(sk - b2);
            }
            f /= L;
            dst = a.out + (size_t)y.r * a.out_stride + (size_t)y.h * hd + d0;
        }
        if (!p.nrec || M > -INFINITY) {
#pragma unroll
            for (int n = 0; n < N; n += 4) *(f4u *)(dst + n) = f4{r[n] * f, r[n + 1] * f, r[n + 2] * f, r[n + 3] * f};
        }
    }
    for (uint32_t z = bad; z; z &= z - 1) slow_row<T>(a, p, w, from + __builtin_ctz(z), ratio, &mo[0][0][0]);
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void k_rows_n(PromptArgs a, RowsPlan p) {
    __shared__ SharedN<HD, 4> sh;
    Work w;
    if (find_work<MN>(a, p, a.n_heads / a.n_kv, w)) rows_n<T, HD, 4>(a, p, w, 0, sh);
}

/* ---- float32 caches on the f16 matrix units ----
 *
 * The same products with K and V split as q and the weights are: x 2^k = hi +
 * lo, 22 bits, and three MFMAs a product (hi hi, hi lo, lo hi; lo lo is below
 * 2^-22).  k is chosen for each group of 8 positions from its largest finite
 * magnitude: a value down to 2^-17 of that keeps 22 bits, a smaller one is off
 * by 2^-39 of it.  (f32 MFMAs run at a sixteenth of the f16 rate, three bf16
 * planes would take six products.)
 *
 * A group is one wave's share of a tile's loads, and positions 8 g .. 8 g + 7
 * are registers 4 g .. 4 g + 3 of the scores in both halves of the wave: K's
 * scale only changes the factor to base 2.  V's groups have scales of their
 * own; o is in units of 2^-U, U the smallest k so far, and a group's weights
 * take 2^(U - k), which is part of their exponent and taken back in their sum.
 *
 * What a position holds must not cost the others their precision, the less so
 * where a row does not see it, and a channel that is large throughout not
 * that of the others, which are outputs of their own (V) or all that counts
 * where q is small in it (K).  So the positions of a group may differ by
 * 2^SPREAD in their largest magnitudes (zeros aside), its channels too (then a
 * value is off by 2^-27 of its channel's largest in the group at most; fewer
 * positions than 8, the last of a span, have small values by chance and are not
 * asked, unless they are all there is), and so may the groups of V; where
 * they differ by more, or a group that is not all zeros lies below 2^-85, the
 * workgroup's rows are computed as few rows are, with f32 products (rows_n), 16
 * at a time (1,000 rows of 32 heads of 128: 254 us instead of 51; value by
 * value 19,400).
 *
 * A tile of 32 positions is loaded into registers two tiles ahead, split and
 * stored to one of two LDS buffers one tile ahead (plane [K hi, K lo, V hi,
 * V lo][32][HD]).
 *
 * Bound: the matrix units and the splitting beside them.  500 rows of 64 heads
 * of 64 behind 30,001 positions: 793 us, 0.94 PFLOP/s counting the three
 * products, 77% of a large f16 product's rate; 2,020 packed rows of 32 heads
 * of 128: 59 us, where the longest sequence's last tiles are most of it. */
constexpr int KF = 32, SPREAD = 12;
constexpr int ALL_ZERO = 100;   /* exponent of a group of zeros; the others' is less */
/* scale_exp of a group's largest magnitude, as its word; a word below 42 << 23,
 * less one step, is below 2^-85 and its exponent would not be */
__device__ inline int group_exp(uint32_t bits) { return 141 - (int)(bits >> 23); }
constexpr uint32_t TOO_LOW = ((uint32_t)(142 - ALL_ZERO) << 23) - 1u;

/* The kernel's arguments read again, for what is hardly ever done: kept from
 * the start of the kernel, they took scalar registers that the loop needs. */
struct RowsKernelArgs {
    PromptArgs a;
    RowsPlan p;
};
__device__ inline RowsKernelArgs kernel_args() {
    struct Words {
        uint32_t w[sizeof(RowsKernelArgs) / 4];
    } k;
    auto at = (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
    asm("" : "+s"(at));
#pragma unroll
    for (unsigned i = 0; i < sizeof k / 4; i++) k.w[i] = at[i];
    return __builtin_bit_cast(RowsKernelArgs, k);
}

/* the largest of the HD / 4 lanes that hold a position, and of the lanes HD / 4
 * apart, which hold the same dims */
__device__ inline uint32_t swap_umax(uint32_t v, bool rows) {
    const auto r = rows ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}
template <int HD>
__device__ inline uint32_t row_umax(uint32_t v) {
    v = max(v, (uint32_t)dpp_i<0xB1>((int)v));
    v = max(v, (uint32_t)dpp_i<0x4E>((int)v));
    v = max(v, (uint32_t)dpp_i<0x141>((int)v));
    v = max(v, (uint32_t)dpp_i<0x140>((int)v));
    return HD == 128 ? swap_umax(v, true) : v;
}
template <int HD>
__device__ inline uint32_t dim_umax(uint32_t v) {
    v = swap_umax(v, false);
    return HD == 64 ? swap_umax(v, true) : v;
}

template <int HD, int MW, int KG>
struct SharedF {
    __attribute__((aligned(1024))) uint8_t bufs[KG][2][4][KF * HD * 2];
    int exps[KG][2][8];
    int range[MW * KG][2];   /* each wave's least and most */
    uint32_t bad_rows[MW];
    long long where[KG == 2 ? 32 * MW : 1];
};
template <int HD, int MW, int KG>
__device__ inline __attribute__((always_inline)) void rows_f(const PromptArgs &a, const RowsPlan &p, SharedF<HD, MW, KG> &sh,
                                                             SharedN<HD, MW * KG> &shn) {
    constexpr int RB = HD * 2, PLANE = KF * RB;
    constexpr int UNITS = 8 / MW;                    /* groups a wave loads: K 0 .. 3, V 4 .. 7 */
    constexpr int LR = 256 / HD, NL = 8 / LR;        /* rows a load of the wave covers, loads a group */
    constexpr int DB = HD / 32, STEPS = HD / 16;
    auto &bufs = sh.bufs;
    auto &range = sh.range;
    auto &bad_rows = sh.bad_rows;
    auto &where = sh.where;
    const int ratio = a.n_heads / a.n_kv, hd = a.head_dim;
    Work w;
    if (!find_work<32 * MW>(a, p, ratio, w)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, group = wave / MW, mwave = wave % MW;
    static_assert(KG == 1 || sizeof bufs >= MW * 256 * (HD / 2 + 3), "merge_groups");
    uint8_t(*buf)[4][PLANE] = bufs[group];
    int(*exps)[8] = sh.exps[group];

    /* loads: lane l of load j of group g holds dims 4 (l % (HD / 4)) .. of position 8 g + LR j + l / (HD / 4) */
    const uint32_t rb = (uint32_t)hd * 4u;
    const float *kp = region<float>(a, w, a.kv_k, a.pre_k), *vp = region<float>(a, w, a.kv_v, a.pre_v);
    const Buf kd = make_buf_uniform(UNITS == 2 || mwave < 4 ? kp : vp, (uint32_t)w.hi * rb);   /* of the first unit */
    const Buf vd = make_buf_uniform(vp, (uint32_t)w.hi * rb);
    const int lrow = lane / (HD / 4), ldim = 4 * (lane % (HD / 4));
    const uint32_t loff = ldim < hd ? (uint32_t)lrow * rb + 4u * (uint32_t)ldim : 0x7FFFFF00u;
    u32x4 raw[UNITS][NL];
    auto load_tile = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int g = u * MW + mwave;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const uint32_t at = loff + (uint32_t)(t0 + 8 * (g & 3) + LR * j) * rb;
                raw[u][j] = ld16(u == 0 ? kd : vd, at);
            }
        }
    };
    const uint64_t padding = __ballot(ldim >= hd);
    /* Of the wave's groups the least magnitude but zeros, less one step (zeros
     * become the largest word), and V's largest; 0: a group that no scale serves */
    uint32_t lowest[UNITS], highest = 0;
#pragma unroll
    for (int u = 0; u < UNITS; u++) lowest[u] = ~0u;
    bool few = false;   /* some group's channels differ, perhaps one of less than 8 positions */
    auto split_tile = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UNITS; u++) {
            const int g = u * MW + mwave;
            float top[NL], col[4] = {0.f, 0.f, 0.f, 0.f}, big = 0.f;   /* of the lane's positions, of its dims */
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const f4 y = __builtin_bit_cast(f4, raw[u][j]);
                top[j] = max_nan(max_nan(max_nan(fabsf(y[0]), fabsf(y[1])), fabsf(y[2])), fabsf(y[3]));
                big = max_nan(big, top[j]);
#pragma unroll
                for (int e = 0; e < 4; e++) col[e] = max_nan(col[e], fabsf(y[e]));
            }
            uint32_t bits = wave_umax(__float_as_uint(big));
            if (__builtin_expect(bits >= 0x7F800000u, 0)) {   /* uniform: the largest of the finite ones */
                uint32_t fin = 0, of_col[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < NL; j++) {
                    uint32_t of_row = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t y = raw[u][j][e] & 0x7FFFFFFFu;
                        y = y < 0x7F800000u ? y : 0u;
                        of_row = max(of_row, y), of_col[e] = max(of_col[e], y);
                    }
                    top[j] = __uint_as_float(of_row);
                    fin = max(fin, of_row);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) col[e] = __uint_as_float(of_col[e]);
                bits = wave_umax(fin);
            }
            const int ex = min(group_exp(bits), ALL_ZERO);
            /* every position and every channel come near the largest: mostly
             * in each lane's share of each, else it takes one lane of a position
             * or channel, or zeros */
            const float near = __uint_as_float(bits > ((uint32_t)SPREAD << 23) ? bits - ((uint32_t)SPREAD << 23) : 0u);
            float low = top[0];
#pragma unroll
            for (int j = 1; j < NL; j++) low = __builtin_elementwise_minimum(low, top[j]);
#pragma unroll
            for (int e = 0; e < 4; e++) low = __builtin_elementwise_minimum(low, col[e]);
            if (__builtin_expect((__ballot(low >= near) | padding) != ~0ull, 0)) {
                bool row = true, dim = true, there = true;
#pragma unroll
                for (int j = 0; j < NL; j++) {
                    const uint32_t x = row_umax<HD>(__float_as_uint(top[j]));
                    row = row && (x == 0 || __uint_as_float(x) >= near), there = there && x != 0;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t x = dim_umax<HD>(__float_as_uint(col[e]));
                    dim = dim && (x == 0 || __uint_as_float(x) >= near);
                }
                const bool dims = __all(dim);
                if (!__all(row) || (!dims && __all(there))) lowest[u] = 0;
                few = few || !dims;
            }
            lowest[u] = min(lowest[u], bits - 1u);
            if (u == UNITS - 1) highest = max(highest, bits);
            const float f = __uint_as_float((uint32_t)(ex + 127) << 23);
            if (lane == 0) exps[b][g] = ex;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int key = 8 * (g & 3) + LR * j + lrow;
                const uint32_t at = (uint32_t)(key * RB + (((ldim >> 3) ^ swz<HD>(key)) << 4) + 2 * (ldim & 4));
                h4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    h2 y, z;
                    const float x0 = __uint_as_float(raw[u][j][e]), x1 = __uint_as_float(raw[u][j][e + 1]);
                    split2(x0 * f, x1 * f, x0, x1, f, y, z);
                    hi[e] = y[0], hi[e + 1] = y[1], lo[e] = z[0], lo[e + 1] = z[1];
                }
                *(h4 *)(buf[b][2 * (g >> 2)] + at) = hi;
                *(h4 *)(buf[b][2 * (g >> 2) + 1] + at) = lo;
            }
        }
    };
    const int t1 = w.lo + group * KF;   /* the group's first tile; past the span: zeros */
    load_tile(t1);
    if constexpr (KG == 2) copy_q<HD, 32 * MW>(a, w, ratio, wave, MW * KG, bufs[0][1][0], bufs[1][1][0]);
    const Lane x = lane_rows(a, w, 32 * mwave, lane & 31, 32, ratio);

    h8 qh[STEPS], ql[STEPS];
    float c;
    if constexpr (KG == 2) {
        wait_copies();
        bar_lds();
        const uint8_t *mine = bufs[mwave / (MW / 2)][1][0] + (mwave % (MW / 2) * 32 + (lane & 31)) * (HD * 4);
        c = load_q<HD>(hd, half, [&](int i) { return *(const f4 *)(mine + row_piece<HD>(lane & 31, i)); }, qh, ql);
    } else {
        c = load_q<HD>(hd, half, memory_q(a, x), qh, ql);
    }
    f16v o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[d][v] = 0.f;
    float mx = -INFINITY, l = 0.f;
    int U = ALL_ZERO;
    const float one = opaque_one();
    const uint32_t kaddr = k_operand<HD>(lane);
    uint32_t vaddr[DB][2];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 2; e++) vaddr[d][e] = 2 * PLANE + v_operand<HD>(lane, d, e);

    /* Of the two waves of a SIMD one splits its share of the next tile before
     * it computes and one behind, so that one's VALU work meets the other's
     * MFMAs (500 rows of 64-value heads behind 30,001: 821 us, both behind, and
     * 793; 4,096 rows of 128: 405 and 398).  Workgroups of four waves share
     * the SIMDs with others, whose barriers are their own. */
    const bool early = KG == 2 ? group == 1 : MW == 8 && wave >= 4;
    auto next_tile = [&](int t, int to) __attribute__((always_inline)) {
        split_tile(to);
        load_tile(t + 2 * KG * KF);
    };
    split_tile(0);
    load_tile(t1 + KG * KF);
    __syncthreads();
    int b = 0;
    for (int t0 = w.lo; t0 < w.hi; t0 += KG * KF, b ^= 1) {
        const int t = t0 + group * KF;
        const bool more = t + KG * KF < w.hi;
        if (early && more) next_tile(t, b ^ 1);
        if (t <= x.any_hi && t + KF > x.any_lo && t < w.hi) {   /* uniform in the wave */
            const Lds tile = (Lds)buf[b][0];
            const int ex = exps[b][lane & 7];
            int ke[4], ve[4];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                ke[g] = __builtin_amdgcn_readlane(ex, g);
                ve[g] = __builtin_amdgcn_readlane(ex, 4 + g);
            }
            f16v s;
#pragma unroll
            for (int v = 0; v < 16; v++) s[v] = 0.f;
            h8 kh = lds_row(tile + kaddr), kl = lds_row(tile + kaddr + PLANE);
#pragma unroll
            for (int st = 0; st < STEPS; st++) {   /* the next step's operands are read a step ahead */
                const Lds at = tile + (kaddr ^ (uint32_t)((st + 1) << 5));
                const h8 nh = st + 1 < STEPS ? lds_row(at) : kh, nl = st + 1 < STEPS ? lds_row(at + PLANE) : kl;
                s = MFMA_H(kl, qh[st], s);
                s = MFMA_H(kh, ql[st], s);
                s = MFMA_H(kh, qh[st], s);
                kh = nh, kl = nl;
            }
            auto column = [&](int i, int lo) __attribute__((always_inline)) {
                const int q = i / DB, d = i % DB, at = q * 16 * RB + lo * PLANE;
                return h8_of(lds_column(tile + vaddr[d][0] + at), lds_column(tile + vaddr[d][1] + at));
            };
            h8 vh = column(0, 0), vl = column(0, 1);
            mask_scores(s, t + 4 * half, x);
            float cg[4], top = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                /* no further down than a normal value, where every score vanishes: 0 * -inf
                 * would send the rows of a group of zeros and small q to slow_row */
                cg[g] = fmaxf(__builtin_amdgcn_ldexpf(c, -ke[g]), 0x1p-126f);
                top = max_nan(top, max_nan(max_nan(max_nan(s[4 * g], s[4 * g + 1]), s[4 * g + 2]), s[4 * g + 3]) * cg[g]);
            }
            top = other_half_max(top);
            const int un = min(min(U, min(ve[0], ve[1])), min(ve[2], ve[3]));
            if (__any(top > mx + LAG_F) || un != U) {
                const float mn = max_nan(mx, top);
                const float alpha = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
                mx = mn;
                const float beta = __builtin_amdgcn_ldexpf(alpha, un - U);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[d][v] *= beta;
            }
            U = un;
            const float sh = mx == -INFINITY ? 0.f : SHIFT_F - mx;
            /* the scheduler's order of MFMAs and exponentials: 4,096 rows 402 us without, 398; 500 behind 30,001 789 and 793 */
            __builtin_amdgcn_iglp_opt(3);
            h8 ph[2], pl[2];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int d = min(ve[g] - un, SPREAD);   /* more: zeros, or rows_n does the rows again */
                const float shg = sh - (float)d;
                float sum[2] = {0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float y0 = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], cg[g], shg));
                    const float y1 = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e + 1], cg[g], shg));
                    sum[0] += y0, sum[1] += y1;
                    h2 hi, lo;
                    split2(y0, y1, y0, y1, one, hi, lo);
                    const int at = 4 * (g & 1) + e;
                    ph[g >> 1][at] = hi[0], ph[g >> 1][at + 1] = hi[1];
                    pl[g >> 1][at] = lo[0], pl[g >> 1][at + 1] = lo[1];
                }
                l = fmaf(sum[0] + sum[1], __uint_as_float((uint32_t)(d + 127) << 23), l);
            }
#pragma unroll
            for (int i = 0; i < 2 * DB; i++) {
                const h8 nh = i + 1 < 2 * DB ? column(i + 1, 0) : vh, nl = i + 1 < 2 * DB ? column(i + 1, 1) : vl;
                const int q = i / DB, d = i % DB;
                o[d] = MFMA_H(vl, ph[q], o[d]);
                o[d] = MFMA_H(vh, pl[q], o[d]);
                o[d] = MFMA_H(vh, ph[q], o[d]);
                vh = nh, vl = nl;
            }
        }
        if (!early && more) next_tile(t, b ^ 1);
        bar_lds();
    }
    int least = ALL_ZERO, most = -2 * ALL_ZERO;   /* exponents of the wave's groups of V; 1000: rows_n's rows */
    if (UNITS == 2 || mwave >= 4) {
        if (highest) least = group_exp(highest), most = group_exp(lowest[UNITS - 1] + 1u);
    }
#pragma unroll
    for (int u = 0; u < UNITS; u++)
        if (lowest[u] < TOO_LOW || (few && w.hi - w.lo < 8)) most = 1000;
    if (lane == 0) range[wave][0] = least, range[wave][1] = most;
    __syncthreads();
    for (int v = 0; v < MW * KG; v++) least = min(least, range[v][0]), most = max(most, range[v][1]);
    if (most - least > SPREAD) {
        const RowsKernelArgs k = kernel_args();
        Work v;
        if (!find_work<32 * MW>(k.a, k.p, k.a.n_heads / k.a.n_kv, v)) return;
        for (int from = 0; from < 32 * MW; from += MN) {
            int i, j;
            v.row(from, k.a.n_heads / k.a.n_kv, i, j);
            if (i >= v.sq.n) return;
            __syncthreads();
            rows_n<float, HD, MW * KG>(k.a, k.p, v, from, shn);
        }
        return;
    }
    l = other_half_sum(l);
    if (KG == 2 && w.hi - w.lo > KF) merge_groups<HD, MW>((float *)bufs, wave, lane, mx, l, U, o);
    else __syncthreads();   /* one group, or the second had no tile: all are done with the tiles */
    constexpr int STRIDE = 64 * (HD / 2 + 3) * 4;   /* a wave's share of merge_groups' room */
    if (group == 0) {
        const uint32_t bad = write_rows<HD, true>(a, p, w, x, lane, mx, l, U, o, KG == 2 ? (uint8_t *)bufs + wave * STRIDE : nullptr,
                                                  where + (KG == 2 ? 32 * wave : 0));
        if (lane == 0) bad_rows[wave] = bad;
    }
    __syncthreads();
    if constexpr (KG == 2) {
        store_rows<HD, 32 * MW>(hd, (const uint8_t *)bufs, STRIDE, where, p.nrec ? p.o : a.out, wave, MW * KG);
        __syncthreads();
    }
    for (int wv = 0; wv < MW; wv++)
        for (uint32_t y = bad_rows[wv]; y; y &= y - 1)
            slow_row<float>(a, p, w, 32 * wv + __builtin_ctz(y), ratio, (float *)bufs);
}

template <int HD, int MW, int KG>
__global__ __launch_bounds__(64 * MW * KG, 2) void k_rows_f(PromptArgs a, RowsPlan p) {
    __shared__ union {
        SharedF<HD, MW, KG> f;
        SharedN<HD, MW * KG> n;
    } sh;
    rows_f<HD, MW, KG>(a, p, sh.f, sh.n);
}

/* A prefix's tiles of 128 m-rows and the sequences' of 16 in one launch: a CU
 * takes a workgroup of each, so that the products of the ones, which run at
 * the power limit, pass while the others wait for their caches. */
template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void k_rows_both(PromptArgs a, RowsPlan p) {
    constexpr bool HALF = sizeof(T) == 2;
    __shared__ union {
        std::conditional_t<HALF, SharedH<HD, 4, 1>, SharedF<HD, 4, 1>> wide;
        SharedN<HD, 4> narrow;
    } sh;
    if ((int)blockIdx.x < p.pre_tiles * p.pre_ns * a.n_kv) {
        if constexpr (HALF) rows_h<HD, 4, 1, 2>(a, p, sh.wide);
        else rows_f<HD, 4, 1>(a, p, sh.wide, sh.narrow);
        return;
    }
    Work w;
    if (find_work<MN>(a, p, a.n_heads / a.n_kv, w)) rows_n<T, HD, 4>(a, p, w, 0, sh.narrow);
}

/* The records of a row and head, and its sink, as one: W waves each, wave g
 * the records g (mod W), G lanes a record (four dims a lane), N records of a
 * lane's loads at a time.  1,536 rows of 25
 * records of 128 values, 20 MB: 7.4 us with four waves; few rows 3 - 4 us, the
 * launch and two memory round trips. */
template <int W, int G, int N>
__global__ __launch_bounds__(256) void k_rows_combine(PromptArgs a, RowsPlan p) {
    __shared__ __attribute__((aligned(16))) float so[W > 1 ? W : 1][4 * G];
    __shared__ float sl[W];
    constexpr int PER = 64 / G;   /* records a wave reads at a time */
    const int tid = threadIdx.x, lane = tid & 63, wave = W > 1 ? tid >> 6 : 0, hd = a.head_dim;
    const long long at = W > 1 ? (long long)blockIdx.x : (long long)blockIdx.x * 4 + (tid >> 6);
    if (at >= (long long)a.s.rows * a.n_heads) return;
    const int r = (int)(at / a.n_heads), h = (int)(at - (long long)r * a.n_heads);
    const float *ml = p.ml + 4 * (size_t)at * p.nrec, *po = p.o + (size_t)at * p.nrec * hd;
    const int g = lane / G, d = 4 * (lane % G);
    /* lane i holds record W i + wave of each 64 W.  The first ones' statistics
     * and sums are read before it is known that they are there (there is room
     * for them), so that nothing waits for the row's sequence. */
    f4 stat = {-INFINITY, 0.f, 0.f, 0.f}, y[N];
    if (W * lane + wave < p.nrec) stat = *(const f4 *)(ml + 4 * (W * lane + wave));
    float m0 = -INFINITY, m1 = -INFINITY;   /* at most 128 records (rows_cut) */
    if (lane < p.nrec) m0 = ml[4 * lane];
    if (lane + 64 < p.nrec) m1 = ml[4 * (lane + 64)];
    const int count = __float_as_int(ml[4 * p.pre_ns + 2]);
    auto load = [&](int c0, int j0) {
#pragma unroll
        for (int q = 0; q < N; q++) {
            const int c = c0 + W * (j0 + q * PER + g) + wave;
            y[q] = f4{0.f, 0.f, 0.f, 0.f};
            if (c < p.nrec && d < hd) y[q] = *(const f4 *)(po + (size_t)c * hd + d);
        }
    };
    load(0, 0);
    Seq sq;
    int i;
    if (!wave_seq_of(a.s, r, sq, i)) return;
    const float sink = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
    const int nrec = min(p.pre_ns + max(count, 0), p.nrec);   /* the prefix's records and the tile's own */
    const float M = fmaxf(wave_max(fmaxf(lane < nrec ? m0 : -INFINITY, lane + 64 < nrec ? m1 : -INFINITY)), sink);
    const float base = M == -INFINITY ? 0.f : M;
    float l = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = 0; c0 < nrec; c0 += 64 * W) {
        const int c = c0 + W * lane + wave;
        if (c0 && c < p.nrec) stat = *(const f4 *)(ml + 4 * c);
        /* -1: a record of no position, whose sums are not written */
        const float e = c < nrec && stat[0] != -INFINITY ? exp2f(stat[0] - base) : -1.f;
        l += e < 0.f ? 0.f : stat[1] * e;
        const int n = min(64, (nrec - c0 - wave + W - 1) / W);
        for (int j0 = 0; j0 < n; j0 += N * PER) {
            if (c0 + j0) load(c0, j0);
#pragma unroll
            for (int q = 0; q < N; q++) {
                const int j = j0 + q * PER + g;
                const float f = __shfl(e, j & 63, 64);
                if (j < n && !(f < 0.f)) o += y[q] * f;
            }
        }
    }
    l = wave_sum(l);
#pragma unroll
    for (int q = 32; q >= G; q >>= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += __shfl_xor(o[e], q, 64);
    if constexpr (W > 1) {
        if (lane < G) *(f4 *)&so[wave][4 * lane] = o;
        if (lane == 0) sl[wave] = l;
        __syncthreads();
        if (wave) return;
        if (lane < G) {
#pragma unroll
            for (int q = 1; q < W; q++) {
                o += *(const f4 *)&so[q][4 * lane];
                l += sl[q];
            }
        }
    }
    if (lane >= G || d >= hd) return;
    if (a.sinks) l += exp2f(sink - base);
    *(f4u *)(a.out + (size_t)r * a.out_stride + (size_t)h * hd + d) = o * (1.f / l);
}

/* How a call is cut, from the host's arguments alone (the lengths are on the
 * device).  Each part, the sequences' slots and the prefix, has a shape:
 *   narrow  16 m-rows a workgroup, positions over its waves
 *   wide    128 m-rows, two groups of four waves on tiles in turn: two waves
 *           a SIMD where there are few workgroups (1,024 tokens of 32 heads of
 *           128, f16 and f32: 31.9 and 52.4 us, full 36.1 and 71.6)
 *   short   128 m-rows, four waves, for few positions a row (128 tokens, f16:
 *           11.6 us, wide 12.3)
 *   full    the same, two workgroups a CU on long spans (8,192 tokens, f16:
 *           883 us, wide 925; 3,000 144 and 150; 2,048 77 and 72)
 *   tall    256 m-rows, eight waves, long f32 caches: half the splitting of K
 *           and V a row (4,096 tokens: 398 us, full 466; 3,000 248 and 248) */
enum Shape { NARROW, SHORT, WIDE, FULL, TALL };
constexpr int SHAPE_ROWS[] = {16, 128, 128, 128, 256}, SHAPE_THREADS[] = {256, 256, 512, 256, 512};
struct Cut {
    RowsPlan p;
    Shape own, pre;
    bool both;   /* of different shapes, in one launch */
};
/* The shape for m m-rows (a KV head) in `seqs` sequences that see `positions`.
 * 9 rows of 8 heads on narrow and wide: 13.6 and 19.6 us behind 1,000
 * positions (f32; f16 13.2 and 16.1), 29.0 and 23.7 behind 8,000; 16
 * sequences of them behind 2,000 92 and 47 (f16 65 and 33). */
constexpr long long NARROW_WORK = 1 << 18, TALL_WORK = 512 * 4096;
constexpr int SHORT_BELOW = 512;
static Shape shape_of(long long m, long long seqs, int n_kv, int positions, bool half) {
    if (m <= 16 * seqs || (m <= 128 * seqs && m * positions <= NARROW_WORK)) return NARROW;
    if (positions < SHORT_BELOW) return SHORT;
    if (!half && m / 256 * n_kv * positions >= TALL_WORK) return TALL;
    return m / 128 * n_kv > 512 ? FULL : WIDE;
}
static Cut rows_cut(const PromptArgs &a, bool half) {
    Cut k = {};
    RowsPlan &p = k.p;
    const int n_rows = a.s.rows, n_seqs = a.s.n, n_kv = a.n_kv, head_dim = a.head_dim, kv_max = a.s.kv_max;
    const int pre_len = a.pre_len, window = a.window, ratio = a.n_heads / n_kv;
    const long long m = (long long)n_rows * ratio;
    /* Spans of a tile at `positions`: us(n) = time of a span + what the
     * records of n spans take to write and read (+ the combine's launch,
     * where it is not there anyway).  A workgroup takes 3.4 us for 128
     * positions of 128-value heads of f16 caches, 5.9 of f32 (half of that
     * for 64 values), 1.2 us for 64 on the narrow kernel; the records stream
     * at 4.5 TB/s. */
    auto slots = [](Shape s) { return s == NARROW ? 512 : 256; };   /* workgroups at once */
    /* two tiles, one of each group: 32 positions each of f32 caches (64 rows
     * behind 2,000 positions, in multiples of 128: 26.2 and 28.3 us) */
    auto unit = [&](Shape s) { return !half && s != NARROW ? 64 : 128; };
    auto spans = [&](Shape s, long long wgs, int positions, bool joined) {
        const double t = positions * (s == NARROW ? 1.2 / 64 : (half ? 3.4 : 5.9) / 128) * (head_dim > 64 ? 1 : 0.5);
        const double r = (double)m * n_kv * head_dim * 8 / 4.5e6;
        const int most = (int)std::min<long long>({64, (positions + unit(s) - 1) / unit(s), std::max(1ll, slots(s) / wgs)});
        auto us = [&](int n) { return t / n + r * n + (joined || n == 1 ? 0 : 4) - (joined || n > 1 ? 0 : r); };
        const int n = std::max(1, std::min(most, (int)std::sqrt(t / r)));   /* the best, or the next */
        const int best = n < most && us(n + 1) < us(n) ? n + 1 : n;
        return us(best) < us(1) ? best : 1;
    };
    auto tiles = [&](Shape s, long long seqs) { return std::max((m + SHAPE_ROWS[s] - 1) / SHAPE_ROWS[s], seqs); };
    auto sees = [&](int rows) { return window > 0 ? (int)std::min<long long>(kv_max, (long long)window + rows / ratio + 1) : kv_max; };
    k.own = shape_of(m, n_seqs, n_kv, sees(128), half);
    const int own_sees = sees(SHAPE_ROWS[k.own]);
    const long long own_tiles = tiles(k.own, n_seqs);
    p.cap = spans(k.own, own_tiles * n_kv, own_sees, pre_len > 0);
    p.target = std::max(1, slots(k.own) / n_kv);
    p.unit = unit(k.own);
    if (n_seqs > 1 && p.cap > 1)   /* room for a sequence much longer than the others */
        p.cap = (int)std::min<long long>({64, (own_sees + p.unit - 1) / p.unit, std::max<long long>(4ll * p.cap, 4ll * p.target / own_tiles)});
    /* 256, 512 and 1,024 rows of as many sequences behind 100 positions, in us:
     * counted 20.2, 46.1 and 110, searched 22.5, 39.7 and 71 (the places that
     * sequences leave over are workgroups with nothing to do) */
    p.search = p.cap == 1 && n_seqs > 256;
    p.items = p.search ? (int)(m / SHAPE_ROWS[k.own]) + n_seqs
                       : (int)std::min(m / SHAPE_ROWS[k.own] + n_seqs, m) + (p.cap > 1 ? p.target : 0);
    if (pre_len) {
        k.pre = shape_of(m, 1, n_kv, pre_len, half);
        p.pre_tiles = (int)tiles(k.pre, 1);
        p.pre_unit = unit(k.pre);
        p.pre_ns = spans(k.pre, (long long)p.pre_tiles * n_kv, pre_len, true);
        /* In us, two launches and one: 48 rows behind 8,000 positions and up to
         * 500 of their own, 4 KV heads of 128, 44.2 and 33.9 (f16), 55.7 and
         * 48.4 (f32).  With f32 caches the prefix's part alone is slower in this
         * form, which shows where it is most of the work: 24 rows behind 20,000
         * and 30 of their own 56.6 and 68.5. */
        k.both = k.own == NARROW && k.pre != NARROW && k.pre != TALL &&
                 (half || 2ll * n_seqs * own_sees >= (long long)p.pre_tiles * pre_len);
    }
    p.nrec = p.cap + p.pre_ns > 1 ? p.cap + p.pre_ns : 0;
    return k;
}

static size_t ml_bytes(const RowsPlan &p, int n_rows, int n_heads) {
    return ((size_t)n_rows * n_heads * p.nrec * 16 + 255) & ~(size_t)255;
}

static size_t scratch_bytes(const RowsPlan &p, int n_rows, int n_heads, int head_dim) {
    return p.nrec ? ml_bytes(p, n_rows, n_heads) + (size_t)n_rows * n_heads * p.nrec * head_dim * 4 : 0;
}

/* For every call of at most these sizes, so that a program's one allocation
 * serves a prompt and the decode steps behind it: fewer rows are cut into more
 * spans, and what a call needs does not rise with its rows.  Tiles of a shape
 * are cut only while their spans, with those of the other tiles, are at most
 * the workgroups that run at once; of several sequences, four times as many.  So
 * the m-rows times their spans are at most the m-rows of so many tiles. */
size_t attention_rows_scratch(int n_rows, int n_seqs, int n_heads, int n_kv, int head_dim, int kv_max, int pre_len) {
    const long long m = (long long)n_rows * (n_heads / n_kv), row_heads = (long long)n_rows * n_heads;
    auto cut = [&](int positions, int times) {   /* records of a part that is cut */
        const long long spans = std::min(64, (positions + 63) / 64);
        const bool tall = m / 256 * n_kv * positions >= TALL_WORK;
        return spans == 1 ? 0 : std::min(row_heads * spans, (m <= 16 ? 16ll * 512 : tall ? 256ll * 256 : 128ll * 256) * times);
    };
    long long records = cut(kv_max, n_seqs > 1 ? 4 : 1);
    if (pre_len) records = std::max(records, row_heads) + std::max(cut(pre_len, 1), row_heads);
    return records ? (size_t)records * (16 + 4 * (size_t)head_dim) + 256 : 0;
}

/* the workgroups of one part, or of both */
template <int HD>
static void launch_part(const PromptArgs &a, const RowsPlan &p, bool half, Shape s, hipStream_t st) {
    const dim3 grid((unsigned)((p.items + p.pre_tiles * p.pre_ns) * a.n_kv)), block(SHAPE_THREADS[s]);
    if (!grid.x) return;
#define ROWS(...) hipLaunchKernelGGL((__VA_ARGS__), grid, block, 0, st, a, p)
    if (half) {
        if (s == NARROW) ROWS(k_rows_n<_Float16, HD>);
        else if (s == SHORT) ROWS(k_rows_h<HD, 4, 1, 1>);
        else if (s == WIDE) ROWS(k_rows_h<HD, 4, 2, 2>);
        else ROWS(k_rows_h<HD, 4, 1, 2>);
    } else {
        if (s == NARROW) ROWS(k_rows_n<float, HD>);
        else if (s == WIDE) ROWS(k_rows_f<HD, 4, 2>);
        else if (s == TALL) ROWS(k_rows_f<HD, 8, 1>);
        else ROWS(k_rows_f<HD, 4, 1>);
    }
#undef ROWS
}

template <int HD>
static void launch_rows(const PromptArgs &a, const Cut &k, bool half, void *scratch, hipStream_t st) {
    RowsPlan p = k.p;
    p.ml = (float *)scratch;
    p.o = (float *)((uint8_t *)scratch + ml_bytes(p, a.s.rows, a.n_heads));
    if (k.both) {
        const dim3 grid((unsigned)((p.items + p.pre_tiles * p.pre_ns) * a.n_kv));
        if (half) hipLaunchKernelGGL((k_rows_both<_Float16, HD>), grid, dim3(256), 0, st, a, p);
        else hipLaunchKernelGGL((k_rows_both<float, HD>), grid, dim3(256), 0, st, a, p);
    } else if (p.pre_tiles && k.own != k.pre) {
        RowsPlan one = p;
        one.items = 0;
        launch_part<HD>(a, one, half, k.pre, st);
        one = p;
        one.pre_tiles = 0;
        launch_part<HD>(a, one, half, k.own, st);
    } else {
        launch_part<HD>(a, p, half, k.own, st);
    }
    if (!p.nrec) return;
    const long long rows = (long long)a.s.rows * a.n_heads;
    const dim3 four((unsigned)((rows + 3) / 4));
    if (p.nrec > 16) hipLaunchKernelGGL((k_rows_combine<4, HD / 4, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, p);
    else if (p.nrec > 256 / HD) hipLaunchKernelGGL((k_rows_combine<1, HD / 4, 4>), four, dim3(256), 0, st, a, p);
    else hipLaunchKernelGGL((k_rows_combine<1, HD / 4, 1>), four, dim3(256), 0, st, a, p);
}

size_t attention_rows_need(const PromptArgs &a, bool half) {
    return scratch_bytes(rows_cut(a, half).p, a.s.rows, a.n_heads, a.head_dim);
}

void launch_attention_rows(const PromptArgs &a, bool half, void *scratch, hipStream_t st) {
    const Cut k = rows_cut(a, half);
    if (a.head_dim > 64) launch_rows<128>(a, k, half, scratch, st);
    else launch_rows<64>(a, k, half, scratch, st);
}

}  // namespace tg
