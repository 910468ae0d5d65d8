/*
 * tg_paged.hip -- caches of signed bytes in pages: rows of several sequences
 * into them, back out, and attention over them.
 *
 * A value is n 2^e: n a byte, e one exponent for a block of 16 positions of a
 * KV head, for K and V each.  A block's exponent rises when a later row needs
 * more, which re-rounds the rows that it holds; a power of two doubles at
 * least, so that all of a value's roundings together are off by at most one
 * step of the last unit (an arbitrary scale that creeps up could add half a
 * step each time), and applying it is exact.
 *
 *   append     K and V of each row, normed and turned, into its page
 *              (k_paged_append)
 *   read       positions as f32 or f16, into slots of a dense cache
 *              (k_paged_read)
 *   attention  the formulas of tg_prompt.hip; kernels by sizes (paged_cut):
 *              k_paged_n   16 query rows of a KV head a workgroup
 *              k_paged_w   128
 */
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "tg_paged.h"
#include "tg_rows.hpp"
#include "tg_turn.hpp"

namespace tg {

namespace {

/* Place of block j of sequence s and KV head kh among all blocks of the
 * pages (< 2^31); -1: no page */
__device__ inline int block_at(const Pages &p, int n_kv, int s, int kh, int j) {
    const int page = p.table[(size_t)s * p.stride + (j >> p.shift)];
    return (unsigned)page < (unsigned)p.n_pages ? ((page * n_kv + kh) << p.shift) + (j & ((1 << p.shift) - 1)) : -1;
}
__device__ inline bool good_exp(int byte) { return (unsigned)(byte - (127 + PAGE_EXP_MIN)) <= (unsigned)(PAGE_EXP_MAX - PAGE_EXP_MIN); }
/* 2^(byte - 127) and 2^(127 - byte) */
__device__ inline float exp_up(int byte) { return __int_as_float(byte << 23); }
__device__ inline float exp_down(int byte) { return __int_as_float((254 - byte) << 23); }

/* sum over groups of G lanes (8 or 16), in each of them */
template <int CTRL>
__device__ inline double dpp_d(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)dpp_i<CTRL>((int)(u >> 32)) << 32 | (uint32_t)dpp_i<CTRL>((int)(uint32_t)u)));
}
template <int G>
__device__ inline double group_sum(double v) {
    v += dpp_d<0xB1>(v);    /* lanes 1 and 2 apart, then mirrors of 8 and of 16 */
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    return G == 16 ? v + dpp_d<0x140>(v) : v;
}
/* 1 / sqrt(x): the instruction's 2^-26 or better, doubled twice by Newton's step */
__device__ inline double rsqrt_d(double x) {
    double r = __builtin_amdgcn_rsq(x);
    const double h = 0.5 * x;
    r = fma(r, fma(-h * r, r, 0.5), r);
    return fma(r, fma(-h * r, r, 0.5), r);
}

/* The least e with |x| <= 127 2^e: x = m 2^k, m in [1/2, 1), and 127 / 128 is
 * the border.  Values beyond the exponents' range, infinities and NaN
 * (which no comparison holds for) give more than PAGE_EXP_MAX. */
__device__ inline int block_exp(double big) {
    if (!(big <= 127.0 * (double)(1ll << PAGE_EXP_MAX))) return PAGE_EXP_MAX + 1;
    if (big == 0.0) return PAGE_EXP_MIN;
    const int e = __builtin_amdgcn_frexp_exp(big) - 7 + (__builtin_amdgcn_frexp_mant(big) > 127.0 / 128.0);
    return max(e, PAGE_EXP_MIN);
}

/* Where sequence s's blocks are among a call's, at most two more than n / 16
 * of its n rows touch */
__device__ inline int block_start(int r0, int s) { return (r0 >> 4) + 2 * s; }
/* the last sequence whose place is at or before b, by the whole wave */
__device__ inline bool seq_of_block(const PackedSeqs &p, int b, Seq &q, int &s, int &place) {
    const int lane = threadIdx.x & 63;
    int at = 0, count = p.n;
    while (count > 64) {
        const int step = (count + 63) / 64, t = at + min(lane * step, count - 1);
        const uint64_t m = __ballot(lane * step < count && block_start(min(max(p.cu[t], 0), p.rows), t) <= b);
        if (!m) return false;
        const int k = (63 - __builtin_clzll(m)) * step;
        at += k, count = min(step, count - k);
    }
    Seq mine = {0, 0, 0, 0};
    if (lane < count) mine = seq_at(p, at + lane);
    const uint64_t m = __ballot(lane < count && block_start(mine.r0, at + lane) <= b);
    if (!m) return false;
    const int k = 63 - __builtin_clzll(m);
    q = lane_seq(mine, k);
    s = at + k;
    place = b - block_start(q.r0, s);
    return q.n > 0;
}

/* What a wave has of a block of K or V of a head: 64 / G rows, G lanes each.
 * From the norm to the byte all is in 64 bits, so that what is stored is the
 * formula's nearest byte; the rate of 64-bit operations is half that of 32 here and
 * the kernel waits for memory. */
struct BlockRows {
    d4 x, y;
    Pieces p;
    int8_t *page;      /* the lane's row */
    uint8_t *exp;
    int old, old_rows;
    int e;             /* the exponent that the wave's rows need, NO_ROWS: it has none */
    bool live, on;
};
constexpr int NO_ROWS = -1000;
template <int G>
__device__ inline BlockRows block_rows(const PagedAppendArgs &a, const Seq &q, int s, int j, int kh, bool v, int sub) {
    const int lane = threadIdx.x & 63, row = sub * (64 / G) + lane / G, l = lane % G, hd = a.head_dim;
    BlockRows b = {};
    b.e = NO_ROWS;
    const int B = block_at(a.pages, a.n_kv, s, kh, j);
    if (B < 0) return b;
    b.on = 8 * l < hd;
    b.exp = (v ? a.pages.ev : a.pages.ek) + B;
    b.page = (v ? a.pages.v : a.pages.k) + ((size_t)B * PAGE_BLOCK + row) * hd;
    b.old_rows = max(0, min(PAGE_BLOCK, q.past - PAGE_BLOCK * j));   /* rows that the block holds */
    b.old = b.old_rows ? *b.exp : 127 + PAGE_EXP_MIN;
    Turn turn = a.turn;
    if (v) turn.cos = nullptr;
    b.p = turn_pieces(turn, l);
    const float *nw = v ? nullptr : a.k_norm;
    const int pos = PAGE_BLOCK * j + row, i = pos - q.past;
    b.live = i >= 0 && i < q.n && (!a.turn.cos || pos < a.turn.len);
    if (!__ballot(b.live)) return b;
    f4 u = {0.f, 0.f, 0.f, 0.f}, w = u, c = u, sn = u;
    if (b.live && b.on) {
        const float *src = (v ? a.v : a.k) + (size_t)(q.r0 + i) * a.kv_stride + (size_t)kh * hd;
        u = *(const f4u *)(src + b.p.a), w = *(const f4u *)(src + b.p.b);
        if (b.p.turned) {
            const size_t at = (size_t)pos * (turn.dim / 2) + 4 * l;
            c = *(const f4u *)(turn.cos + at), sn = *(const f4u *)(turn.sin + at);
        }
    }
    b.x = __builtin_convertvector(u, d4), b.y = __builtin_convertvector(w, d4);
    if (nw) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) ss += b.x[e] * b.x[e] + b.y[e] * b.y[e];
        ss = group_sum<G>(ss);
        if (b.on) {
            const double f = rsqrt_d(ss / (double)hd + (double)a.eps);
            b.x = b.x * f * __builtin_convertvector((f4)*(const f4u *)(nw + b.p.a), d4);
            b.y = b.y * f * __builtin_convertvector((f4)*(const f4u *)(nw + b.p.b), d4);
        }
    }
    if (b.p.turned) turn_pair(turn.inter, __builtin_convertvector(c, d4), __builtin_convertvector(sn, d4), b.x, b.y);
    double big = 0.0;
    bool odd = false;   /* a value that is not finite */
    if (b.live && b.on) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double f = fabs(b.x[e]), g = fabs(b.y[e]);
            odd |= !(f < INFINITY) || !(g < INFINITY);
            big = fmax(big, fmax(f, g));
        }
    }
    const int mine = odd ? PAGE_EXP_MAX + 1 : block_exp(big);
    b.e = (int)wave_umax((uint32_t)(mine - NO_ROWS)) + NO_ROWS;
    return b;
}
/* ... stored with the exponent that the rows of all waves need */
__device__ inline void store_block(const BlockRows &b, int e, int row, int l, bool first) {
    if (b.old_rows) e = max(e, good_exp(b.old) ? b.old - 127 : PAGE_EXP_MAX + 1);
    const bool bad = e > PAGE_EXP_MAX;
    if (b.on && b.live) {
        const double f = __builtin_amdgcn_ldexp(1.0, -e);
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            lo |= ((uint32_t)(int)__builtin_rint(b.x[c] * f) & 255u) << (8 * c);
            hi |= ((uint32_t)(int)__builtin_rint(b.y[c] * f) & 255u) << (8 * c);
        }
        *(uint32_t *)(b.page + b.p.a) = bad ? 0u : lo;
        *(uint32_t *)(b.page + b.p.b) = bad ? 0u : hi;
    } else if (b.on && !bad && row < b.old_rows && e > b.old - 127) {   /* rows from before in the new unit */
        const float g = exp_up(127 - (e - (b.old - 127)));
        uint32_t *at = (uint32_t *)(b.page + 8 * l);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const uint32_t w = at[c];
            uint32_t z = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) z |= ((uint32_t)(int)__builtin_rintf((float)(int8_t)(w >> (8 * k)) * g) & 255u) << (8 * k);
            at[c] = z;
        }
    }
    if (first) *b.exp = bad ? PAGE_EXP_NAN : (uint8_t)(e + 127);
}

}  // namespace

/* ---- append ----
 * Workgroups of two kinds: those of the first `rows` (0 without q_out) turn a
 * row's query heads, as k_kv_append does; the others have four waves (heads of
 * up to 64 values: two) for each block, KV head and one of K and V (all 16 rows
 * by one wave: 1,000 rows of 4 KV heads of 128 15.1 us).  Two blocks more a sequence than its rows
 * fill have room (block_start), so that no lengths are summed. */
template <int G>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendArgs a, int rows) {
    const int tid = threadIdx.x, hd = a.head_dim;
    if ((int)blockIdx.x >= rows) {
        constexpr int WAVES = PAGE_BLOCK * G / 64;   /* of a block */
        __shared__ int need[4];
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), sub = wave % WAVES, lane = tid & 63;
        const long long unit = (long long)((int)blockIdx.x - rows) * (4 / WAVES) + wave / WAVES;
        const int item = (int)(unit / (2 * a.n_kv)), rest = (int)(unit - (long long)item * (2 * a.n_kv));
        BlockRows b = {};
        b.e = NO_ROWS;
        Seq q;
        int s, place;
        if (seq_of_block(a.s, item, q, s, place)) {
            const int j = (q.past >> 4) + place;
            if (place >= 0 && PAGE_BLOCK * j < q.past + q.n) b = block_rows<G>(a, q, s, j, rest >> 1, rest & 1, sub);
        }
        if (lane == 0) need[wave] = b.e;
        __syncthreads();
        int e = NO_ROWS;
#pragma unroll
        for (int k = 0; k < WAVES; k++) e = max(e, need[wave - sub + k]);
        if (e > NO_ROWS) store_block(b, e, sub * (64 / G) + lane / G, lane % G, sub == 0 && lane == 0);
        return;
    }
    const int r = (int)blockIdx.x;
    Seq q;
    int i;
    if (!wave_seq_of(a.s, r, q, i)) return;
    const int pos = q.past + i;
    if (a.turn.cos && pos >= a.turn.len) return;
    const int seg = tid / G, l = tid % G;
    const bool on = 8 * l < hd;
    const Pieces p = turn_pieces(a.turn, l);
    f4 c = {1.f, 1.f, 1.f, 1.f}, sn = {0.f, 0.f, 0.f, 0.f};
    if (p.turned && on) {
        c = *(const f4u *)(a.turn.cos + (size_t)pos * (a.turn.dim / 2) + 4 * l);
        sn = *(const f4u *)(a.turn.sin + (size_t)pos * (a.turn.dim / 2) + 4 * l);
    }
    for (int h0 = 0; h0 < a.n_heads; h0 += 256 / G) {
        const int h = h0 + seg;
        const bool live = h < a.n_heads && on;
        const float *src = a.q + (size_t)r * a.q_stride + (size_t)h * hd;
        f4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
        if (live) x = *(const f4u *)(src + p.a), y = *(const f4u *)(src + p.b);
        if (a.q_norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
            if (on) {
                const float f = 1.f / sqrtf(ss / (float)hd + a.eps);
                x = x * f * (f4)*(const f4u *)(a.q_norm + p.a);
                y = y * f * (f4)*(const f4u *)(a.q_norm + p.b);
            }
        }
        if (!live) continue;
        if (p.turned) turn_pair(a.turn.inter, c, sn, x, y);
        float *dst = a.q_out + (size_t)r * a.q_out_stride + (size_t)h * hd;
        *(f4u *)(dst + p.a) = x;
        *(f4u *)(dst + p.b) = y;
    }
}

void launch_paged_append(const PagedAppendArgs &a, hipStream_t st) {
    const int rows = a.q_out ? a.s.rows : 0;
    const long long items = (long long)(a.s.rows >> 4) + 2ll * a.s.n;
    const int units = a.head_dim <= 64 ? 2 : 1;   /* of a workgroup */
    const dim3 grid((unsigned)(rows + (items * 2 * a.n_kv + units - 1) / units)), block(256);
    if (a.head_dim <= 64) hipLaunchKernelGGL((k_paged_append<8>), grid, block, 0, st, a, rows);
    else hipLaunchKernelGGL((k_paged_append<16>), grid, block, 0, st, a, rows);
}

/* ---- read ----
 * A block's bytes and its rows in a slot both lie in one piece, so a wave
 * turns 4 bytes a lane into 16 (8 of f16) in order, two blocks at a time: what
 * finds them takes as long as they do.  15,518 positions of 8 heads of 64 into f16
 * slots: one at a time 12.2 us, two 10.6, four 10.7; of 4 heads of 128 10.2, 10.4 and
 * 10.8.  Bound: the bytes, 4.5 to 5.2 TB/s (20,000 positions of 4 heads of 128 into f32 slots
 * 21 us). */
constexpr int READ_BLOCKS = 2;
template <typename T>
__global__ __launch_bounds__(256) void k_paged_read(PagedReadArgs a, int per) {
    typedef T V __attribute__((ext_vector_type(4)));
    constexpr int N = READ_BLOCKS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hd = a.head_dim;
    int at = blockIdx.x / per;
    const int v = at & 1, kh = (at >> 1) % a.n_kv, s = (at >> 1) / a.n_kv;
    at = blockIdx.x - at * per;
    const int len = a.len[s], slot = a.slot ? a.slot[s] : s;
    if (slot < 0 || slot >= a.n_slots || len < 0 || len > a.most) return;
    T *const to = (T *)(v ? a.v : a.k) + ((size_t)slot * a.n_kv + kh) * a.kv_max * hd;
    for (int j0 = N * (4 * at + wave); PAGE_BLOCK * j0 < len; j0 += 4 * N * per) {
        const int j = j0 + (lane & (N - 1));
        int mine = -1, exp = 0;
        if (PAGE_BLOCK * j < len) mine = block_at(a.pages, a.n_kv, s, kh, j);
        if (mine >= 0) exp = (v ? a.pages.ev : a.pages.ek)[mine];
        uint32_t w[N][8];
        int n[N];
#pragma unroll
        for (int b = 0; b < N; b++) {
            const int B = __builtin_amdgcn_readlane(mine, b);
            n[b] = min(PAGE_BLOCK, len - PAGE_BLOCK * (j0 + b)) * hd / 4;   /* words; none behind the end */
            const uint32_t *src = (const uint32_t *)((v ? a.pages.v : a.pages.k) + (size_t)max(B, 0) * PAGE_BLOCK * hd);
#pragma unroll
            for (int i = 0; i < 8; i++) w[b][i] = B >= 0 && 64 * i + lane < n[b] ? src[64 * i + lane] : 0u;
        }
#pragma unroll
        for (int b = 0; b < N; b++) {
            const int e = __builtin_amdgcn_readlane(exp, b);   /* 0 where there is no page */
            const float f = good_exp(e) ? exp_up(e) : __int_as_float(0x7FC00000);
            T *dst = to + (size_t)(PAGE_BLOCK * (j0 + b)) * hd;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (64 * i + lane < n[b]) {
                    V y;
#pragma unroll
                    for (int c = 0; c < 4; c++) y[c] = (T)((float)(int8_t)(w[b][i] >> (8 * c)) * f);
                    *(V *)(dst + 4 * (64 * i + lane)) = y;
                }
        }
    }
}

void launch_paged_read(const PagedReadArgs &a, bool half, hipStream_t st) {
    /* eight blocks a workgroup, more where the slots have room for so many that the grid would not */
    const long long heads = 2ll * a.n_kv * a.n, groups = (a.most + 4 * READ_BLOCKS * PAGE_BLOCK - 1) / (4 * READ_BLOCKS * PAGE_BLOCK);
    const int per = (int)std::max(1ll, std::min(groups, (1ll << 20) / heads));
    const dim3 grid((unsigned)(heads * per)), block(256);
    if (half) hipLaunchKernelGGL((k_paged_read<_Float16>), grid, block, 0, st, a, per);
    else hipLaunchKernelGGL((k_paged_read<float>), grid, block, 0, st, a, per);
}

/* ---- attention ----
 *
 * Weights go to the matrix units with V's power of two in them: the product
 * takes 2^(z_j + e_j - m) n_j, z_j a score in base 2, e_j the exponent of V's
 * block, and the reference m follows the largest z_j + e_j of blocks seen.
 * So whatever counts most in the output is near 1 there, however the blocks'
 * magnitudes differ, and nothing but small integers is V.  The sum l of
 * 2^(z_j - m) takes each block's sum times 2^-e_j; with exponents within
 * +-42 f32 holds both.  m is a whole number: every rescaling is exact.
 *
 * Bytes are finite, so what a row does not see meets a weight of 0 and no
 * value; rows that see a position of a block without a page, or one that
 * holds a value that was not finite, are NaN, and so are those whose query is
 * not finite (poison: l is NaN). */
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
constexpr int QMAX = 8300000;    /* three signed digits of base 256 */
constexpr float UNSHIFT = 1.f / (float)(1 << (int)SHIFT_H);
/* A score's factor c 2^e stays above 0 (-inf * 0 would be NaN): q's own power of two is at most 2^103, its f16 planes' 2^100,
 * log2 e / sqrt(head_dim) above 2^-3, and f32's least is 2^-149. */
static_assert(103 + 3 - PAGE_EXP_MIN < 149, "a score's factor");

/* A wave's next 64 blocks, one a lane: where they are, and their exponents'
 * bytes (K, V << 8) with bit 16 for one that makes rows NaN */
struct Blocks {
    int at, exps;
};
__device__ inline Blocks load_blocks(const PromptArgs &a, const Pages &p, const Work &w, int j, bool there) {
    Blocks b = {0, 127 | 127 << 8};
    if (!there) return b;
    const int B = block_at(p, a.n_kv, w.sq.slot, w.kh, j);
    if (B < 0) {
        b.exps |= 1 << 16;
        return b;
    }
    const int ek = p.ek[B], ev = p.ev[B];
    b.at = B;
    if (good_exp(ek) && good_exp(ev)) b.exps = ek | ev << 8;
    else b.exps |= 1 << 16;
    return b;
}

/* One part of a call: the sequences of at least `least` and at most `most`
 * m-rows.  Where a part's tiles are cut, spans of a dense part write records
 * as those of dense caches do, [row and head][nrec]; those of a part of a
 * mixed call [item][KV head][m-row of the tile], as only some tiles are cut
 * and it is not known which: a tile of one span writes its rows at once, and
 * where the records of the others are stands at the tile's place in `tiles`. */
struct Part {
    RowsPlan p;
    int least, most;
    struct Tile {
        int item, count, step, last;   /* of the first span; spans; from one to the next, but the last one's */
    } *tiles;                          /* null: dense */
};
struct Class {
    int least, most, ratio;
    __device__ inline void operator()(Seq &q) const {
        const int m = q.n * ratio;
        if (m < least || m > most) q.n = 0;
    }
};

/* a part of at most FEW m-rows a sequence has that many places for each */
constexpr int FEW = 128;
template <int MTILE>
__device__ inline int tile_place(const Part &pt, const Work &w, int ratio) {
    return (pt.most == FEW ? w.sq.slot * (FEW / MTILE) : start_of<MTILE>(w.sq.r0, w.sq.slot, ratio)) + w.m0 / MTILE;
}
/* Item b of a call of at most 64 sequences: as find_span, but the whole spans of
 * all tiles come first and what is left of each behind them, so that short
 * spans fill the end.  last: the item of the tile's last span. */
template <int MTILE>
__device__ inline bool find_cut(const PromptArgs &a, const RowsPlan &p, int ratio, int b, Work &w, const Class &keep, int &last) {
    const int lane = threadIdx.x & 63;
    Seq q = {0, 0, 0, 0};
    if (lane < a.s.n) q = seq_at(a.s, lane);
    keep(q);
    const int nt = div_up(q.n * ratio, MTILE), end = q.past + q.n;
    const int sees = a.window > 0 ? min(end, a.window + (MTILE - 1) / ratio + 1) : end;   /* at most */
    const float sum = wave_sum((float)nt * (float)sees);
    int per = div_up(max(1, (int)fminf(ceilf(sum / (float)p.target), 1e9f)), p.unit) * p.unit;
    if (div_up(sees, per) > p.cap) per = div_up(div_up(sees, p.cap), p.unit) * p.unit;
    const int whole_end = wave_scan(nt * (int)((unsigned)sees / (unsigned)per)), rest_end = wave_scan(nt);
    const int wholes = __builtin_amdgcn_readlane(whole_end, 63);
    const bool rest = b >= wholes;
    const int place = rest ? b - wholes : b;
    const uint64_t past = __ballot((rest ? rest_end : whole_end) > place);
    if (!past) return false;
    const int at = __builtin_ctzll(past), n = __builtin_amdgcn_readlane(nt, at);
    const int whole0 = at ? __builtin_amdgcn_readlane(whole_end, at - 1) : 0, rest0 = at ? __builtin_amdgcn_readlane(rest_end, at - 1) : 0;
    per = __builtin_amdgcn_readlane(per, at);
    w.sq = lane_seq(q, at);
    const int in = place - (rest ? rest0 : whole0);
    int split = rest ? 0 : in / n;
    const int tile = in - split * n;
    w.m0 = (n - 1 - tile) * MTILE;
    set_rows(w, ratio);
    const int lo = tile_lo(a, w), hi = tile_hi<MTILE>(w, ratio), whole = (int)((unsigned)(hi - lo) / (unsigned)per);
    const bool left = hi - lo > whole * per;
    if (rest ? !left : split >= whole) return false;
    if (rest) split = whole;
    w.rec = p.pre_ns + split;
    w.count = split ? 0 : whole + left;
    last = left ? wholes + rest0 + tile : whole0 + (whole - 1) * n + tile;
    w.lo = lo + split * per;
    w.hi = min(hi, w.lo + per);
    return true;
}

/* Item b of a call of at most 64 sequences in tiles of 128: the shortest span
 * that makes no more of them than run at once, or than half as many beyond the
 * tiles that there are anyway; a tile's spans are of one length.  Too many or
 * too uneven spans cost more than they fill: each writes 128 records.  Cut as
 * tiles of 16 are (find_cut), two sequences of 256 rows behind 15,000
 * positions took 463 us (64 + 8 heads of 64; so 276), eight single tokens and two chunks of
 * 512 behind 1,000 and 6,000 174 (32 + 4 of 128; 148), seven sequences of 1 to 1,000
 * rows as long (56). */
template <int MTILE>
__device__ inline bool find_even(const PromptArgs &a, const RowsPlan &p, int ratio, int b, Work &w, const Class &keep) {
    const int lane = threadIdx.x & 63;
    Seq q = {0, 0, 0, 0};
    if (lane < a.s.n) q = seq_at(a.s, lane);
    const int end = q.past + q.n, seen = a.window > 0 ? min(end, a.window + (MTILE - 1) / ratio + 1) : end;   /* at most */
    const float all = (float)div_up(q.n * ratio, 16) * (float)seen;
    keep(q);
    const int nt = div_up(q.n * ratio, MTILE), sees = nt ? seen : 0;
    /* Where the other part's blocks take longer to read than these tiles to compute, it gets half of the places: 60 single
     * tokens behind 2,960 positions and a chunk of 500 behind 1,500 113 us with all, 94 with half (64 + 8 heads of 64
     * 111 and 84); 31 tokens and a chunk of 512 behind 4,000 114 either way. */
    const float few = wave_sum(nt ? 0.f : all), many = wave_sum((float)nt * (float)(a.window > 0 ? sees : (q.past + end) / 2));
    const int places = few > 2.f * many ? p.target / 2 : p.target;
    const int tiles = __builtin_amdgcn_readlane(wave_scan(nt), 63), limit = max(places, tiles + places / 2);
    int lo = 0, hi = div_up((int)wave_umax((uint32_t)sees), KT);   /* per is in (lo, hi], in tiles of positions */
    while (hi - lo > 1) {
        const int per = (lo + hi) >> 1;
        const bool fits = __builtin_amdgcn_readlane(wave_scan(nt * min(div_up(sees, per * KT), p.cap)), 63) <= limit;
        hi = fits ? per : hi, lo = fits ? lo : per;
    }
    if (!hi) return false;
    const int n = max(1, min(div_up(sees, hi * KT), p.cap));
    int per = div_up(div_up(sees, n), KT) * KT;
    const int ends = wave_scan(nt * n);
    const uint64_t past = __ballot(ends > b);
    if (!past) return false;
    const int at = __builtin_ctzll(past), steps = __builtin_amdgcn_readlane(nt, at);
    const int in = b - (at ? __builtin_amdgcn_readlane(ends, at - 1) : 0), split = in / steps;
    per = __builtin_amdgcn_readlane(per, at);
    w.sq = lane_seq(q, at);
    w.m0 = (steps - 1 - (in - split * steps)) * MTILE;
    set_rows(w, ratio);
    const int first = tile_lo(a, w), last = tile_hi<MTILE>(w, ratio), count = div_up(last - first, per);
    if (split >= count) return false;
    w.rec = p.pre_ns + split;
    w.count = split ? 0 : count;
    w.lo = first + split * per;
    w.hi = min(last, w.lo + per);
    return true;
}

/* The work of item b / n_kv.  Whole blocks: a span starts at one and, but for
 * the tile's last, ends at one. */
template <int MTILE>
__device__ inline bool find_blocks(const PromptArgs &a, const Part &pt, int ratio, int b, Work &w) {
    const RowsPlan &p = pt.p;
    const int item = b / a.n_kv;
    w.prefix = false;
    w.kh = b - item * a.n_kv;
    const Class keep = {pt.least, pt.most, ratio};
    int last = -1;
    if (p.search) {
        if (!find_tile<MTILE>(a, p, ratio, item, w, keep)) return false;
    } else if (pt.tiles && MTILE == 128 && a.s.n <= 64) {
        if (!find_even<MTILE>(a, p, ratio, item, w, keep)) return false;
    } else if (p.cap > 1 && a.s.n <= 64) {
        if (!find_cut<MTILE>(a, p, ratio, item, w, keep, last)) return false;
    } else if (!find_span<MTILE>(a, p, ratio, item, w, keep)) {
        return false;
    }
    if (w.hi < tile_hi<MTILE>(w, ratio)) w.hi &= ~(PAGE_BLOCK - 1);
    w.lo &= ~(PAGE_BLOCK - 1);
    if (pt.tiles) {
        if (w.count && w.kh == 0 && threadIdx.x == 0) {
            const int n = div_up(w.sq.n * ratio, MTILE);
            pt.tiles[tile_place<MTILE>(pt, w, ratio)] = Part::Tile{item, w.count, n, last < 0 ? item + (w.count - 1) * n : last};
        }
        w.rec = item;
    }
    return true;
}
/* where m-row `at` of the tile goes: -1 straight to the output, else its record */
template <int MTILE>
__device__ inline long long record_of(const PromptArgs &a, const Part &pt, const Work &w, const Lane &x, int at) {
    if (pt.tiles) return w.count == 1 ? -1 : ((long long)w.rec * a.n_kv + w.kh) * MTILE + at;
    return pt.p.nrec ? ((long long)x.r * a.n_heads + x.h) * pt.p.nrec + w.rec : -1;
}

/* Beyond 2^24 in base 2 f32 does not hold what is added to a score or taken from it: mx + LAG_H, SHIFT_H - mx and its sum with
 * V's exponent would be rounded, by enough for weights that f16 does not hold.  Once a wave has a reference beyond FAR (all of
 * that is exact before it) each step goes where references move, and a score is replaced by its exact difference from the
 * reference, with a factor of 1 and nothing else to add but V's exponent; the largest score's own rounding adds 4 at most up to
 * BEYOND.  Past that a row is NaN, and scores below -BEYOND have no weight. */
constexpr float FAR = 0x1p23f, BEYOND = 0x1p27f;
__device__ inline bool far_ref(float &m) {
    if (!__any(fabsf(m) > FAR && m > -INFINITY)) return false;
    m = m < BEYOND ? m > -INFINITY ? fmaxf(m, -BEYOND) : m : __int_as_float(0x7FC00000);
    return true;
}
__device__ inline float far_score(float s, float ck, float m) { return fmaf(s, ck, m == -INFINITY ? 0.f : -m) + SHIFT_H; }

/* A record's statistics.  m of -inf says that its row sees no position there, and
 * its sum is left out where records meet; a sum that is NaN has to reach the row
 * (queries that are not finite may leave m as it began), so m is NaN with it. */
__device__ inline void write_stat(const RowsPlan &p, const Work &w, size_t rec, float m, float l) {
    write_ml(p, w, rec, l == l ? m : l, l);
}

__device__ inline float max16(float v) {   /* with the lanes 16 apart */
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

/* four bytes, two pairs of f16 */
__device__ inline void to_half(uint32_t w, h2 &a, h2 &b) {
    const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    w ^= 0x80808080u;   /* + 128; under the top byte of 1024 that is 1024 + 128 + n */
    a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
    b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
}

/* ---- few rows: positions over the waves ----
 *
 * A workgroup of four waves takes 16 m-rows; a wave walks blocks
 * in pairs (every fourth pair), bytes straight from the pages into registers,
 * no LDS and no barrier until the four waves' sums meet.
 *
 * S^T[position][m-row] is integer: K as it is, q as three signed digits of
 * base 256 of q 2^s, its head's largest value to 2^22 .. 2^23 (24 bits of it),
 * on v_mfma_i32_16x16x64_i8.  A digit's sum is exact and below 2^21; joined
 * they are rounded twice, the upper two (below 2^29) as they become f32 and the
 * whole.  D lane l holds m-row l % 16, positions 4 (l / 16) + v.
 * O^T[dim][m-row] is f16 (16x16x32) over both blocks' 32 positions in the
 * order in which the lanes hold their weights, split in two f16; the lanes
 * load V rows 4 (l / 16) .. + 3 of each block, dims HD / 16 (l % 16) .., and one byte
 * permutation a pair both transposes and widens them.
 *
 * Bound: the pages' bytes where they are many.  64 rows of 32 + 4 heads of 128
 * behind 61 .. 8,314 positions, 277 MB, over three states in turn: 58.5 - 61 us, 4.6 -
 * 4.75 TB/s (256 behind 4,000 each, 1,049 MB, 184 - 193 us, 5.4 - 5.7); one of 64 + 8
 * heads of 64 behind 30,001 11 - 13 us, where the chain of a workgroup is most: its
 * lengths, its table, its first blocks, then four steps.  (Two steps loaded ahead take 20 registers more and no time less; 32 m-rows a
 * workgroup 15.4 us instead of 12.2 at nine rows behind 1,000 positions.)  Three
 * waves a SIMD: 168 registers of heads of 128, 108 of 64, none spilled. */
constexpr int MN = 16;
template <int HD>
struct SharedPN {
    __attribute__((aligned(16))) float mo[4][MN][HD];
    float mm[4][MN], ml[4][MN];
};
template <int HD>
__device__ inline __attribute__((always_inline)) void paged_n(const PromptArgs &a, const Pages &pg, const Part &pt, int item,
                                                              SharedPN<HD> &sh) {
    constexpr int N = HD / 16, J = HD / 64, WORDS = N / 4;
    const int ratio = a.n_heads / a.n_kv, hd = a.head_dim;
    const RowsPlan &p = pt.p;
    Work w;
    if (!find_blocks<MN>(a, pt, ratio, item, w)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, kq = lane >> 4;

    /* step n of the wave: blocks j0 + 8 n + 2 wave, + 1; a chunk is 32 steps */
    const int j0 = (w.lo >> 4) + 2 * wave, steps = max(0, (w.hi - w.lo - 32 * wave + 127) >> 7);
    auto chunk = [&](int n) {
        const int j = j0 + 8 * (n + (lane >> 1)) + (lane & 1);
        return load_blocks(a, pg, w, j, PAGE_BLOCK * j < w.hi);
    };
    Blocks bl = chunk(0);
    const size_t bytes = (size_t)PAGE_BLOCK * hd;
    uint32_t koff[J], voff[4];
#pragma unroll
    for (int j = 0; j < J; j++) koff[j] = 64 * j + 16 * kq < hd ? c16 * hd + 64 * j + 16 * kq : 0;   /* q is 0 there */
#pragma unroll
    for (int e = 0; e < 4; e++) voff[e] = N * c16 < hd ? (4 * kq + e) * hd + N * c16 : 0;            /* not written */
    struct Raw {
        u32x4 k[2][J];
        uint32_t v[8][WORDS];
    };
    auto load = [&](int i, Raw &r) __attribute__((always_inline)) {   /* blocks i, i + 1 of the chunk */
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const size_t at = (size_t)__builtin_amdgcn_readlane(bl.at, i + t) * bytes;
            const int8_t *kb = pg.k + at, *vb = pg.v + at;
#pragma unroll
            for (int j = 0; j < J; j++) r.k[t][j] = *(const u32x4 *)(kb + koff[j]);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int n = 0; n < WORDS; n++) r.v[4 * t + e][n] = *(const uint32_t *)(vb + voff[e] + 4 * n);
        }
    };
    Raw cur;
    load(0, cur);   /* without steps: block 0 of the pages, which is there */

    v4i q[3][J];
    v4f o[N];
    const float base2 = LOG2E / sqrtf((float)hd);
    const Lane x = lane_rows(a, w, 0, c16, MN, ratio);
    const float *src = a.q + (size_t)x.r * a.q_stride + (size_t)x.h * hd;
    f4 u[J][4];
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const int d = 64 * j + 16 * kq + 4 * n;
            u[j][n] = x.live && d < hd ? (f4)*(const f4u *)(src + d) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) big = max_nan(big, fabsf(u[j][n][e]));
        }
    big = other_half_max(max16(big));
    /* 2^s that takes the largest to QMAX at most; a query below 2^-80 scores 0 */
    const bool fine = big < INFINITY, some = fine && big > 0x1p-80f;
    const int ex = some ? (__builtin_amdgcn_frexp_mantf(big) > (float)QMAX / 0x1p23f ? 22 : 23) - __builtin_amdgcn_frexp_expf(big) : 0;
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
        for (int n = 0; n < 4; n++) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[e] = some ? (uint32_t)((int)__builtin_rintf(__builtin_amdgcn_ldexpf(u[j][n][e], ex)) + 0x808080) : 0x808080u;
#pragma unroll
            for (int b = 0; b < 3; b++) {
                const uint32_t sel = (uint32_t)(b | (4 + b) << 8);
                const uint32_t lo = __builtin_amdgcn_perm(y[1], y[0], sel), hi = __builtin_amdgcn_perm(y[3], y[2], sel);
                q[b][j][n] = (int)(__builtin_amdgcn_perm(hi, lo, 0x05040100u) ^ 0x80808080u);
            }
        }
    const float c = __builtin_amdgcn_ldexpf(base2, -ex);
    float mx = -INFINITY, lag = LAG_H, l = fine ? 0.f : __int_as_float(0x7FC00000);
#pragma unroll
    for (int n = 0; n < N; n++) o[n] = v4f{0.f, 0.f, 0.f, 0.f};

    const float one = opaque_one();
    for (int n = 0; n < steps; n++) {
        const int i = 2 * (n & 31), t = w.lo + 32 * wave + 128 * n;
        int ex[2];
#pragma unroll
        for (int b = 0; b < 2; b++) ex[b] = __builtin_amdgcn_readlane(bl.exps, i + b);
        const Raw r = cur;
        if (n + 1 < steps) {
            if (((n + 1) & 31) == 0) bl = chunk(n + 1);
            load(2 * ((n + 1) & 31), cur);
        }
        h8 ph, pl;
        float s[2][4], ck[2], top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            v4i d[3];
#pragma unroll
            for (int g = 0; g < 3; g++) {
                d[g] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < J; j++)
                    d[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, r.k[b][j]), q[g][j], d[g], 0, 0, 0);
            }
            ck[b] = c * exp_up(ex[b] & 255);
#pragma unroll
            for (int v = 0; v < 4; v++) s[b][v] = fmaf((float)(d[2][v] * 256 + d[1][v]), 256.f, (float)d[0][v]);
        }
        if (t + 31 > x.all_hi || t < x.all_lo) {   /* uniform */
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int pos = t + 16 * b + 4 * kq + v;
                    s[b][v] = pos <= x.last && pos >= x.first ? s[b][v] : -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const float u = fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3]));
            top = fmaxf(top, fmaf(u, ck[b], (float)((ex[b] >> 8 & 255) - 127)));
        }
        top = other_half_max(max16(top));
        float ref = mx;
        if (__any(top > mx + lag)) {
            float mn = fmaxf(mx, ceilf(top));
            ref = mn;
            if (__builtin_expect(far_ref(mn), false)) {   /* hardly ever */
                lag = ref = -INFINITY;
#pragma unroll
                for (int b = 0; b < 2; b++) {
#pragma unroll
                    for (int v = 0; v < 4; v++) s[b][v] = far_score(s[b][v], ck[b], mn);
                    ck[b] = 1.f;
                }
            }
            const float alpha = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
            mx = mn;
            l *= alpha;
#pragma unroll
            for (int k = 0; k < N; k++) o[k] *= alpha;
        }
        ref = ref == -INFINITY ? 0.f : SHIFT_H - ref;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int ev = ex[b] >> 8 & 255;
            const float add = ref + (float)(ev - 127);
            float e[4];
#pragma unroll
            for (int v = 0; v < 4; v++) e[v] = __builtin_amdgcn_exp2f(fmaf(s[b][v], ck[b], add));
            l = fmaf((e[0] + e[1]) + (e[2] + e[3]), exp_down(ev), l);
#pragma unroll
            for (int v = 0; v < 4; v += 2) {
                h2 hi, lo;
                split2(e[v], e[v + 1], e[v], e[v + 1], one, hi, lo);
                ph[4 * b + v] = hi[0], ph[4 * b + v + 1] = hi[1];
                pl[4 * b + v] = lo[0], pl[4 * b + v + 1] = lo[1];
            }
        }
        if ((ex[0] | ex[1]) >> 16) {   /* uniform, hardly ever */
#pragma unroll
            for (int b = 0; b < 2; b++)
                if (ex[b] >> 16 && x.first <= t + 16 * b + 15 && x.last >= t + 16 * b) l = __int_as_float(0x7FC00000);
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            h8 v;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
                const uint32_t sel = 0x0C000C00u | (uint32_t)(4 + (k & 3)) << 16 | (uint32_t)(k & 3);
                const h2 y = __builtin_bit_cast(h2, __builtin_amdgcn_perm(r.v[e + 1][k >> 2], r.v[e][k >> 2], sel) ^ 0x64806480u) - bias;
                v[e] = y[0], v[e + 1] = y[1];
            }
            o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[k], 0, 0, 0);
            o[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[k], 0, 0, 0);
        }
    }

    /* the waves' sums as one, in wave order: 16 threads a row, HD / 16 dims each */
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
        for (int n = 0; n < N; n += 4)
            *(f4 *)&sh.mo[wave][c16][N * (4 * kq + v) + n] = f4{o[n][v], o[n + 1][v], o[n + 2][v], o[n + 3][v]};
    if (kq == 0) sh.mm[wave][c16] = mx, sh.ml[wave][c16] = l;
    __syncthreads();
    const int row = tid >> 4, d0 = (tid & 15) * N;
    const Lane y = lane_rows(a, w, 0, row, MN, ratio);
    float M = sh.mm[0][row];
#pragma unroll
    for (int g = 1; g < 4; g++) M = fmaxf(M, sh.mm[g][row]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, r[N];
#pragma unroll
    for (int n = 0; n < N; n++) r[n] = 0.f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const float e = __builtin_amdgcn_exp2f(sh.mm[g][row] - base);
        L = fmaf(sh.ml[g][row], e, L);
#pragma unroll
        for (int n = 0; n < N; n++) r[n] = fmaf(sh.mo[g][row][d0 + n], e, r[n]);
    }
    if (!y.live || d0 >= hd) return;
    float *dst, f;
    const long long rec = record_of<MN>(a, pt, w, y, row);
    if (rec >= 0) {
        f = UNSHIFT;
        if (d0 == 0) write_stat(p, w, rec, M, L * f);
        if (M == -INFINITY) return;   /* a record of no position has no sums */
        dst = p.o + rec * hd + d0;
    } else {
        f = 1.f;
        if (a.sinks) {
            const float ref = M - SHIFT_H, sk = a.sinks[y.h] * LOG2E, mn = fmaxf(ref, sk), b2 = mn == -INFINITY ? 0.f : mn;
            f = exp2f(ref - b2);
            L = L * f + exp2f(sk - b2);
        }
        f /= L;
        dst = a.out + (size_t)y.r * a.out_stride + (size_t)y.h * hd + d0;
    }
#pragma unroll
    for (int n = 0; n < N; n += 4) *(f4u *)(dst + n) = f4{r[n] * f, r[n + 1] * f, r[n + 2] * f, r[n + 3] * f};
}

template <int HD>
__global__ __launch_bounds__(256, 3) void k_paged_n(PromptArgs a, Pages pg, Part pt) {
    __shared__ SharedPN<HD> sh;
    paged_n<HD>(a, pg, pt, blockIdx.x, sh);
}

/* ---- many rows ----
 *
 * The products of k_rows_h (tg_prompt.hip), 32 m-rows a wave on 32x32x16 f16:
 * S^T = K Q^T with q as two f16, O^T += V^T P^T with the weights as two.  Bytes
 * are loaded two tiles of 64 positions ahead and widened to f16, which holds
 * them, as they are stored to one of two LDS buffers one tile ahead.  With
 * KG = 2, two groups of MW waves take the tiles in turn; J blocks of 32
 * positions are computed together.
 *
 * Bound for long prompts: the matrix units at the power limit and the issue of
 * the softmax beside them.  8,192 rows of 32 heads of 128: 915 us, 1.20 PFLOP/s
 * counting both products (a large f16 product runs at 1.15 - 1.2); of 64 heads of 64
 * 1,060, where a product is half as long and the softmax is not: three waves a
 * SIMD, 168 registers and 2 spilled (two waves 5% more).  Heads of 128 have 256 registers, of
 * which 2 (256 rows) to 10 (128 rows in one or two groups) are spilled.  Widening costs a quarter more VALU
 * instructions than f16 caches take.  (Integer products for the scores, as few rows have, would be a
 * quarter less of the first product and twice that in joining its digits; the widening before the
 * products in half of the waves and behind them in the others changed nothing.) */
template <int HD, int MW, int KG>
struct SharedPW {
    __attribute__((aligned(1024))) uint8_t bufs[KG][2][2][KT * HD * 2];
    long long where[KG == 2 ? 32 * MW : 1];
};

/* The wave's rows finished, as write_rows does for dense caches; a NaN is the
 * row's own here. */
template <int HD, int MTILE>
__device__ inline void write_paged(const PromptArgs &a, const Part &pt, const Work &w, const Lane &x, int from, int lane, float mx,
                                   float l, const f16v (&o)[HD / 32], uint8_t *stage, long long *where) {
    const int half = lane >> 5, row = lane & 31, hd = a.head_dim;
    bool write = x.live;
    long long at;
    float f;
    const long long rec = record_of<MTILE>(a, pt, w, x, from + row);   /* uniform whether there is one */
    if (rec >= 0) {
        f = UNSHIFT;
        if (write && half == 0) write_stat(pt.p, w, rec, mx, l * f);
        write = write && mx > -INFINITY;      /* a record of no position has no sums */
        at = rec * hd;
    } else {
        f = 1.f;
        if (a.sinks && write) {
            const float ref = mx - SHIFT_H, sk = a.sinks[x.h] * LOG2E, M = fmaxf(ref, sk), base = M == -INFINITY ? 0.f : M;
            f = exp2f(ref - base);
            l = l * f + exp2f(sk - base);
        }
        f /= l;
        at = (long long)x.r * a.out_stride + (long long)x.h * hd;
    }
    if (stage && half == 0) where[row] = write ? at : -1;
    float *dst = (rec >= 0 ? pt.p.o : a.out) + at;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const int dim = 32 * d + 8 * v + 4 * half;
            f4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = o[d][4 * v + e] * f;
            if (stage) *(f4 *)(stage + row * (HD * 4) + row_piece<HD>(row, 8 * d + 2 * v + half)) = y;
            else if (write && dim < hd) *(f4u *)(dst + dim) = y;
        }
}

template <int HD, int MW, int KG, int J>
__device__ inline __attribute__((always_inline)) void paged_w(const PromptArgs &a, const Pages &pg, const Part &pt, int item,
                                                              SharedPW<HD, MW, KG> &sh) {
    constexpr int RB = HD * 2, TILE = KT * RB;          /* bytes of a row in LDS, of a tile of K or V */
    constexpr int DB = HD / 32, STEPS = HD / 16;
    constexpr int LR = 1024 / HD, LOADS = KT / LR;      /* rows a load of a wave covers, loads of a tile of K or V */
    constexpr int NL = 2 * LOADS / MW;                  /* a wave's: mwave + MW k of K's, then V's */
    static_assert(NL >= 1 && 16 % LR == 0, "a load is of one block");
    auto &bufs = sh.bufs;
    const int ratio = a.n_heads / a.n_kv, hd = a.head_dim;
    Work w;
    if (!find_blocks<32 * MW>(a, pt, ratio, item, w)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, group = wave / MW, mwave = wave % MW;
    static_assert(KG == 1 || sizeof bufs >= MW * 256 * (HD / 2 + 3), "merge_groups");
    uint8_t(*buf)[2][TILE] = bufs[group];

    /* tile n: blocks j0 + 4 n ..; a chunk of blocks is 16 tiles */
    const int j0 = w.lo >> 4, tiles = (w.hi - w.lo + KT - 1) / KT;
    auto chunk = [&](int n) {
        const int j = j0 + 4 * (n & ~15) + lane;
        return load_blocks(a, pg, w, j, PAGE_BLOCK * j < w.hi);
    };
    Blocks bl = chunk(0);
    int have = 0;   /* the chunk that bl is of */
    const size_t bytes = (size_t)PAGE_BLOCK * hd;
    const int lrow = lane / (HD / 16), piece = lane % (HD / 16);
    /* pieces past head_dim get its first: finite, q is 0 there, and of V such dims are not written */
    const uint32_t lane_off = (uint32_t)(lrow * hd + (16 * piece < hd ? 16 * piece : 0));
    u32x4 raw[NL];
    auto load = [&](int n) __attribute__((always_inline)) {
        if (n >> 4 != have) bl = chunk(n), have = n >> 4;
#pragma unroll
        for (int k = 0; k < NL; k++) {
            const int u = mwave + MW * k, row = LR * (u % LOADS);
            const size_t at = (size_t)__builtin_amdgcn_readlane(bl.at, (4 * n & 63) + (row >> 4)) * bytes;
            raw[k] = *(const u32x4 *)((u < LOADS ? pg.k : pg.v) + at + (uint32_t)((row & 15) * hd) + lane_off);
        }
    };
    int stored[4];   /* the stored tile's exponents */
    auto store = [&](int n, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) stored[e] = __builtin_amdgcn_readlane(bl.exps, (4 * n & 63) + e);
#pragma unroll
        for (int k = 0; k < NL; k++) {
            const int u = mwave + MW * k, key = LR * (u % LOADS) + lrow;
            h2 y[8];
#pragma unroll
            for (int e = 0; e < 4; e++) to_half(raw[k][e], y[2 * e], y[2 * e + 1]);
            uint8_t *at = &buf[b][u < LOADS ? 0 : 1][key * RB];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const h8 z = {y[4 * e][0], y[4 * e][1], y[4 * e + 1][0], y[4 * e + 1][1],
                              y[4 * e + 2][0], y[4 * e + 2][1], y[4 * e + 3][0], y[4 * e + 3][1]};
                *(h8 *)(at + (((2 * piece + e) ^ swz<HD>(key)) << 4)) = z;
            }
        }
    };
    load(group);
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
    /* a query that is not finite makes its row NaN, and its f16 nothing else's: the m-row is the lane */
    float l = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) l = fmaf((float)qh[s][e], 0.f, l);
    f16v o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[d][v] = 0.f;
    float mx = -INFINITY, lag = LAG_H;
    const uint32_t kaddr = k_operand<HD>(lane);
    uint32_t vaddr[DB][2];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 2; e++) vaddr[d][e] = TILE + v_operand<HD>(lane, d, e);
    const float one = opaque_one();

    int ex[4];
    store(group, 0);
    if (group + KG < tiles) load(group + KG);
    int b = 0;
    for (int n0 = 0; n0 < tiles; n0 += KG, b ^= 1) {
        const int n = n0 + group, t = w.lo + KT * n;
        bar_lds();   /* every wave has stored this tile, and is done with the other buffer */
#pragma unroll
        for (int e = 0; e < 4; e++) ex[e] = stored[e];
        if (n + KG < tiles) {
            store(n + KG, b ^ 1);
            if (n + 2 * KG < tiles) load(n + 2 * KG);
        }
        if (t > x.any_hi || t + KT <= x.any_lo || n >= tiles) continue;   /* uniform in the wave */
#pragma unroll 1
        for (int i = 0; i < KT; i += 32 * J) {
            const int at = t + i;
            if (J == 1 && (at > x.any_hi || at + 32 <= x.any_lo)) continue;
            const Lds tile = (Lds)buf[b][0] + i * RB;
            int eg[2 * J];   /* of each 16 positions */
#pragma unroll
            for (int g = 0; g < 2 * J; g++) eg[g] = J == 1 && i ? ex[2 + g] : ex[g];
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
                const Lds ahead = tile + (kaddr ^ (uint32_t)((st + 1) << 5));
#pragma unroll
                for (int j = 0; j < J; j++) k1[j] = st + 1 < STEPS ? lds_row(ahead + j * 32 * RB) : k0[j];
#pragma unroll
                for (int j = 0; j < J; j++) s[j] = MFMA_H(k0[j], ql[st], s[j]);
#pragma unroll
                for (int j = 0; j < J; j++) s[j] = MFMA_H(k0[j], qh[st], s[j]);
#pragma unroll
                for (int j = 0; j < J; j++) k0[j] = k1[j];
            }
            auto column = [&](int u) __attribute__((always_inline)) {
                const int q = u / DB, d = u % DB;
                return h8_of(lds_column(tile + vaddr[d][0] + q * 16 * RB), lds_column(tile + vaddr[d][1] + q * 16 * RB));
            };
            h8 v0 = column(0), v1 = column(1);
            float top = -INFINITY, ck[2 * J];
#pragma unroll
            for (int j = 0; j < J; j++) {
                mask_scores(s[j], at + 32 * j + 4 * half, x);
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    float u = s[j][8 * g];
#pragma unroll
                    for (int v = 1; v < 8; v++) u = max_nan(u, s[j][8 * g + v]);
                    ck[2 * j + g] = c * exp_up(eg[2 * j + g] & 255);
                    top = max_nan(top, fmaf(u, ck[2 * j + g], (float)((eg[2 * j + g] >> 8 & 255) - 127)));
                }
            }
            top = other_half_max(top);
            float ref = mx;
            if (__any(top > mx + lag)) {
                float mn = max_nan(mx, ceilf(top));
                ref = mn;
                if (__builtin_expect(far_ref(mn), false)) {   /* hardly ever */
                    lag = ref = -INFINITY;
#pragma unroll
                    for (int g = 0; g < 2 * J; g++) {
#pragma unroll
                        for (int v = 8 * (g & 1); v < 8 * (g & 1) + 8; v++) s[g >> 1][v] = far_score(s[g >> 1][v], ck[g], mn);
                        ck[g] = 1.f;
                    }
                }
                const float alpha = mn == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
                mx = mn;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[d][v] *= alpha;
            }
            ref = ref == -INFINITY ? 0.f : SHIFT_H - ref;
            __builtin_amdgcn_iglp_opt(2);
            h8 ph[2 * J], pl[2 * J];
#pragma unroll
            for (int g = 0; g < 2 * J; g++) {
                const float add = ref + (float)((eg[g] >> 8 & 255) - 127);
                float sum[2] = {0.f, 0.f};
#pragma unroll
                for (int v = 0; v < 8; v += 2) {
                    const float e0 = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + v], ck[g], add));
                    const float e1 = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + v + 1], ck[g], add));
                    sum[0] += e0, sum[1] += e1;
                    h2 hi, lo;
                    split2(e0, e1, e0, e1, one, hi, lo);
                    ph[g][v] = hi[0], ph[g][v + 1] = hi[1], pl[g][v] = lo[0], pl[g][v + 1] = lo[1];
                }
                l = fmaf(sum[0] + sum[1], exp_down(eg[g] >> 8 & 255), l);
            }
#pragma unroll
            for (int u = 0; u < 2 * J * DB; u += 2) {
                const bool more = u + 2 < 2 * J * DB;
                const h8 n0 = more ? column(u + 2) : v0, n1 = more ? column(u + 3) : v1;
                const int q = u / DB, d = u % DB;
                o[d] = MFMA_H(v0, pl[q], o[d]);
                o[d + 1] = MFMA_H(v1, pl[q], o[d + 1]);
                o[d] = MFMA_H(v0, ph[q], o[d]);
                o[d + 1] = MFMA_H(v1, ph[q], o[d + 1]);
                v0 = n0, v1 = n1;
            }
            int odd = 0;
#pragma unroll
            for (int g = 0; g < 2 * J; g++) odd |= eg[g];
            if (odd >> 16) {   /* uniform, hardly ever */
#pragma unroll
                for (int g = 0; g < 2 * J; g++)
                    if (eg[g] >> 16 && x.first <= at + 16 * g + 15 && x.last >= at + 16 * g) l = __int_as_float(0x7FC00000);
            }
        }
    }
    l = other_half_sum(l);
    int oexp = 0;
    if (KG == 2 && tiles > 1) merge_groups<HD, MW>((float *)bufs, wave, lane, mx, l, oexp, o);
    else __syncthreads();   /* one group, or the second had no tile: all are done with the tiles */
    constexpr int STRIDE = 64 * (HD / 2 + 3) * 4;   /* a wave's share of merge_groups' room */
    if (group == 0)
        write_paged<HD, 32 * MW>(a, pt, w, x, 32 * mwave, lane, mx, l, o, KG == 2 ? (uint8_t *)bufs + wave * STRIDE : nullptr,
                                 sh.where + (KG == 2 ? 32 * wave : 0));
    if constexpr (KG == 2) {
        __syncthreads();
        const bool records = pt.tiles ? w.count != 1 : pt.p.nrec > 0;
        store_rows<HD, 32 * MW>(hd, (const uint8_t *)bufs, STRIDE, sh.where, records ? pt.p.o : a.out, wave, MW * KG);
    }
}

template <int HD, int MW, int KG, int J>
__global__ __launch_bounds__(64 * MW * KG, HD == 64 && MW * KG == 4 ? 3 : 2) void k_paged_w(PromptArgs a, Pages pg, Part pt) {
    __shared__ SharedPW<HD, MW, KG> sh;
    paged_w<HD, MW, KG, J>(a, pg, pt, blockIdx.x, sh);
}

/* A mixed call in one launch: sequences of many rows in tiles of 128, those of
 * few in tiles of 16, each kind cut into spans by its own positions.  In two
 * launches 60 single tokens and a chunk of 500 rows took 119 us (32 + 4 heads of 128; in one, cut the same way, 108),
 * seven sequences of 1 to 1,000 rows 73 (68).  Both kinds have the larger one's registers and LDS: at heads of 128 256 (11
 * spilled) and 65 KB, so that tiles of 16 run at two waves a SIMD here and not at three. */
template <int HD>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void k_paged_both(PromptArgs a, Pages pg, Part many, Part few) {
    __shared__ union {
        SharedPW<HD, 4, 1> w;
        SharedPN<HD> n;
    } sh;
    const int first = many.p.items * a.n_kv;
    if ((int)blockIdx.x < first) paged_w<HD, 4, 1, 2>(a, pg, many, blockIdx.x, sh.w);
    else paged_n<HD>(a, pg, few, (int)blockIdx.x - first, sh.n);
}

/* The records of a cut tile's rows as one: a workgroup of 16 waves has a KV
 * head and a tile of 16 rows, or half of one of 128; a wave a row at a time,
 * HD / 4 lanes a record. */
template <int HD, int MTILE>
__device__ inline __attribute__((always_inline)) void join_tile(const PromptArgs &a, const Part &pt, int b) {
    constexpr int G = HD / 4, PER = 64 / G, N = 4, ROWS = MTILE == 16 ? 16 : 64;
    const int ratio = a.n_heads / a.n_kv, hd = a.head_dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int place = b / a.n_kv, from = 0;
    Work w;
    w.prefix = false, w.kh = b - place * a.n_kv;
    const Class keep = {pt.least, pt.most, ratio};
    if (pt.most == FEW) {
        const int s = place / (FEW / MTILE);
        w.sq = seq_at(a.s, s);
        keep(w.sq);
        w.m0 = MTILE * (place - s * (FEW / MTILE));
        if (w.m0 >= w.sq.n * ratio) return;
        set_rows(w, ratio);
    } else {
        from = ROWS * (place % (MTILE / ROWS));
        if (!find_tile<MTILE>(a, pt.p, ratio, place / (MTILE / ROWS), w, keep)) return;
        place = tile_place<MTILE>(pt, w, ratio);
    }
    const Part::Tile tile = pt.tiles[place];
    /* Offsets that decrease overlap, and make more spans than there are items: some are computed by none, and their tile's entry
     * is whatever the scratch held.  No record outside the part's is read for it. */
    const unsigned items = (unsigned)pt.p.items;
    if (tile.count <= 1 || tile.count > pt.p.cap || (unsigned)tile.item >= items || (unsigned)tile.last >= items ||
        (unsigned)tile.step >= items || (unsigned)tile.item + (unsigned)(tile.count - 2) * (unsigned)tile.step >= items)
        return;
    const int rows = min(from + ROWS, min(MTILE, w.sq.n * ratio - w.m0)), g = lane / G, d = 4 * (lane % G);
    for (int m = from + wave; m < rows; m += 16) {
        int i, j;
        w.row(m, ratio, i, j);
        const int r = w.sq.r0 + i, h = w.kh * ratio + j;
        const float sink = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
        auto rec = [&](int c) {
            return ((size_t)(c == tile.count - 1 ? tile.last : tile.item + c * tile.step) * a.n_kv + w.kh) * MTILE + m;
        };
        f4 stat = {-INFINITY, 0.f, 0.f, 0.f}, y[N];   /* at most 64 records */
        if (lane < tile.count) stat = *(const f4 *)(pt.p.ml + 4 * rec(lane));
        auto load = [&](int c0) {
#pragma unroll
            for (int q = 0; q < N; q++) {
                const int c = c0 + q * PER + g;
                y[q] = f4{0.f, 0.f, 0.f, 0.f};
                if (c < tile.count && d < hd) y[q] = *(const f4 *)(pt.p.o + rec(c) * hd + d);
            }
        };
        load(0);
        const float M = fmaxf(wave_max(stat[0]), sink), base = M == -INFINITY ? 0.f : M;
        /* -1: a record of no position, whose sums are not written */
        const float e = stat[0] != -INFINITY ? exp2f(stat[0] - base) : -1.f;
        float l = wave_sum(e < 0.f ? 0.f : stat[1] * e);
        f4 o = {0.f, 0.f, 0.f, 0.f};
        for (int c0 = 0; c0 < tile.count; c0 += N * PER) {
            if (c0) load(c0);
#pragma unroll
            for (int q = 0; q < N; q++) {
                const int c = c0 + q * PER + g;
                const float f = __shfl(e, c & 63, 64);
                if (c < tile.count && !(f < 0.f)) o += y[q] * f;
            }
        }
#pragma unroll
        for (int q = 32; q >= G; q >>= 1)
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] += __shfl_xor(o[k], q, 64);
        if (a.sinks) l += exp2f(sink - base);
        if (lane < G && d < hd) *(f4u *)(a.out + (size_t)r * a.out_stride + (size_t)h * hd + d) = o * (1.f / l);
    }
}
template <int HD>
__global__ __launch_bounds__(1024) void k_paged_join(PromptArgs a, Part many, Part few, int first) {
    if ((int)blockIdx.x < first) join_tile<HD, 16>(a, few, blockIdx.x);
    else join_tile<HD, 128>(a, many, (int)blockIdx.x - first);
}

}  // namespace

/* How a call is cut, from the host's arguments alone (the lengths are on the
 * device), as rows_cut does for dense caches:
 *   narrow  16 m-rows a workgroup, positions over its waves
 *   wide    128 m-rows, two groups of four waves on tiles in turn
 *   short   128 m-rows, four waves, for few positions a row
 *   full    the same, two workgroups a CU on long spans
 *   tall    256 m-rows, eight waves: half the widening a row, where there are
 *           enough of them (32 heads of 128: 4,096 rows 250 us, full 279; 8,192 930 and 966; 2,999
 *           161 and 154; heads of 64, bound by the softmax's issue, 299 and 296)
 *   mixed   several sequences, of many rows together: full for those of more
 *           than FEW m-rows, narrow for the others */
namespace {

enum Shape { NARROW, SHORT, WIDE, FULL, TALL, MIXED };
int tile_of(Shape s) { return s == NARROW ? 16 : s == TALL ? 256 : 128; }
constexpr int SHORT_BELOW = 512, MOST_SPANS = 64;
struct Cut {
    Shape shape;
    bool items;       /* records by item */
    Part part, few;   /* few: of a mixed call */
};
/* Whether tiles of 16 take less time, in us, from fits to one call of many shapes (1 to 1,500 rows behind 0 to 16,000 positions,
 * 32 + 4 heads of 128 and 64 + 8 of 64; off by a tenth mostly): what starts, each workgroup, and each 2^20 pairs of an
 * m-row and a position.  Tiles of 128 do the pairs faster and start later.  128 rows 8.8 us in tiles of 16 and 13.5 in tiles
 * of 128, 300 behind 1,000 positions 30.7 and 34.9, 1,024 44.2 and 39.5, nine behind 4,000 14.3 and 19.7, 100 behind 8,000 58.3
 * and 45.6 (heads of 128). */
bool narrow_is_faster(long long m, long long rows, long long seqs, int n_kv, int head_dim, int positions, bool window) {
    const bool big = head_dim > 64;
    /* how many positions a row sees on average: of a chunk known, of several sequences half the longest's */
    const double seen = seqs > 1 ? positions / 2.0 : window ? positions : positions - (double)std::min<long long>(rows, positions) / 2;
    const double pairs = m * seen * n_kv / (1 << 20), wgs = (double)std::max(m / 16, seqs) * n_kv;
    const double narrow = (wgs < 512 && positions > 640 ? 10 : 5) + wgs * (big ? 0.0115 : 0.005) + pairs * (big ? 1.5 : 1.05);
    if (positions < SHORT_BELOW) return narrow < 8 + positions * (big ? 0.035 : 0.022) * std::max(1.0, wgs / 8 / 512);
    return narrow < (seqs > 1 ? 8 : 0) + (big ? 19 : 14) + wgs * (big ? 0.004 : 0.002) + pairs * (big ? 1.05 : 0.64);
}
Shape shape_of(long long m, long long rows, long long seqs, int n_kv, int head_dim, int positions, bool window) {
    if (m <= 16 * seqs || narrow_is_faster(m, rows, seqs, n_kv, head_dim, positions, window)) return NARROW;
    if (positions < SHORT_BELOW) return SHORT;
    if (seqs > 1) return MIXED;
    if (head_dim > 64 && m / 256 * n_kv >= 512) return TALL;
    return m / 128 * n_kv > 512 ? FULL : WIDE;
}

/* A part in tiles of `tile` m-rows whose records are by item.  Beyond OFTEN
 * places for tiles (of 128 m-rows; twice as many of 16), each sequence with one
 * of its own, it is not cut.  Of many single tokens and a chunk that is before
 * the chunk's own tiles are so many: those places cost the join more than cuts
 * gain at ordinary depths (128 sequences of 64 + 8 heads, one of them 500 rows, behind
 * 1,000 positions 53 us uncut and 79 cut; behind 8,000 202 and 191, 30,000 668 and 567). */
constexpr int OFTEN = 1024;
int often(int tile) { return tile == 16 ? 2 * OFTEN : OFTEN; }
/* tiles that there can be at most, of sequences of at least `least` m-rows */
long long most_tiles(long long m, int n, int tile, int least) { return std::min(m / tile + std::min<long long>(n, m / least), m); }
Part item_part(const PromptArgs &a, long long m, int tile, int slots, int least, int most) {
    Part k = {};
    k.least = least, k.most = most;
    long long tiles = most_tiles(m, a.s.n, tile, least), places = most_tiles(m, a.s.n, tile, 1);
    if (most == FEW) tiles = places = std::min(tiles, (long long)a.s.n * (FEW / tile));
    k.p.target = std::max(1, slots / a.n_kv);
    k.p.unit = 128;
    k.p.cap = places * a.n_kv > often(tile) ? 1 : MOST_SPANS;
    k.p.items = (int)tiles + (k.p.cap > 1 ? k.p.target : 0);
    return k;
}

Cut paged_cut(const PromptArgs &a) {
    Cut k = {};
    const int n_seqs = a.s.n, n_kv = a.n_kv, ratio = a.n_heads / n_kv;
    const long long m = (long long)a.s.rows * ratio;
    auto sees = [&](int rows) { return a.window > 0 ? (int)std::min<long long>(a.s.kv_max, (long long)a.window + rows / ratio + 1) : a.s.kv_max; };
    k.shape = shape_of(m, a.s.rows, n_seqs, n_kv, a.head_dim, sees(128), a.window > 0);
    if (k.shape == MIXED) {
        k.items = true;
        k.part = item_part(a, m, 128, 512, FEW + 1, INT_MAX);
        k.few = item_part(a, m, 16, 512, 1, FEW);
        return k;
    }
    k.part.least = 1, k.part.most = INT_MAX;
    RowsPlan &p = k.part.p;
    const int tile = tile_of(k.shape), positions = sees(tile);
    const int slots = k.shape == NARROW ? 512 : 256;
    const long long tiles = std::max((m + tile - 1) / tile, (long long)n_seqs), wgs = tiles * n_kv;
    /* of several sequences fewer than run at once: what their cuts leave over fills the rest (64 rows behind 61 .. 8,314
     * positions, 4 KV heads of 128: 65.9 us; as many as run 74.3, half 74.0) */
    const int at_once = k.shape == NARROW && n_seqs > 1 && a.head_dim > 64 ? 384 : slots;
    p.target = std::max(1, at_once / n_kv);
    p.unit = 128;
    /* us(n): a span's positions (measured on workgroups alone: one row of 64 + 8 heads of 64 behind 1,000 and 4,000 positions 11.0
     * and 26.9 us uncut, of 32 + 4 of 128 13.7 and 33.7), and what n records a row take to write and read, at 4.5 TB/s, with the
     * combine's launch */
    const double t = positions * (k.shape == NARROW ? (a.head_dim > 64 ? 0.9 : 0.75) : (a.head_dim > 64 ? 3.4 : 1.7)) / 128;
    const double r = (double)m * n_kv * a.head_dim * 8 / 4.5e6;
    if (k.shape == NARROW && n_seqs > 1) {
        /* Cut, all finish together; uncut, the longest takes t while the others, half as long on average, fill the rest: what
         * that leaves idle against the second kernel's time.  64 rows of 64 + 8 heads behind up to 2,000 positions 20 us uncut and
         * 25 cut, 48 behind up to 6,000 52 and 38.  A quarter of t always counts: one may be far longer than the others. */
        const double idle = t * (1 - std::min(0.75, wgs / (2.0 * slots)));
        const Part cut = item_part(a, m, tile, at_once, 1, INT_MAX);
        k.items = positions > 2 * p.unit && idle > 6 && cut.p.cap > 1;
        if (k.items) {
            k.part = cut;
            return k;
        }
    }
    const int most = (int)std::min<long long>({MOST_SPANS, (positions + p.unit - 1) / p.unit, std::max(1ll, slots / wgs)});
    auto us = [&](int n) { return t / n + r * n + (n == 1 ? -r : 4); };
    const int n = std::max(1, std::min(most, (int)std::sqrt(t / r)));   /* the best, or the next */
    const int best = n < most && us(n + 1) < us(n) ? n + 1 : n;
    p.cap = us(best) < us(1) && !(k.shape == NARROW && n_seqs > 1) ? best : 1;
    if (n_seqs > 1 && p.cap > 1)   /* room for a sequence much longer than the others */
        p.cap = (int)std::min<long long>({MOST_SPANS, (positions + p.unit - 1) / p.unit, std::max<long long>(4ll * p.cap, 4ll * p.target / tiles)});
    p.search = p.cap == 1 && n_seqs > 256;
    p.items = p.search ? (int)(m / tile) + n_seqs : (int)std::min(m / tile + n_seqs, m) + (p.cap > 1 ? p.target : 0);
    p.nrec = p.cap > 1 ? p.cap : 0;
    return k;
}

/* A part's scratch, in order: statistics and sums of the records, and where
 * each tile's are, if by item */
struct Room {
    size_t records, places;   /* of a part */
    size_t ml() const { return (records * 16 + 255) & ~(size_t)255; }
    size_t o(int hd) const { return records * 4 * (size_t)hd; }
    size_t at() const { return (places * sizeof(Part::Tile) + 255) & ~(size_t)255; }
    size_t all(int hd) const { return ml() + o(hd) + at(); }
};
Room room_of(const PromptArgs &a, const Part &k, int tile, bool items) {
    if (k.p.cap <= 1) return Room{0, 0};
    if (!items) return Room{(size_t)a.s.rows * a.n_heads * k.p.nrec, 0};
    const long long m = (long long)a.s.rows * (a.n_heads / a.n_kv);
    return Room{(size_t)k.p.items * a.n_kv * tile, (size_t)(k.most == FEW ? a.s.n * (FEW / tile) : m / tile + a.s.n)};
}

template <int HD>
void launch_paged(const PromptArgs &a, const Pages &pg, const Cut &k, hipStream_t st) {
    const dim3 grid((unsigned)((k.part.p.items + k.few.p.items) * a.n_kv));
#define PAGED(threads, ...) hipLaunchKernelGGL((__VA_ARGS__), grid, dim3(threads), 0, st, a, pg, k.part)
    if (k.shape == NARROW) PAGED(256, k_paged_n<HD>);
    else if (k.shape == SHORT) PAGED(256, k_paged_w<HD, 4, 1, 1>);
    else if (k.shape == WIDE) PAGED(512, k_paged_w<HD, 4, 2, 2>);
    else if (k.shape == FULL) PAGED(256, k_paged_w<HD, 4, 1, 2>);
    else if (k.shape == TALL) {
        if constexpr (HD > 64) PAGED(512, k_paged_w<HD, 8, 1, 2>);   /* no smaller head is TALL (shape_of) */
    } else {
        hipLaunchKernelGGL((k_paged_both<HD>), grid, dim3(256), 0, st, a, pg, k.part, k.few);
    }
#undef PAGED
    if (!k.items) {
        if (k.part.p.nrec) launch_rows_combine(a, k.part.p, st);
        return;
    }
    /* tiles of 16, then halves of those of 128 */
    const Part &small = k.shape == MIXED ? k.few : k.part, &large = k.part;
    const long long m = (long long)a.s.rows * (a.n_heads / a.n_kv);
    const int first = (small.p.cap <= 1 ? 0 : small.most == FEW ? a.s.n * (FEW / 16) : (int)(m / 16) + a.s.n) * a.n_kv;
    const int more = (k.shape != MIXED || large.p.cap <= 1 ? 0 : 2 * ((int)(m / 128) + a.s.n)) * a.n_kv;
    if (first + more) hipLaunchKernelGGL((k_paged_join<HD>), dim3((unsigned)(first + more)), dim3(1024), 0, st, a, large, small, first);
}

}  // namespace

size_t attention_paged_need(const PromptArgs &a) {
    const Cut k = paged_cut(a);
    return room_of(a, k.part, tile_of(k.shape), k.items).all(a.head_dim) +
           (k.shape == MIXED ? room_of(a, k.few, 16, true).all(a.head_dim) : 0);
}

/* For every call of at most these sizes.  Tiles of a dense cut are cut only
 * while their spans are at most the workgroups that run at once, with several
 * sequences four times as many, so the m-rows times their spans are at most the
 * m-rows of so many tiles.  Records by item have room for every m-row of the
 * items: tiles up to often() workgroups, or none, and what the target adds. */
size_t attention_paged_scratch(int n_rows, int n_seqs, int n_heads, int n_kv, int head_dim, int kv_max) {
    const long long m = (long long)n_rows * (n_heads / n_kv);
    const long long row_heads = (long long)n_rows * n_heads, spans = std::min(MOST_SPANS, (kv_max + 127) / 128);
    if (spans == 1) return 0;
    auto bytes = [&](long long records) { return (size_t)records * (16 + 4 * (size_t)head_dim) + 512; };
    size_t most = bytes(std::min(row_heads * spans, (m <= 16 ? 16ll * 512 : 128ll * 256) * (n_seqs > 1 ? 4 : 1)));
    if (n_seqs > 1) {
        auto part = [&](int tile, int least) {
            const long long tiles = std::min(most_tiles(m, n_seqs, tile, least), std::max(1ll, (long long)often(tile) / n_kv));
            return bytes((tiles + std::max(1, 512 / n_kv)) * n_kv * tile);
        };
        const size_t places = (size_t)(m / 128 + m / 16 + (FEW / 16 + 1) * (long long)n_seqs) * sizeof(Part::Tile) + 512;
        most = std::max(most, part(128, FEW + 1) + part(16, 1) + places);
    }
    return most;
}

void launch_attention_paged(const PromptArgs &a, const Pages &pg, void *scratch, hipStream_t st) {
    Cut k = paged_cut(a);
    uint8_t *at = (uint8_t *)scratch;
    auto place = [&](Part &x, int tile) {
        const Room room = room_of(a, x, tile, k.items);
        x.p.ml = (float *)at;
        x.p.o = (float *)(at + room.ml());
        x.tiles = room.places ? (Part::Tile *)(at + room.ml() + room.o(a.head_dim)) : nullptr;
        at += room.all(a.head_dim);
    };
    place(k.part, tile_of(k.shape));
    if (k.shape == MIXED) place(k.few, 16);
    if (a.head_dim > 64) launch_paged<128>(a, pg, k, st);
    else launch_paged<64>(a, pg, k, st);
}

}  // namespace tg
