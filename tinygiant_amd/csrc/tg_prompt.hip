/*
 * tg_prompt.hip -- packed rows of several sequences: their K and V rows into
 * the caches, and their attention over them.
 *
 * The reference runs attention one row at a time (tg_attention_v2,
 * csrc/libtinygiant.c:939-983, called row by row at tinygiant/engine.py:
 * 232-275); these are the same formulas for many rows a call.
 */
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "tg_device.hpp"
#include "tg_prompt.h"

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

}  // namespace

/* ---- append ----
 * One workgroup a row; a segment of G lanes (16, or 8 for heads of up to 64
 * values) takes a head: lane i the pairs (4 i + e, head_dim / 2 + 4 i + e),
 * so the loads are 16 bytes and RoPE needs no exchange.  The norm is
 * tg_rms_norm's (csrc/libtinygiant.c:680-698), the rotation
 * apply_rope_inplace's (:702-719); an f16 cache gets K and V rounded once, to
 * nearest. */
template <bool HALF, int G>
__global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
    const int r = blockIdx.x, s = seq_of(a.s, r);
    if (s < 0) return;
    const Seq sq = seq_at(a.s, s);
    const int i = r - sq.r0;
    if (i < 0 || i >= sq.n) return;
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
 * One workgroup per (row, query head): 256 keys at a time, a thread a key's
 * score, then a thread an output value's sum; running maximum and sum. */
template <typename T>
__global__ __launch_bounds__(256) void k_attn_row(PromptArgs a) {
    __shared__ float qs[PROMPT_MAX_HEAD_DIM];
    __shared__ float sc[256];
    __shared__ float red[4];
    const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, hd = a.head_dim;
    const int s = seq_of(a.s, r);
    if (s < 0) return;
    const Seq sq = seq_at(a.s, s);
    const int i = r - sq.r0;
    if (i < 0 || i >= sq.n) return;
    const int kh = h / (a.n_heads / a.n_kv);
    const int pos = a.pre_len + sq.past + i;           /* the last position that the row sees */
    const int first = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    if (tid < hd) qs[tid] = a.q[(size_t)r * a.q_stride + (size_t)h * hd + tid];
    const T *pk = (const T *)a.pre_k + (size_t)kh * a.pre_max * hd, *pv = (const T *)a.pre_v + (size_t)kh * a.pre_max * hd;
    const size_t own = ((size_t)sq.slot * a.n_kv + kh) * a.s.kv_max * hd;
    const T *ok = (const T *)a.kv_k + own, *ov = (const T *)a.kv_v + own;
    const float scale = 1.f / sqrtf((float)hd);
    float m = -INFINITY, l = 0.f, o = 0.f;
    __syncthreads();
    for (int t0 = first; t0 <= pos; t0 += 256) {
        const int p = t0 + tid;
        float z = -INFINITY;
        if (p <= pos) {
            const T *row = p < a.pre_len ? pk + (size_t)p * hd : ok + (size_t)(p - a.pre_len) * hd;
            float acc = 0.f;
            for (int d = 0; d < hd; d++) acc = fmaf(qs[d], (float)row[d], acc);
            z = acc * scale;
        }
        float t = wave_max(z);
        if ((tid & 63) == 0) red[tid >> 6] = t;
        __syncthreads();
        t = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(m, t), base = mn == -INFINITY ? 0.f : mn, alpha = expf(m - base);
        const float e = p <= pos ? expf(z - base) : 0.f;
        sc[tid] = e;
        const float w = wave_sum(e);
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = w;
        __syncthreads();
        l = l * alpha + ((red[0] + red[1]) + (red[2] + red[3]));
        m = mn;
        if (tid < hd) {
            o *= alpha;
            const int n = min(256, pos + 1 - t0);
            for (int j = 0; j < n; j++) {
                const int p2 = t0 + j;
                const T *row = p2 < a.pre_len ? pv + (size_t)p2 * hd : ov + (size_t)(p2 - a.pre_len) * hd;
                o = fmaf(sc[j], (float)row[tid], o);
            }
        }
        __syncthreads();
    }
    if (tid >= hd) return;
    if (a.sinks) {
        const float sk = a.sinks[h], mn = fmaxf(m, sk), base = mn == -INFINITY ? 0.f : mn, f = expf(m - base);
        l = l * f + expf(sk - base);
        o *= f;
    }
    a.out[(size_t)r * a.out_stride + (size_t)h * hd + tid] = o / l;
}

size_t attention_rows_scratch(int n_rows, int n_seqs, int n_heads, int n_kv, int head_dim, int kv_max, int pre_len) {
    (void)n_rows, (void)n_seqs, (void)n_heads, (void)n_kv, (void)head_dim, (void)kv_max, (void)pre_len;
    return 0;
}

void launch_attention_rows(const PromptArgs &a, bool half, void *scratch, hipStream_t st) {
    (void)scratch;
    const dim3 grid(a.s.rows, a.n_heads);
    if (half) hipLaunchKernelGGL(k_attn_row<_Float16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_attn_row<float>, grid, dim3(256), 0, st, a);
}

}  // namespace tg
