/*
 * tg_rope.hip -- rotary positions: tables of cosines and sines, rows turned.
 *
 * The reference's engine makes one table on the host and turns whole heads in
 * half layout (apply_rope_inplace, csrc/libtinygiant.c:702-719).
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_paged.h"
#include "tg_turn.hpp"

namespace tg {

/* ---- tables ----
 * cos and sin of 2 pi t, t = position * (frequency / 2 pi) turns.  t is a
 * product in 64 bits, off by 2^-53 of itself and by as much again from the
 * rounded frequency.  Its nearest quarter is taken off, which is exact, and the rest,
 * at most an eighth of a turn, goes through the Taylor sums of both functions
 * in 64 bits to below 2^-50.  So what is stored is off by half an f32 step of
 * the value and by a few 2^-53 of the angle: of the fastest pair 2e-10 at
 * position 2^20 (one entry in some 2,000 is not the nearest f32; a sine near 0 has
 * steps smaller than that) and 2e-7 at 2^30; a 32-bit product is off by 0.06 turns
 * at 2^20.  A lane has four pairs of a position, 16 bytes of each table.
 * Bound: the stores, beside about 30 64-bit operations a pair. */
__device__ inline void turn_of(double t, double &c, double &s) {
    t -= __builtin_rint(t);
    const double k = __builtin_rint(4.0 * t);
    const double x = (t - 0.25 * k) * 6.283185307179586476925, y = x * x;
    double p = -7.6471637318198165e-13;                 /* -1 / 15! */
    p = fma(p, y, 1.6059043836821614e-10);
    p = fma(p, y, -2.5052108385441719e-08);
    p = fma(p, y, 2.7557319223985893e-06);
    p = fma(p, y, -1.9841269841269841e-04);
    p = fma(p, y, 8.3333333333333333e-03);
    p = fma(p, y, -1.6666666666666666e-01);
    const double sn = fma(x * y, p, x);
    double q = 4.7794773323873853e-14;                  /* 1 / 16! */
    q = fma(q, y, -1.1470745597729725e-11);
    q = fma(q, y, 2.0876756987868099e-09);
    q = fma(q, y, -2.7557319223985891e-07);
    q = fma(q, y, 2.4801587301587302e-05);
    q = fma(q, y, -1.3888888888888889e-03);
    q = fma(q, y, 4.1666666666666664e-02);
    q = fma(q, y, -0.5);
    const double cs = fma(q, y, 1.0);
    const int n = (int)k;   /* -2 .. 2 quarters */
    const double a = n & 1 ? sn : cs, b = n & 1 ? cs : sn;
    c = n == 1 || n == 2 || n == -2 ? -a : a;
    s = n == -1 || n == 2 || n == -2 ? -b : b;
}

/* A lane has ROWS positions in a row.  Those behind the first are turned on by
 * one position's angle, four products each instead of both sums, off by 2^-53 a
 * step: 131,072 positions of 32 pairs 8.8 us in the kernel with four, 11.4 with one
 * (calls 8.0 and 9.9); 4,096 of 64, where there are too few lanes then, 3.5 and 3.0
 * (calls 5.2). */
template <int ROWS>
__global__ __launch_bounds__(256) void k_rope_tables(RopeTablesArgs a) {
    const unsigned per = (unsigned)a.pairs / 4, at = blockIdx.x * 256 + threadIdx.x, group = at / per;
    const int row0 = ROWS * (int)group, i = 4 * (int)(at - group * per);
    if (row0 >= a.len) return;
    const double pos = (double)((long long)a.first + row0), m = (double)a.mscale;
    double x[4], y[4], c1[4], s1[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        turn_of(pos * a.turns[i + e], x[e], y[e]);
        x[e] *= m, y[e] *= m;
        if (ROWS > 1) turn_of(a.turns[i + e], c1[e], s1[e]);
    }
#pragma unroll
    for (int n = 0; n < ROWS; n++) {
        if (row0 + n >= a.len) return;
        f4 c, s;
#pragma unroll
        for (int e = 0; e < 4; e++) c[e] = (float)x[e], s[e] = (float)y[e];
        const size_t to = (size_t)(row0 + n) * a.pairs + i;
        *(f4u *)(a.cos + to) = c;
        *(f4u *)(a.sin + to) = s;
#pragma unroll
        for (int e = 0; ROWS > 1 && e < 4; e++) {
            const double u = x[e] * c1[e] - y[e] * s1[e];
            y[e] = y[e] * c1[e] + x[e] * s1[e];
            x[e] = u;
        }
    }
}

void launch_rope_tables(const RopeTablesArgs &a, hipStream_t st) {
    const long long n = (long long)a.len * (a.pairs / 4);
    if (n < 4 * 256 * 512) {   /* two workgroups a CU */
        hipLaunchKernelGGL((k_rope_tables<1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    } else {
        const long long lanes = (long long)((a.len + 3) / 4) * (a.pairs / 4);
        hipLaunchKernelGGL((k_rope_tables<4>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, st, a);
    }
}

/* ---- rows ----
 * A lane takes eight values of a head in two pieces of four that hold whole
 * pairs (turn_pieces), so that nothing is exchanged and out may be x.  A
 * workgroup has 256 such units of a row's.  Bound: the rows' bytes. */
__global__ __launch_bounds__(256) void k_rope(RopeArgs a) {
    const int per = a.head_dim / 8;   /* units of a head */
    const int u = (int)blockIdx.y * 256 + (int)threadIdx.x, r = (int)blockIdx.x;
    if (u >= a.heads * per) return;
    const int pos = a.pos[r];
    if (pos < 0 || pos >= a.turn.len) return;
    const int h = u / per, l = u - h * per;
    const Pieces p = turn_pieces(a.turn, l);
    const float *src = a.x + (size_t)r * a.x_stride + (size_t)h * a.head_dim;
    float *dst = a.out + (size_t)r * a.out_stride + (size_t)h * a.head_dim;
    f4 x = *(const f4u *)(src + p.a), y = *(const f4u *)(src + p.b);
    if (p.turned) {
        const f4 c = *(const f4u *)(a.turn.cos + (size_t)pos * (a.turn.dim / 2) + 4 * l);
        const f4 s = *(const f4u *)(a.turn.sin + (size_t)pos * (a.turn.dim / 2) + 4 * l);
        turn_pair(a.turn.inter, c, s, x, y);
    }
    *(f4u *)(dst + p.a) = x;
    *(f4u *)(dst + p.b) = y;
}

void launch_rope(const RopeArgs &a, hipStream_t st) {
    const int units = a.heads * (a.head_dim / 8);
    hipLaunchKernelGGL(k_rope, dim3((unsigned)a.rows, (unsigned)((units + 255) / 256)), dim3(256), 0, st, a);
}

}  // namespace tg
