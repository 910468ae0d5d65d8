/*
 * tg_logits.hip -- penalties for repeated tokens, biases and a grammar's mask
 * on rows of logits, with the argmax of the result.
 *
 *   l = l > 0 ? l / r : l r          tokens in the row's history
 *   l = l - f c - p                  tokens generated c > 0 times
 *   l = l + b                        tokens with a bias
 *   l = -inf                         tokens whose bit is 0
 *
 * each step one correctly rounded f32 operation (products, differences and
 * quotients are not contracted), so the results are the formulas' bits.
 *
 * A workgroup takes a slice of one row's tokens.  It scans the row's whole
 * history and bias list and counts those that fall into its slice in LDS
 * (integer atomics: the order does not matter), so no table of the
 * vocabulary's size is cleared, written and read in memory; a history is at
 * most some ten KB, which the slices of a row read from L2.  Then one pass
 * over the slice's logits, which were requested before the scan.  The largest
 * value's key goes to the slice's word of the scratch; k_logits_pick takes the
 * row's best.
 *
 * Bound: the bytes of the logits, read and written.  64 rows of 151,936 with
 * histories of 4,000, 300 biases and masks: 26 us, 80 MB (3.1 TB/s; with four
 * times the scans and one token a load 32).  One row: two launches.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_device.hpp"
#include "tg_logits.h"

namespace tg {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i4u __attribute__((ext_vector_type(4), aligned(4)));

/* Values in the order of unsigned words above 0: -0 ties with +0, a NaN of
 * either sign is the largest (numpy.argmax's rules). */
__device__ inline uint32_t pick_order(float v) {
    uint32_t u = v == 0.f ? 0u : __float_as_uint(v);
    u = v != v ? 0x7FC00000u : u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t KEY_NEG_INF = ~0xFF800000u;

__device__ inline uint64_t wave_max_key(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), o, 64);
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, o, 64);
        const uint64_t w = ((uint64_t)hi << 32) | lo;
        v = w > v ? w : v;
    }
    return v;
}

}  // namespace

template <int SLICE, int LT>
__global__ __launch_bounds__(LT) void k_logits_adjust(LogitsArgs a, int nslices, uint64_t *best) {
#pragma clang fp contract(off)
    constexpr int N = SLICE / (4 * LT);   /* groups of four logits a thread */
    __shared__ __attribute__((aligned(16))) int cnt[SLICE];    /* times generated; bit 30: in the history's first part */
    __shared__ __attribute__((aligned(16))) int last[SLICE];   /* 1 + the place of the token's last bias entry */
    __shared__ uint64_t red[LT / 64];
    const int j = blockIdx.y, t0 = blockIdx.x * SLICE, tid = threadIdx.x;
    const int n = min(SLICE, a.nrows - t0);
    const int hl = a.hist ? min(max(a.hist_len[j], 0), a.hist_stride) : 0;
    const int bl = a.bias_tok ? min(a.bias_len ? max(a.bias_len[j], 0) : a.bias_stride, a.bias_stride) : 0;
    const float *src = a.logits + (size_t)j * a.nrows + t0;
    f4 v[N];   /* requested before the lists are read */
#pragma unroll
    for (int q = 0; q < N; q++) {
        const int i = 4 * (tid + q * LT);
        if (i + 4 <= n) v[q] = *(const f4u *)(src + i);
        else
            for (int e = 0; e < 4; e++) v[q][e] = i + e < n ? src[i + e] : 0.f;
    }
    const i4 zero = {0, 0, 0, 0};
    if (hl)
        for (int i = tid; i < SLICE / 4; i += LT) *(i4 *)&cnt[4 * i] = zero;
    if (bl)
        for (int i = tid; i < SLICE / 4; i += LT) *(i4 *)&last[4 * i] = zero;
    __syncthreads();
    if (hl) {
        const int gs = a.gen_start ? a.gen_start[j] : 0;
        const int32_t *h = a.hist + (size_t)j * a.hist_stride;
        auto count = [&](int token, int i) {
            const uint32_t t = (uint32_t)token - (uint32_t)t0;
            if (t < (uint32_t)n) {
                if (i >= gs) atomicAdd(&cnt[t], 1);
                else atomicOr(&cnt[t], 1 << 30);
            }
        };
        const int whole = hl & ~3;
        for (int i = 4 * tid; i < whole; i += 4 * LT) {
            const i4 t = *(const i4u *)(h + i);
#pragma unroll
            for (int e = 0; e < 4; e++) count(t[e], i + e);
        }
        if (tid < hl - whole) count(h[whole + tid], whole + tid);
    }
    if (bl) {
        const int32_t *bt = a.bias_tok + (size_t)j * a.bias_stride;
        for (int i = tid; i < bl; i += LT) {
            const uint32_t t = (uint32_t)bt[i] - (uint32_t)t0;
            if (t < (uint32_t)n) atomicMax(&last[t], i + 1);
        }
    }
    __syncthreads();
    const float rep = hl ? a.pen[3 * j] : 1.f, freq = hl ? a.pen[3 * j + 1] : 0.f, pres = hl ? a.pen[3 * j + 2] : 0.f;
    const float *bv = a.bias_val + (size_t)j * a.bias_stride;
    const uint32_t *al = a.allow ? a.allow + (size_t)j * a.allow_stride : nullptr;
    float *dst = a.out ? a.out + (size_t)j * a.nrows + t0 : nullptr;
    uint32_t top = 0, at = 0;   /* the largest so far and its place: a thread's places rise, so ties keep the first */
#pragma unroll
    for (int q = 0; q < N; q++) {
        const int i = 4 * (tid + q * LT);
        if (i >= n) break;
        const uint32_t bits = al ? al[(uint32_t)(t0 + i) >> 5] >> ((t0 + i) & 31) : 15u;
        const i4 c = hl ? *(const i4 *)&cnt[i] : zero, b = bl ? *(const i4 *)&last[i] : zero;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float x = v[q][e];
            if (c[e]) {
                x = x > 0.f ? x / rep : x * rep;
                const int g = c[e] & ((1 << 30) - 1);
                if (g) x = x - freq * (float)g - pres;
            }
            if (b[e]) x = x + bv[b[e] - 1];
            if (!((bits >> e) & 1u)) x = -INFINITY;
            v[q][e] = x;
            const uint32_t u = pick_order(x);
            if (i + e < n && u > top) top = u, at = (uint32_t)(t0 + i + e);
        }
        if (dst) {
            if (i + 4 <= n) *(f4u *)(dst + i) = v[q];
            else
                for (int e = 0; e < 4; e++)
                    if (i + e < n) dst[i + e] = v[q][e];
        }
    }
    if (!best) return;
    uint64_t mine = wave_max_key(((uint64_t)top << 32) | (uint64_t)(0xFFFFFFFFu - at));
    if ((tid & 63) == 0) red[tid >> 6] = mine;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < LT / 64; w++) mine = red[w] > mine ? red[w] : mine;
        best[(size_t)j * nslices + blockIdx.x] = mine;
    }
}

/* one wave a row: the best of its slices; -1 where nothing is above -inf */
__global__ __launch_bounds__(64) void k_logits_pick(const uint64_t *best, int nslices, int32_t *argmax, float *maxval) {
    const int j = blockIdx.x;
    uint64_t m = 0;
    for (int i = threadIdx.x; i < nslices; i += 64) {
        const uint64_t k = best[(size_t)j * nslices + i];
        m = k > m ? k : m;
    }
    m = wave_max_key(m);
    if (threadIdx.x) return;
    const uint32_t u = (uint32_t)(m >> 32);
    if (argmax) argmax[j] = u <= KEY_NEG_INF ? -1 : (int32_t)(0xFFFFFFFFu - (uint32_t)m);
    if (maxval) maxval[j] = __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}

/* Tokens of a slice: 2,048 with 256 threads, or 8,192 with 1,024 (a fourth of
 * the scans of the lists) where the rows alone fill the card and the lists are
 * long.  64 rows of 151,936 tokens: 22.7 against 23.4 us with histories of
 * 500, 30.6 against 27.3 with 8,000. */
constexpr int SMALL = 2048, LARGE = 8192;
size_t logits_scratch(int k, int nrows) { return (size_t)k * ((nrows + SMALL - 1) / SMALL) * 8; }

void launch_logits_adjust(const LogitsArgs &a, void *scratch, hipStream_t st) {
    const bool large = (long long)a.k * ((a.nrows + LARGE - 1) / LARGE) >= 512 &&
                       (a.hist ? a.hist_stride : 0) + (a.bias_tok ? a.bias_stride : 0) >= 2048;
    const int slice = large ? LARGE : SMALL, nslices = (a.nrows + slice - 1) / slice;
    uint64_t *best = a.argmax || a.maxval ? (uint64_t *)scratch : nullptr;
    const dim3 grid(nslices, a.k);
    if (large) hipLaunchKernelGGL((k_logits_adjust<LARGE, 1024>), grid, dim3(1024), 0, st, a, nslices, best);
    else hipLaunchKernelGGL((k_logits_adjust<SMALL, 256>), grid, dim3(256), 0, st, a, nslices, best);
    if (best) hipLaunchKernelGGL(k_logits_pick, dim3(a.k), dim3(64), 0, st, best, nslices, a.argmax, a.maxval);
}

}  // namespace tg
