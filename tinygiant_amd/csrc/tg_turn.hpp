/*
 * tg_turn.hpp -- how a lane turns its part of a head (tg_rope.hip,
 * tg_paged.hip).
 */
#ifndef TG_TURN_HPP
#define TG_TURN_HPP
#include <hip/hip_runtime.h>

#include "tg_paged.h"

namespace tg {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   /* rows need only 4-byte alignment */
typedef double d4 __attribute__((ext_vector_type(4)));

/* Lane l's eight values of a head: dims a .. a + 3 and b .. b + 3, which hold
 * pairs 4 l .. 4 l + 3 whole.  turn.dim is a multiple of 8, so behind the
 * turned part both layouts are eight dims in a row. */
struct Pieces {
    int a, b;
    bool turned;
};
__device__ inline Pieces turn_pieces(const Turn &t, int l) {
    const bool turned = t.cos && 8 * l < t.dim;
    if (turned && !t.inter) return Pieces{4 * l, t.dim / 2 + 4 * l, true};
    return Pieces{8 * l, 8 * l + 4, turned};
}

/* (x, y) <- (x c - y s, y c + x s) for the four pairs of a lane */
template <typename V>
__device__ inline void turn_pair(bool inter, const V &c, const V &s, V &x, V &y) {
    if (inter) {
        const V a = {x[0], x[2], y[0], y[2]}, b = {x[1], x[3], y[1], y[3]};
        const V u = a * c - b * s, w = b * c + a * s;
        x = V{u[0], w[0], u[1], w[1]};
        y = V{u[2], w[2], u[3], w[3]};
    } else {
        const V u = x * c - y * s;
        y = y * c + x * s;
        x = u;
    }
}

}  // namespace

}  // namespace tg
#endif
