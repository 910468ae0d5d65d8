"""GPU checks of packed attention over f32 caches whose values lie far apart or
at the ends of f32's range, dimension by dimension against 64 bits."""

import sys

import numpy as np
import pytest

from tests._packed import EPS, Dev

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


# query heads, KV heads, rows, cached before them: tiles of 128 rows of one and of two groups of waves, of 256, few rows
SHAPES = [(8, 2, 40, 300), (8, 2, 130, 0), (8, 2, 600, 700), (64, 8, 520, 16100), (8, 2, 2, 300)]


def _inputs(seed, shape, hd, q_scale=0.5):
    nh, nkv, rows, past = shape
    rng = np.random.default_rng(seed)
    q = (rng.standard_normal((rows, nh, hd)) * q_scale).astype(np.float32)
    k, v = rng.standard_normal((2, nkv, past + rows, hd)).astype(np.float32)
    return q, k, v


def _attend(tg, q, k, v):
    """The rows of one sequence, the last of the cache's positions."""
    (rows, nh, hd), (nkv, n, _) = q.shape, k.shape
    lib, dev = tg.lib(), Dev(tg)
    out = dev(np.full_like(q, 7.5))
    scratch = dev.room(lib.tg_hip_attention_prompt_scratch_bytes(rows, 1, nh, nkv, hd, n, 0))
    lib.tg_hip_clear_error()
    lib.tg_hip_attention_prompt_dev(dev(q), nh * hd, 0, dev(k), dev(v), 1, n, dev(np.array([0, rows], np.int32)),
                                    dev(np.array([n - rows], np.int32)), None, 1, rows, 0, None, nh, nkv, hd, out, nh * hd,
                                    scratch, None)
    lib.tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    got = dev.read(out, q)
    dev.free()
    return got


def _check(got, q, k, v, weights=True):
    """Some rows and heads, every dimension by itself.

    A score is off by `off`: the products and sums of f32 (tests/_packed.py).
    A weight is off by that, relative to itself, and so is their sum: 2 off
    times the weighted mean of |v|.  `weights`: where the matrix units take
    them, they are besides off by up to 2^-25 of the largest weight, and V by
    2^-27 of the dimension's largest value (2^-39 of the largest of its
    neighbours, which may be 2^12 larger).  Sums end at f32's smallest step."""
    (rows, nh, hd), (nkv, n, _) = q.shape, k.shape
    worst = 0.0
    for r in sorted({0, 1, rows // 2, rows - 2, rows - 1} & set(range(rows))):
        for h in sorted({0, nh // 2 + 1, nh - 1}):
            m = n - rows + r + 1
            kk, vv, qq = k[h * nkv // nh, :m].astype(np.float64), v[h * nkv // nh, :m].astype(np.float64), q[r, h].astype(np.float64)
            z = kk @ qq * hd ** -0.5
            p = np.exp(z - z.max())
            off = (8 * np.sqrt(2 * hd) + 4) * EPS * (np.abs(kk) @ np.abs(qq)).max() * hd ** -0.5 + (8 * np.sqrt(m) + 24) * EPS
            tol = 2 * off * (p @ np.abs(vv)) / p.sum() + 4 * m * 2.0 ** -149
            if weights:
                tol = tol + (m * 2.0 ** -25 + 2.0 ** -27) * np.abs(v[h * nkv // nh]).max(0)
            err = np.abs(got[r, h] - (p @ vv) / p.sum())
            assert np.all(err <= tol), (r, h, float((err / tol).max()), float(err.max()))
            worst = max(worst, float((err / tol).max()))
    return worst


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_tiny_values_among_ordinary_ones(tg, hd, shape):
    """16 adjacent positions (whole groups that share a scale) of tiny V, which
    hold nearly all of the weight: what the others' scale makes of them shows."""
    for size in (1e-24, 2e-26, 7e-27, 1e-30):
        q, k, v = _inputs(hd + shape[2], shape, hd)
        at = slice(16, 32)
        q[:, :, 0], k[:, at, 0] = 4.0, 8.0 * hd ** 0.5   # these scores are 32 above the others
        v[:, at] *= np.float32(size)
        say(f"tiny V {shape} hd={hd} size={size}")
        say(f"  worst error / tolerance {_check(_attend(tg, q, k, v), q, k, v, weights=False):.3f}")


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_tiny_caches(tg, hd, shape):
    """All of V tiny, down to f32's smallest normal values, and all of K, with
    queries that make ordinary scores of them."""
    for size in (1e-24, 1e-26, 1e-30, 1e-34, 2e-37):
        q, k, v = _inputs(hd + shape[2], shape, hd)
        v *= np.float32(size)
        say(f"tiny caches {shape} hd={hd} V {size}")
        _check(_attend(tg, q, k, v), q, k, v)
    for power in (80, 90, 110, 120):
        q, k, v = _inputs(hd + shape[2], shape, hd)
        q, k = q * np.float32(2.0 ** power), k * np.float32(2.0 ** -power)
        say(f"tiny caches {shape} hd={hd} K 2^-{power}")
        _check(_attend(tg, q, k, v), q, k, v)
