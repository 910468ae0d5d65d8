"""GPU checks of packed attention over f32 caches whose values lie far apart or
at the ends of f32's range, dimension by dimension against 64 bits."""

import sys

import numpy as np
import pytest

from tests._packed import EPS, Batch, Dev

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


def _one_position(q, k, at=20):
    """Nearly all of the weight on one position, for the rows that see it."""
    q[:, :, 1], k[:, at, 1] = 4.0, 8.0 * q.shape[-1] ** 0.5


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_channels_of_different_sizes(tg, hd, shape):
    """One channel far above the others at every position: in K, where q has a
    zero for it, and in V, where each channel is an output of its own; and one
    far below the others.  A little: the matrix units' path.  A lot: f32."""
    for power in (10, 30, 80):
        q, k, v = _inputs(hd + shape[2], shape, hd)
        q[:, :, 7] = 0
        k[:, :, 7] *= np.float32(2.0 ** power)
        say(f"channels {shape} hd={hd} K 2^{power}")
        say(f"  worst error / tolerance {_check(_attend(tg, q, k, v), q, k, v, weights=power == 10):.3f}")
    for power in (10, 30, 80, -10, -20, -60):
        q, k, v = _inputs(hd + shape[2], shape, hd)
        _one_position(q, k)
        v[:, :, 7] *= np.float32(2.0 ** power)
        say(f"channels {shape} hd={hd} V 2^{power}")
        say(f"  worst error / tolerance {_check(_attend(tg, q, k, v), q, k, v, weights=abs(power) == 10):.3f}")


@pytest.mark.parametrize("hd", [64, 72, 128])
def test_channels_of_zeros(tg, hd):
    """Channels that are zeros throughout, and in some groups only, are none
    of different sizes; beside infinities that no row sees, channels still are."""
    shape = (8, 2, 130, 300)
    q, k, v = _inputs(hd, shape, hd)
    _one_position(q, k)
    k[:, :, 9], v[:, :, 9] = 0, 0
    k[:, 40:200, 11], v[:, 64:72, 12:15] = 0, 0
    say(f"channels of zeros hd={hd}")
    got = _attend(tg, q, k, v)
    _check(got, q, k, v)
    assert np.all(got[:, :, 9] == 0)
    q, k, v = _inputs(hd, shape, hd)
    _one_position(q, k)
    v[:, :, 7] *= np.float32(2.0 ** -20)
    ref = v.copy()
    k[:, -1], v[:, -1] = np.inf, np.nan   # the last row's alone
    say("  beside infinities")
    got = _attend(tg, q, k, v)
    assert np.isnan(got[-1]).all()
    _check(got[:-1], q[:-1], k[:, :-1], ref[:, :-1], weights=False)


@pytest.mark.parametrize("hd", [64, 128])
def test_channels_of_few_positions(tg, hd):
    """A shared prefix of fewer positions than share a scale.  A channel of V
    that is 2^-30 throughout is the same computation, times that."""
    for prefix in (1, 5, 7, 13):
        say(f"channels of a prefix of {prefix} hd={hd}")
        b = Batch(prefix + hd, 8, 2, hd, [1] * 70, [i % 3 for i in range(70)], False, prefix=prefix)
        ref, tol = b.attend()
        for t in (b.v, b.pv):
            t[..., 7] *= np.float32(2.0 ** -30)
        dev = Dev(tg)
        tg.lib().tg_hip_clear_error()
        out, _ = b.call(dev)
        tg.lib().tg_hip_synchronize()
        assert tg.last_error() == "", tg.last_error()
        got = dev.read(out, b.q).astype(np.float64)
        dev.free()
        got.reshape(b.rows, 8, hd)[:, :, 7] *= 2.0 ** 30
        assert np.all(np.abs(got - ref) <= tol), float((np.abs(got - ref) / tol).max())


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_powers_of_two_between_queries_and_keys(tg, hd, shape):
    """A power of two taken from q and given to K changes no bit of the scores,
    nor of the way they are computed: rows of small queries, whose last tile
    ends inside a group, are not computed value by value."""
    q, k, v = _inputs(hd + shape[2], shape, hd)
    say(f"powers of two {shape} hd={hd}")
    first = _attend(tg, q, k, v)
    _check(first, q, k, v)
    for power in (-60, -20, 20, 45, 60, 80):
        got = _attend(tg, q * np.float32(2.0 ** -power), k * np.float32(2.0 ** power), v)
        assert got.tobytes() == first.tobytes(), power


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lens,past", [([40], [300]), ([2], [300]), ([300], [0])])
def test_queries_of_different_sizes(tg, lens, past, half):
    """One dimension of q far above the others, where K is 0: q keeps 2^-39 of
    its head's largest magnitude, so scores are off by that times the sum of
    |k|, beside what they are off without it."""
    for power in (10, 18, 24):
        say(f"queries {lens} half={half} 2^{power}")
        b = Batch(power, 8, 2, 64, lens, past, half, q_scale=0.5)
        q = b.q.reshape(b.rows, 8, 64)
        b.k[..., 7], q[:, :, 7] = 0, 0
        ref, tol = b.attend()
        q[:, :, 7] = 2.0 ** power
        off = 2.0 ** (power - 39) * np.abs(b.k[b.slots[0], :, :b.lens[0] + b.past[0]].astype(np.float64)).sum(-1).max() / 8
        tol = tol + 2 * off * np.abs(b.v[b.slots[0], :, :b.lens[0] + b.past[0]].astype(np.float64)).max()
        dev = Dev(tg)
        tg.lib().tg_hip_clear_error()
        out, was = b.call(dev)
        tg.lib().tg_hip_synchronize()
        assert tg.last_error() == "", tg.last_error()
        got = dev.read(out, b.q)
        dev.free()
        say(f"  worst error / tolerance {b.check(got, was, (ref, tol)):.3f}")
