"""GPU checks of paged attention where queries are not finite beside sinks, and
where scores are larger than f32 has room for a weight's exponent beside them."""

import numpy as np
import pytest

from tests._packed import EPS, Dev
from tests._paged import attend
from tests.test_gpu_paged import Attend, done, say

pytestmark = pytest.mark.gpu

# of several workgroups' shapes, cut into spans and not
CALLS = [
    (64, 8, 64, [1], [5000]), (32, 4, 128, [1, 1, 7], [900, 2000, 40]), (64, 8, 64, [100], [8000]), (32, 4, 128, [250], [3000]),
    (64, 1, 128, [500], [11]), (64, 8, 64, [500, 1, 3, 20], [2500, 60, 700, 300]), (32, 4, 128, [300, 20, 1], [1500, 900, 2000])]


def some_rows(a, rows):
    return {int(r): range(a.nh) for r in rows}


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("nh,nkv,hd,lens,past", CALLS)
def test_queries_not_finite_beside_sinks(tg, nh, nkv, hd, lens, past, bad):
    """All rows of the first sequence, or four that fill a wave's places: NaN in every head, whatever the sinks add, also where
    their own positions' blocks are NaN; the other rows are what they are without them."""
    for rows in (range(lens[0]), range(4, 8)):
        if rows[-1] >= lens[0]:
            continue
        rows = list(rows)
        for blocks in (False, True):
            say(f"attention {nh, nkv, hd, lens, past} rows {rows[:1]}.. q={bad} blocks={blocks}")
            a = Attend(41, nh, nkv, hd, lens, past, 32, sinks=True)
            a.q[rows, 5::hd] = bad
            if blocks:   # as the append of such rows leaves them: later rows of the sequence are NaN, too
                for j in range((past[0] + rows[0]) // 16, (past[0] + rows[-1]) // 16 + 1):
                    a.pages.ek[a.pages.table[0, 16 * j // 32], :, 16 * j % 32 // 16] = 255
            dev = Dev(tg)
            a.call(dev)
            done(tg)
            got = dev.read(a.out, a.q)
            assert np.isnan(got[rows]).all(), int((~np.isnan(got[rows])).sum())
            gone = lens[0] if blocks else len(rows)
            rest = [r for r in range(a.rows) if r not in rows and (not blocks or r >= gone)]
            rest = sorted({*rest[:2], *rest[len(rest) // 2:len(rest) // 2 + 1], *rest[-2:]})
            if rest:
                want, tol = attend(a.q, a.pages, a.cu, lens, past, nh, sinks=a.sinks, only=some_rows(a, rest))
                assert np.all(np.abs(got[rest] - want[rest]) <= tol[rest])
            dev.free()


def large_scores(seed, nh, nkv, hd, lens, past, powers):
    """Scores of 2^24 and more in base 2 (1.2e7) that f32 holds: q is 2^p in one dimension and 2^(p - 17) in the next, K a number
    of 64 .. 127 and one that rises in steps along the positions.  Their sums have 24 bits in every kernel's units, so that no product or
    sum of a score is rounded, only the factor log2 e / sqrt(head_dim), alike for all of a row's positions."""
    a = Attend(seed, nh, nkv, hd, lens, past, 32)
    rng, p = a.rng, a.pages
    p.k[:] = 0
    p.ek[:] = 127
    for s in range(a.n):
        n = lens[s] + past[s]
        for h in range(nkv):
            first = rng.integers(64, 128)
            rise = -120 + np.cumsum(np.where(rng.random(n) < 0.1, rng.integers(1, 13, n), 0))
            rise = np.where(rise > 127, rng.integers(100, 128, n), rise)   # the whole way up, then mixed
            for t in range(n):
                page, i = p.table[s, t // 32], t % 32
                p.k[page, h, i, 0], p.k[page, h, i, 1] = first, rise[t]
    a.q[:] = 0
    for r in range(a.rows):
        for h in range(nh):
            at = 2.0 ** powers[(r + h) % len(powers)]
            a.q[r, h * hd], a.q[r, h * hd + 1] = at, at * 2.0 ** -17
    return a


def chosen(a):
    rows = {0, a.rows - 1, *(int(c) for c in a.cu[:-1]), *(int(c) - 1 for c in a.cu[1:]), *range(a.rows // 2, a.rows // 2 + 3)}
    return some_rows(a, [r for r in rows if 0 <= r < a.rows])


@pytest.mark.parametrize("powers", [(19, 20), (20, 21, 22)])
@pytest.mark.parametrize("nh,nkv,hd,lens,past", CALLS + [(64, 1, 64, [1100], [0]), (64, 2, 128, [2100], [0])])
def test_large_scores(tg, nh, nkv, hd, lens, past, powers):
    """Differences of scores, of which those up to 40 count (2^-40 of a weight is nothing), are off by the factor's three
    roundings and one of their own, 40 (3 + 1) EPS, for numerator and denominator each and log 2 to the base e; the rest as for
    other scores."""
    say(f"attention of large scores {nh, nkv, hd, lens, past} {powers}")
    a = large_scores(42, nh, nkv, hd, lens, past, powers)
    dev = Dev(tg)
    a.call(dev)
    done(tg)
    got, only = dev.read(a.out, a.q), chosen(a)
    want, _ = attend(a.q, a.pages, a.cu, lens, past, nh, only=only)
    rows = sorted(only)
    n = a.longest
    big = max(np.abs(a.pages.values("v", s, lens[s] + past[s])).max() for s in range(a.n))
    tol = (2 * 40 * 4 * EPS + (8 * np.sqrt(n) + 24) * EPS + n * 2.0 ** -31) * big
    assert np.all(np.isfinite(got[rows])), [(r, int((~np.isfinite(got[r])).sum())) for r in rows]
    err = np.abs(got[rows] - want[rows])
    assert np.all(err <= tol), (float(err.max()), tol)
    dev.free()


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [18, 20, 24, 27, 31, 60, 115])
@pytest.mark.parametrize("nh,nkv,hd,lens,past", CALLS)
def test_scores_far_apart(tg, nh, nkv, hd, lens, past, power, sign, sinks):
    """Scores up to 2^120 whose least difference is 2^-7 of them: up to 2^27 in base 2 the largest takes all of the softmax, several
    that are equal share it, and what is off is the rounding of the weights and of sums of n of them. Past 2^27 a row is
    NaN, and where all are below -2^27 the sink's weight is all that is left, or nothing."""
    say(f"attention of scores far apart {nh, nkv, hd, lens, past} 2^{power} {sign} sinks={sinks}")
    a = Attend(43, nh, nkv, hd, lens, past, 32, sinks=sinks)
    a.pages.k[:] = 0
    a.pages.ek[:] = 127
    a.pages.k[..., 0] = a.rng.integers(1, 128, a.pages.k.shape[:-1])
    a.q[:] = 0
    a.q[:, :nh * hd:hd] = sign * 2.0 ** power
    dev = Dev(tg)
    a.call(dev)
    done(tg)
    got, only = dev.read(a.out, a.q), chosen(a)
    want, _ = attend(a.q, a.pages, a.cu, lens, past, nh, sinks=a.sinks, only=only)
    for s in range(a.n):
        keys = a.pages.values("k", s, lens[s] + past[s])[:, :, 0]
        for r in only:
            if a.cu[s] <= r < a.cu[s + 1]:
                z = sign * 2.0 ** power * keys[:, :past[s] + r - a.cu[s] + 1].astype(np.float64) * hd ** -0.5 / np.log(2)
                top = np.repeat(z.max(1), nh // nkv)
                assert np.all(np.abs(np.abs(top) - 2.0 ** 27) > 2.0 ** 20)
                want[r].reshape(nh, hd)[(top > 2.0 ** 27) | ((top < -2.0 ** 27) & (not sinks))] = np.nan
    rows = sorted(only)
    big = max(np.abs(a.pages.values("v", s, lens[s] + past[s])).max() for s in range(a.n))
    tol = ((8 * np.sqrt(a.longest) + 24) * EPS + a.longest * 2.0 ** -31) * big
    assert np.array_equal(np.isnan(got[rows]), np.isnan(want[rows])), (int(np.isnan(got[rows]).sum()), int(np.isnan(want[rows]).sum()))
    err = np.nan_to_num(np.abs(got[rows] - want[rows]))
    assert np.all(err <= tol), (float(err.max()), tol)
    dev.free()


@pytest.mark.parametrize("nh,nkv,hd,rows,n,past,fill", [
    (32, 4, 128, 600, 9, 9000, 0x7F), (32, 4, 128, 600, 9, 9000, 0x00), (64, 8, 64, 500, 20, 900, 0xFF), (32, 4, 128, 40, 30, 4000, 0x11),
    (64, 8, 64, 3, 41, 6000, 0x01), (32, 4, 128, 700, 90, 2000, 0x01)])
def test_offsets_that_overlap(tg, nh, nkv, hd, rows, n, past, fill):
    """Offsets 0, R, 0, R, ... are no packed rows, and what comes out is nothing; but every other sequence has all rows, many
    more spans than a call of so many rows has room for, and nothing may be read or written outside the arrays, whatever
    the scratch held."""
    say(f"attention of overlapping sequences {nh, nkv, hd, rows, n, past} scratch {fill:#x}")
    lens = [rows // n] * n
    lens[0] += rows - sum(lens)
    a = Attend(44, nh, nkv, hd, lens, [past] * n, 64, room=rows)
    a.cu = (rows * (np.arange(n + 1) % 2)).astype(np.int32)
    dev, lib = Dev(tg), tg.lib()
    size = lib.tg_hip_attention_paged_scratch_bytes(a.rows, n, nh, nkv, hd, a.max_kv)
    assert size
    a.call(dev)   # in scratch that holds anything
    was = np.full(size + 64, fill, np.uint8)
    scratch = dev(was)
    a.args = (*a.args[:-1], scratch)
    a.queue(lib)
    done(tg)
    assert np.array_equal(dev.read(a.after, a.guard), a.guard) and np.array_equal(dev.read(scratch, was)[size:], was[size:])
    dev.free()


@pytest.mark.parametrize("nh,nkv,hd,n", [(64, 8, 64, 128), (32, 4, 128, 200), (8, 2, 80, 300)])
def test_a_deep_chunk_among_single_tokens(tg, nh, nkv, hd, n):
    """With and without cuts of the chunk, by how many sequences and KV heads there are."""
    say(f"attention of a chunk among {n} sequences {nh, nkv, hd}")
    rng = np.random.default_rng(45)
    lens, past = [1] * n, [int(x) for x in rng.integers(0, 700, n)]
    lens[n // 3], past[n // 3] = 500 if nh > 8 else 2000, 4000
    lens[n // 2] = 0
    a = Attend(45, nh, nkv, hd, lens, past, 64, sinks=True, lead=1, tail=2)
    at = int(a.cu[n // 3])
    only = some_rows(a, [1, at - 1, at, at + 1, at + 250, at + lens[n // 3] - 1, at + lens[n // 3], a.rows - 3])
    want, tol = attend(a.q, a.pages, a.cu, lens, past, nh, sinks=a.sinks, only=only)
    dev = Dev(tg)
    a.call(dev)
    for again in range(3):   # in scratch that holds a call's records
        done(tg)
        got, rows = dev.read(a.out, a.q), sorted(only)
        assert np.all(np.abs(got[rows] - want[rows]) <= tol[rows])
        assert np.all(np.isfinite(got[1:-2])) and np.all(got[[0, -2, -1]] == 7.0)
        assert np.array_equal(dev.read(a.after, a.guard), a.guard)
        a.queue(tg.lib())
    done(tg)
    dev.free()
