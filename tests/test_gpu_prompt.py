"""GPU checks of the prompt and batch path (tg_hip_kv_append_dev,
tg_hip_attention_prompt_dev, tg_hip_attention_prefix_dev) against plain
computations in 64 bits; tolerances: tests/_packed.py."""

import ctypes
import sys

import numpy as np
import pytest

from tests._packed import EPS, Batch, Dev, Graph

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _run(tg, b, **kw):
    dev = Dev(tg)
    tg.lib().tg_hip_clear_error()
    out, was = b.call(dev, **kw)
    tg.lib().tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    got = dev.read(out, b.q)
    dev.free()
    return got, was


LAYOUTS = [(8, 2, 128), (32, 4, 128), (8, 1, 64), (4, 4, 32), (15, 3, 80), (6, 1, 8), (14, 2, 112), (40, 1, 16)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("lens,past", [
    ([1], [0]), ([1], [1]), ([5], [63]), ([0, 1, 3], [4, 0, 60]), ([33, 0, 64, 1], [0, 5, 1, 130]), ([130], [0]),
    ([17, 31], [100, 257]), ([1] * 9, [0, 1, 15, 16, 63, 64, 65, 127, 300])])
def test_prompt_matches_plain(tg, layout, lens, past, half):
    nh, nkv, hd = layout
    say(f"prompt {layout} lens={lens} past={past} half={half}")
    b = Batch(hash((nh, hd, len(lens), sum(lens))) % 2 ** 31, nh, nkv, hd, lens, past, half, sinks=nh % 4 != 0, lead=len(lens) % 3,
              tail=2, pad=4 * (nkv % 2))
    got, was = _run(tg, b)
    say(f"  worst error / tolerance {b.check(got, was):.3f}")


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 128, 1000])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_windows(tg, window, hd, half):
    say(f"prompt window={window} hd={hd} half={half}")
    b = Batch(window + hd, 8, 1, hd, [1, 90, 200], [500, 0, 77], half, window=window, sinks=hd == 64)
    got, was = _run(tg, b)
    b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,lens,past", [
    (32, 4, 128, [9], [4000]), (64, 8, 64, [3], [9000]), (8, 1, 128, [1], [20011]), (8, 2, 128, [600], [700]),
    (8, 8, 64, [257, 300], [511, 0]), (16, 2, 128, [1] * 12, [37 * i * i % 2900 for i in range(12)])])
def test_prompt_long(tg, nh, nkv, hd, lens, past, half):
    """Long caches: the positions are split over workgroups where rows are few."""
    say(f"prompt long {nh, nkv, hd} lens={lens} past={past[:3]} half={half}")
    b = Batch(sum(lens), nh, nkv, hd, lens, past, half, sinks=hd == 64)
    got, was = _run(tg, b)
    say(f"  worst error / tolerance {b.check(got, was):.3f}")


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("layout", [(8, 2, 128), (64, 8, 64), (15, 3, 80), (40, 1, 16)])
@pytest.mark.parametrize("prefix,lens,past,window", [
    (1, [1], [0], 0), (64, [1, 1, 1], [0, 3, 64], 0), (65, [2, 0, 5], [0, 1, 9], 0), (700, [1] * 20, list(range(20)), 0),
    (500, [1, 1, 4], [0, 100, 200], 150), (130, [1, 40], [300, 0], 128), (127, [3], [200], 16)])
def test_prefix_matches_plain(tg, layout, prefix, lens, past, window, half):
    nh, nkv, hd = layout
    say(f"prefix {layout} prefix={prefix} lens={lens} window={window} half={half}")
    b = Batch(prefix + nh, nh, nkv, hd, lens, past, half, window=window, sinks=nkv % 2 == 0, prefix=prefix, lead=1, tail=1)
    got, was = _run(tg, b)
    b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("layout", [(64, 8, 64), (32, 4, 128), (40, 1, 16)])
@pytest.mark.parametrize("prefix,window", [(600, 0), (300, 0), (600, 250)])
def test_prefix_of_a_batch(tg, layout, prefix, window, half):
    """One row of each of many sequences behind a prefix, a few of other
    lengths among them; f32 caches also with positions of very different
    sizes, in the prefix and in the sequences' own."""
    nh, nkv, hd = layout
    lens, past = [1] * 18 + [0, 2, 1], [100 + 7 * i for i in range(20)] + [0]
    for sizes in ([False] if half else [False, True]):
        say(f"prefix of a batch {layout} prefix={prefix} window={window} half={half} sizes={sizes}")
        b = Batch(prefix + nh, nh, nkv, hd, lens, past, half, window=window, sinks=nkv == 4, prefix=prefix, lead=1, tail=1)
        if sizes:
            b.pv[:, 3:prefix:40] *= np.float32(2.0 ** -20)
            b.v[:, :, 5::30] *= np.float32(2.0 ** -20)
            b.pk[:, 7:prefix:50] *= np.float32(2.0 ** -20)
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 20, 2 ** 20])
def test_window_longer_than_any_cache(tg, window, half):
    for lens, past, prefix in (([3, 40], [500, 9], 0), ([2, 1], [5, 70], 300)):
        say(f"window={window} half={half} prefix={prefix}")
        b = Batch(80, 8, 2, 64, lens, past, half, window=window, prefix=prefix)
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh,nkv,hd", [(1024, 16, 128), (1024, 1024, 8), (64, 1, 128), (1, 1, 128), (1024, 512, 16)])
def test_ends_of_the_layouts(tg, nh, nkv, hd, half):
    say(f"layout {nh, nkv, hd} half={half}")
    for lens, past, prefix in (([2, 1], [70, 0], 0), ([1], [600], 0), ([1, 3], [0, 20], 90)):
        b = Batch(nh + hd, nh, nkv, hd, lens, past, half, prefix=prefix, sinks=True)
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
def test_many_sequences(tg, half):
    """More sequences than one pass over them takes lanes, of few and no rows."""
    for n, prefix, window in ((200, 0, 0), (700, 40, 0), (700, 0, 16), (5000, 0, 0)):
        say(f"{n} sequences half={half}")
        b = Batch(n, 4, 2, 32, [i % 3 for i in range(n)], [(7 * i) % 40 + (900 if i == 150 else 0) for i in range(n)], half,
                  prefix=prefix, window=window, lead=3 * (n > 200), tail=1)
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
def test_out_over_q(tg, half):
    for kw in (dict(lens=[70, 3], past=[0, 9]), dict(lens=[2], past=[3000]), dict(lens=[1, 2], past=[5, 0], prefix=400)):
        say(f"out over q {kw} half={half}")
        b = Batch(3, 16, 2, 64, half=half, lead=1, tail=1, **kw)
        got, was = _run(tg, b, in_place=True)
        b.check(got, was)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_values_a_row_does_not_see(tg, hd, half, bad):
    """Infinities and NaN in K and V of positions behind a row, or in front of
    its window, leave the row as it is; rows that see a NaN in V are NaN."""
    say(f"unseen hd={hd} half={half} bad={bad}")
    for window, at in ((0, 100), (40, 100), (0, 149)):
        b = Batch(hd, 8, 2, hd, [140], [10], half, window=window)
        ref = b.attend()
        b.k[b.slots[0], :, at] = bad
        b.v[b.slots[0], :, at] = bad
        got, was = _run(tg, b)
        hit = np.array([lo <= at <= hi for lo, hi in (b.seen(0, i) for i in range(140))])
        err = np.abs(got[~hit] - ref[0][~hit])
        assert np.all(err <= ref[1][~hit]), float(np.nanmax(err))
        assert np.all(np.isnan(got[hit])) == bool(hit.any()) or not hit.any()


@pytest.mark.parametrize("half", [False, True])
def test_infinite_values(tg, half):
    """An infinity in V alone is the output of the rows that see it, in its
    dimension only, as the sum of weights times values gives it."""
    say(f"infinite V half={half}")
    for hd, lens, past in ((64, [70], [3]), (128, [2], [900])):
        b = Batch(5, 8, 2, hd, lens, past, half, q_scale=0.5)
        ref, tol = b.attend()
        at = past[0] + 1
        b.v[b.slots[0], :, at, 5] = np.inf
        b.v[b.slots[0], :, at, 9] = -np.inf
        got, was = _run(tg, b)
        g, r = got.reshape(b.rows, 8, hd), ref.reshape(b.rows, 8, hd)
        assert np.all(np.abs(g[:1] - r[:1]) <= tol.reshape(r.shape)[:1])
        assert np.all(g[1:, :, 5] == np.inf) and np.all(g[1:, :, 9] == -np.inf)
        rest = [d for d in range(hd) if d not in (5, 9)]
        assert np.all(np.abs(g - r)[:, :, rest] <= tol.reshape(r.shape)[:, :, rest])


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("q_scale", [1e-30, 1e-3, 300.0])
def test_score_ranges(tg, half, q_scale):
    """Queries so small that all weights are equal, and so large that one is all."""
    say(f"q_scale={q_scale} half={half}")
    for hd in (64, 128):
        b = Batch(11, 8, 2, hd, [50, 1], [20, 700], half, q_scale=q_scale, sinks=True)
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
def test_cache_ranges(tg, half):
    """Caches at the ends of their ranges: large values (f16's largest among
    them) and tiny ones, next to each other in a row."""
    say(f"cache ranges half={half}")
    big = 65504.0 if half else 3e6
    for hd in (64, 128):
        b = Batch(12, 8, 2, hd, [40, 1], [9, 500], half, q_scale=1e-4)
        for s in range(2):
            m = b.lens[s] + b.past[s]
            b.k[b.slots[s], :, :m, ::7] *= np.float32(big / 8)
            b.k[b.slots[s], :, :m, 1::7] *= np.float32(1e-4)
            np.clip(b.k, -big, big, out=b.k)
            b.v[b.slots[s], :, :m] *= np.float32(big / 8)
            np.clip(b.v, -big, big, out=b.v)
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("big", [3e38, 1e12, 7e4])
@pytest.mark.parametrize("hd", [64, 128])
def test_large_neighbours(tg, hd, big, what):
    """A position's huge but finite K or V (f32 caches) leaves the rows that do
    not see it as they are to their own precision: in front of it in one group
    of positions, in the next, and where a window has passed it."""
    say(f"large neighbours hd={hd} big={big} {what}")
    for lens, past, window, at in (([5], [0], 0, 4), ([40], [3], 0, 12), ([200], [0], 0, 150), ([60, 9], [100, 700], 30, 107)):
        b = Batch(hd, 8, 2, hd, lens, past, False, window=window, q_scale=0.5)
        ref, tol = b.attend()
        for name in "kv" if what == "both" else what:
            getattr(b, name)[b.slots[0], :, at] *= np.float32(big / 4)
        np.clip(b.k, -3e38, 3e38, out=b.k)
        np.clip(b.v, -3e38, 3e38, out=b.v)
        got, was = _run(tg, b)
        blind = np.zeros(b.rows, bool)
        for s in range(b.n):
            for i in range(b.lens[s]):
                lo, hi = b.seen(s, i)
                blind[b.cu[s] + i] = s != 0 or not lo <= at <= hi
        assert blind.any()
        err = np.abs(got - ref)[blind]
        assert np.all(err <= tol[blind]), float((err / tol[blind]).max())


@pytest.mark.parametrize("hd", [64, 128])
def test_values_of_many_sizes(tg, hd):
    """f32 caches whose positions differ by powers of two: a little (the matrix
    units' path), a lot (value by value); zeros count as neither."""
    for top, zero in ((10, False), (14, True), (40, True)):
        say(f"values of many sizes hd={hd} top={top}")
        b = Batch(hd + top, 8, 2, hd, [33, 4], [90, 300], False, q_scale=0.5)
        rng = np.random.default_rng(top)
        for s in range(2):
            m = b.lens[s] + b.past[s]
            for t in (b.k, b.v):
                t[b.slots[s], :, :m] *= np.exp2(-rng.integers(0, top, m)).astype(np.float32)[None, :, None]
                if zero:
                    t[b.slots[s], :, 5:17] = 0
        got, was = _run(tg, b)
        b.check(got, was)


@pytest.mark.parametrize("rows,past", [(9, 40), (60, 300), (300, 700), (1100, 0), (520, 16100)])
@pytest.mark.parametrize("hd", [64, 128])
def test_values_of_many_sizes_in_long_calls(tg, hd, rows, past):
    """As above where rows or positions are many: every tenth position is
    smaller by 2^20, in V or in K; some rows against 64 bits."""
    say(f"many sizes hd={hd} rows={rows} past={past}")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(rows + hd)
    nh, nkv, n = 64, 8, rows + past
    q = (rng.standard_normal((rows, nh, hd)) * 0.5).astype(np.float32)
    cache = rng.standard_normal((2, 1, nkv, n, hd)).astype(np.float32)
    for which in (0, 1):
        k, v = (x.copy() for x in cache)
        (k, v)[which][:, :, ::10] *= np.float32(2.0 ** -20)
        out = dev(np.zeros_like(q))
        scratch = dev.room(lib.tg_hip_attention_prompt_scratch_bytes(rows, 1, nh, nkv, hd, n, 0))
        lib.tg_hip_clear_error()
        lib.tg_hip_attention_prompt_dev(dev(q), nh * hd, 0, dev(k), dev(v), 1, n, dev(np.array([0, rows], np.int32)),
                                        dev(np.array([past], np.int32)), None, 1, rows, 0, None, nh, nkv, hd, out, nh * hd, scratch,
                                        None)
        lib.tg_hip_synchronize()
        assert tg.last_error() == "", tg.last_error()
        got = dev.read(out, q)
        for r in {0, 1, rows // 2, rows - 2, rows - 1}:
            for h in (0, 7, 40, 63):
                kk, vv = (x[0, h // 8, :past + r + 1].astype(np.float64) for x in (k, v))
                qq = q[r, h].astype(np.float64)
                z = kk @ qq * hd ** -0.5
                p = np.exp(z - z.max())
                off = (8 * np.sqrt(2 * hd) + 4) * EPS * (np.abs(kk) @ np.abs(qq)).max() * hd ** -0.5 + (8 * np.sqrt(len(z)) + 24) * EPS
                assert np.all(np.abs(got[r, h] - (p @ vv) / p.sum()) <= 2 * off * np.abs(vv).max()), (which, r, h)
    dev.free()


def test_sequences_that_do_not_fit_are_left_out(tg):
    """A slot out of range, a negative length, rows past kv_max: those
    sequences' rows stay as they were, the others are computed."""
    for key, vals in (("slots", (-1, 99, 2 ** 31 - 1)), ("kv_len", (-1, 10 ** 6, 2 ** 31 - 1))):
        for v in vals:
            for prefix in (0, 200):
                say(f"left out: {key}={v} prefix={prefix}")
                b = Batch(1, 8, 2, 64, [3, 4, 2], [50, 60, 70], False, prefix=prefix)
                ref = b.attend()
                getattr(b, key)[1] = v
                got, was = _run(tg, b)
                gone = slice(b.cu[1], b.cu[2])
                assert np.array_equal(got[gone], was[gone])
                keep = np.ones(b.rows, bool)
                keep[gone] = False
                assert np.all(np.abs(got[keep] - ref[0][keep]) <= ref[1][keep])


def test_bad_row_offsets_stay_in_bounds(tg):
    """Offsets past the rows and decreasing ones: what is computed of them is
    not specified, the call ends and the rows outside stay."""
    for cu in ([0, 5, 4000], [-7, 3, 6], [4, 2, 1]):
        say(f"row offsets {cu}")
        b = Batch(2, 8, 2, 64, [3, 4], [50, 60], False)
        b.cu = np.array(cu, np.int32)
        _run(tg, b)


def test_null_lengths_and_slots(tg):
    say("null kv_len and slots")
    b = Batch(4, 8, 2, 128, [20, 7], [0, 0], False)
    b.k, b.v = (np.concatenate([t[b.slots], t[:2]]) for t in (b.k, b.v))   # slot s is sequence s's
    b.slots = np.arange(2, dtype=np.int32)
    ref = b.attend()
    dev = Dev(tg)
    out, was = b.call(dev)
    b.ptrs["len"] = b.ptrs["slots"] = None
    b.queue(tg.lib())
    tg.lib().tg_hip_synchronize()
    b.check(dev.read(out, b.q), was, ref)
    dev.free()


@pytest.mark.parametrize("half", [False, True])
def test_replayed_graph(tg, half):
    """Captured once and replayed with other queries and lengths in the same
    arrays, eager work in between; each replay gives the eager call's bits.
    Two graphs with scratch of their own do not disturb each other."""
    lib = tg.lib()
    say(f"graph half={half}")
    dev = Dev(tg)
    bs = [Batch(20, 32, 4, 128, [5], [2500], half), Batch(21, 8, 2, 64, [1, 3], [40, 900], half, prefix=600)]
    eager = []
    for b in bs:
        out, _ = b.call(dev)
        lib.tg_hip_synchronize()
        eager.append(dev.read(out, b.q))
    graphs = [Graph(lambda s, b=b: b.queue(lib, s)) for b in bs]
    for step in range(3):
        for b, g, e in zip(bs, graphs, eager):
            g.replay()
            got = dev.read(b.ptrs["out"], b.q)
            assert got.tobytes() == e.tobytes(), step
            q2 = np.ascontiguousarray(b.q * np.float32(0.5))
            lib.tg_hip_memcpy_h2d(b.ptrs["q"], q2.ctypes.data, q2.nbytes)
            g.replay()
            got = dev.read(b.ptrs["out"], b.q)
            b.queue(lib)
            lib.tg_hip_synchronize()
            assert got.tobytes() == dev.read(b.ptrs["out"], b.q).tobytes()
            lib.tg_hip_memcpy_h2d(b.ptrs["q"], np.ascontiguousarray(b.q).ctypes.data, b.q.nbytes)
    # shorter caches through the graph that was captured with longer ones
    b, g = bs[0], graphs[0]
    b.past, b.kv_len = [7], np.array([7], np.int32)
    lib.tg_hip_memcpy_h2d(b.ptrs["len"], b.kv_len.ctypes.data, 4)
    b.k[b.slots[0], :, 12:], b.v[b.slots[0], :, 12:] = np.nan, np.nan
    for key in "kv":
        a = np.ascontiguousarray(getattr(b, key))
        lib.tg_hip_memcpy_h2d(b.ptrs[key], a.ctypes.data, a.nbytes)
    g.replay()
    b.check(dev.read(b.ptrs["out"], b.q), np.full_like(b.q, 7.5))
    for g in graphs:
        g.free()
    dev.free()


@pytest.mark.parametrize("half", [False, True])
def test_same_bits_every_time(tg, half):
    say(f"same bits half={half}")
    for b in (Batch(30, 32, 4, 128, [9], [3000], half), Batch(31, 64, 8, 64, [100, 1], [0, 800], half, sinks=True),
              Batch(32, 8, 2, 128, [1] * 6, list(range(6)), half, prefix=900)):
        dev = Dev(tg)
        out, _ = b.call(dev)
        tg.lib().tg_hip_synchronize()
        first = dev.read(out, b.q)
        for _ in range(3):
            b.queue(tg.lib())
            tg.lib().tg_hip_synchronize()
            assert dev.read(out, b.q).tobytes() == first.tobytes()
        dev.free()


@pytest.mark.parametrize("half", [False, True])
def test_spans_that_end_behind_a_multiple(tg, half):
    """Sequences that see one position more than a whole number of spans, of
    one KV head, so that the call has its most spans; the records are NaN
    before it."""
    for spans in ([58, 58] + [57] * 7, [33] * 16, [64, 2] * 8):
        say(f"spans {spans[:3]} half={half}")
        b = Batch(50, 1, 1, 64, [1] * len(spans), [128 * x for x in spans], half)
        dev = Dev(tg)
        need = tg.lib().tg_hip_attention_prompt_scratch_bytes(b.rows, b.n, 1, 1, 64, b.kv_max, 0)
        out, was = b.call(dev, scratch=dev(np.full(need // 4, np.nan, np.float32)))
        tg.lib().tg_hip_synchronize()
        got = dev.read(out, b.q)
        dev.free()
        b.check(got, was)


@pytest.mark.parametrize("half", [False, True])
def test_nan_queries(tg, half):
    """A NaN in q makes its own row and head NaN, whether or not its positions
    are split and with sinks too; the others stay."""
    for lens, past, prefix in (([3], [2000], 0), ([2, 1], [5, 0], 900), ([300], [0], 0)):
        say(f"nan in q half={half} past={past} prefix={prefix}")
        b = Batch(60, 8, 2, 64, lens, past, half, prefix=prefix, sinks=True)
        ref, tol = b.attend()
        b.q[1, 3 * 64 + 5] = np.nan
        got, _ = _run(tg, b)
        hit = np.zeros(got.shape, bool)
        hit[1, 3 * 64:4 * 64] = True
        assert np.all(np.isnan(got[hit]))
        assert np.all(np.abs(got - ref)[~hit] <= tol[~hit])


@pytest.mark.parametrize("half", [False, True])
def test_infinite_value_of_a_vanishing_weight(tg, half):
    """An infinity in V stays one, or becomes NaN where its weight underflows,
    however the positions are split."""
    say(f"infinite V of a vanishing weight half={half}")
    b = Batch(61, 8, 2, 64, [2], [3000], half, q_scale=300.0)
    b.v[b.slots[0], :, ::256, 7] = np.inf
    got, _ = _run(tg, b)
    assert not np.isfinite(got.reshape(2, 8, 64)[:, :, 7]).any()
    assert np.isfinite(got.reshape(2, 8, 64)[:, :, 8]).all()


def test_scratch_is_enough_for_every_call(tg):
    """What a call says it needs, with any window and cache type, is at most
    what the size function answers.  The calls have no rows on the device."""
    say("scratch sizes")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(5)
    p, cu, seen = dev(np.zeros(1 << 16, np.float32)), dev(np.zeros(1 << 14, np.int32)), 0
    for _ in range(4000):
        nkv = int(rng.choice([1, 2, 3, 4, 8, 16]))
        nh = nkv * int(rng.choice([1, 2, 4, 5, 8, 16]))
        hd = int(rng.choice([8, 64, 80, 128]))
        kv_max = int(2 ** rng.uniform(0, 18))
        n_rows = int(2 ** rng.uniform(0, 12))
        n_seqs = min(int(2 ** rng.uniform(0, 9)), 2 * n_rows)
        prefix = int(rng.choice([0, 0, 1])) * int(2 ** rng.uniform(0, 15))
        window = int(rng.choice([0, 1, 1])) * int(2 ** rng.uniform(0, 18))
        half = int(rng.integers(2))
        size = lib.tg_hip_attention_prompt_scratch_bytes(n_rows, n_seqs, nh, nkv, hd, kv_max, prefix)
        lib.tg_hip_clear_error()
        front = (p, nh * hd, half, p, p, 1, kv_max)
        back = (cu, cu, None, n_seqs, n_rows, window, None, nh, nkv, hd, p, nh * hd, None, None)
        if prefix:
            lib.tg_hip_attention_prefix_dev(*front, p, p, prefix, prefix, *back)
        else:
            lib.tg_hip_attention_prompt_dev(*front, *back)
        e = tg.last_error()
        need = int(e.split("needs ")[1].split()[0]) if e else 0
        assert need <= size, (need, size, n_rows, n_seqs, nh, nkv, hd, kv_max, prefix, window, half)
        seen += need > 0
    lib.tg_hip_synchronize()
    lib.tg_hip_clear_error()
    dev.free()
    assert seen > 1000


def test_calls_on_two_streams(tg):
    """Calls queued on two streams at once, each with scratch of its own, give
    the bits that they give alone."""
    from tests.test_gpu_decode import _hip_runtime
    say("two streams")
    lib, hip, dev = tg.lib(), _hip_runtime(), Dev(tg)
    bs = [Batch(70, 32, 4, 128, [9, 1], [3000, 40], False), Batch(71, 8, 2, 64, [1] * 5, [40] * 5, True, prefix=1500)]
    alone, streams = [], []
    for b in bs:
        out, _ = b.call(dev)
        lib.tg_hip_synchronize()
        alone.append(dev.read(out, b.q))
        streams.append(ctypes.c_void_p())
        assert hip.hipStreamCreate(ctypes.byref(streams[-1])) == 0
    for _ in range(20):
        for b, s in zip(bs, streams):
            b.queue(lib, s)
    for b, s, want in zip(bs, streams, alone):
        assert hip.hipStreamSynchronize(s) == 0
        assert dev.read(b.ptrs["out"], b.q).tobytes() == want.tobytes()
    for s in streams:
        hip.hipStreamDestroy(s)
    dev.free()


@pytest.mark.parametrize("half", [False, True])
def test_offsets_past_32_bits(tg, half):
    """Slots, rows of q and rows of the output whose byte offsets pass 2^32:
    the last slot of a cache of 2^20 positions, rows 2^21 floats apart."""
    say(f"offsets half={half}")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(9)
    nh, nkv, hd, kv_max, slots, stride, rows, past = 8, 4, 128, 1 << 20, 4, 1 << 21, 600, (1 << 20) - 700
    dtype = np.float16 if half else np.float32
    size = np.dtype(dtype).itemsize
    k = rng.standard_normal((nkv, 700, hd)).astype(dtype)
    v = rng.standard_normal((nkv, 700, hd)).astype(dtype)
    q = rng.standard_normal((rows, nh * hd)).astype(np.float32)
    pk, pv = (dev.room(slots * nkv * kv_max * hd * size) for _ in range(2))
    pq, po = (dev.room(rows * stride * 4) for _ in range(2))
    for h in range(nkv):
        at = (((slots - 1) * nkv + h) * kv_max + past) * hd * size
        lib.tg_hip_memcpy_h2d(pk + at, k[h].ctypes.data, k[h].nbytes)
        lib.tg_hip_memcpy_h2d(pv + at, v[h].ctypes.data, v[h].nbytes)
    for r in range(rows):
        lib.tg_hip_memcpy_h2d(pq + 4 * r * stride, q[r].ctypes.data, q[r].nbytes)
    cu, n, slot = (dev(np.array(x, np.int32)) for x in ([0, rows], [past + 50], [slots - 1]))
    scratch = dev.room(lib.tg_hip_attention_prompt_scratch_bytes(rows, 1, nh, nkv, hd, kv_max, 0))
    lib.tg_hip_clear_error()
    for window in (1, 40):   # the slot in front of the last 650 positions holds anything
        lib.tg_hip_attention_prompt_dev(pq, stride, int(half), pk, pv, slots, kv_max, cu, n, slot, 1, rows, window, None, nh, nkv,
                                        hd, po, stride, scratch, None)
        lib.tg_hip_synchronize()
        assert tg.last_error() == "", tg.last_error()
        for r in (0, 1, 300, 599):
            got = dev.read(po + 4 * r * stride, np.empty((nh, hd), np.float32))
            lo, hi = max(0, 50 + r + 1 - window), 50 + r + 1
            for h in range(nh):
                kk, vv = (x[h // 2, lo:hi].astype(np.float64) for x in (k, v))
                qq = q[r, h * hd:(h + 1) * hd].astype(np.float64)
                z = kk @ qq * hd ** -0.5
                p = np.exp(z - z.max())
                off = (8 * np.sqrt(2 * hd) + 4) * EPS * (np.abs(kk) @ np.abs(qq)).max() * hd ** -0.5 + (8 * np.sqrt(hi - lo) + 24) * EPS
                assert np.all(np.abs(got[h] - (p @ vv) / p.sum()) <= 2 * off * np.abs(vv).max()), (window, r, h)
    # and the append's: three rows at the end of the last slot, from rows 2^21 floats apart
    n2 = dev(np.array([kv_max - 3], np.int32))
    cu2 = dev(np.array([rows - 3, rows], np.int32))
    lib.tg_hip_kv_append_dev(None, pq, pq + 4 * nkv * hd, stride, stride, None, None, 1e-6, None, None, 0, cu2, n2, slot, 1, rows,
                             0, int(half), pk, pv, slots, kv_max, nh, nkv, hd, None, 0, None)
    lib.tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    for h in range(nkv):
        at = (((slots - 1) * nkv + h) * kv_max + kv_max - 3) * hd * size
        for ptr, first in ((pk, h * hd), (pv, (nkv + h) * hd)):
            assert np.array_equal(dev.read(ptr + at, np.empty((3, hd), dtype)), q[rows - 3:, first:first + hd].astype(dtype))
    dev.free()


# ---- append ----

def _rope_tables(n, hd):
    half = hd // 2
    ang = np.arange(n)[:, None] / (10000.0 ** (np.arange(half)[None, :] * 2.0 / hd))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _norm64(x, w, eps):
    x = x.astype(np.float64)
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


def _rope64(x, c, s):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    c, s = c.astype(np.float64), s.astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 4, 128), (64, 8, 64), (15, 3, 80), (6, 1, 8), (4, 4, 32), (14, 2, 112)])
@pytest.mark.parametrize("norm,rope,in_place,base", [(True, True, False, 0), (False, True, True, 37), (True, False, True, 0)])
def test_append_matches_plain(tg, nh, nkv, hd, half, norm, rope, in_place, base):
    """Tolerance: f32 results are a norm (a sum of hd squares, a root, a
    division, two products: hd / 2 + 6 roundings at most, of one sign only in
    the worst case) and a rotation (two products and a sum of values up to
    sqrt(2) of the head's largest); an f16 cache adds half a step of f16."""
    say(f"append {nh, nkv, hd} half={half} norm={norm} rope={rope} in_place={in_place}")
    lib, rng = tg.lib(), np.random.default_rng(nh + hd)
    lens, past, lead, tail = [3, 0, 1, 20], [0, 4, 9, 2], 1, 2
    rows, n, n_slots, kv_max = lead + sum(lens) + tail, 4, 6, 30
    width = (nh + 2 * nkv) * hd + 12
    qkv = rng.standard_normal((rows, width)).astype(np.float32)
    qn, kn = (rng.uniform(0.5, 1.5, hd).astype(np.float32) if norm else None for _ in range(2))
    cos, sin = _rope_tables(base + 22, hd) if rope else (None, None)
    cu = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
    slots = np.array([5, 0, 2, 1], np.int32)
    dtype = np.float16 if half else np.float32
    k0 = rng.standard_normal((n_slots, nkv, kv_max, hd)).astype(dtype)
    v0 = rng.standard_normal((n_slots, nkv, kv_max, hd)).astype(dtype)
    dev = Dev(tg)
    p, pk, pv = dev(qkv, 4), dev(k0), dev(v0)
    q_at, k_at, v_at = p, p + 4 * nh * hd, p + 4 * (nh + nkv) * hd
    q0 = qkv if in_place else np.full((rows, nh * hd + 4), 7.5, np.float32)
    po = p if in_place else dev(q0)
    lib.tg_hip_clear_error()
    lib.tg_hip_kv_append_dev(q_at, k_at, v_at, width, width, dev(qn), dev(kn), 1e-6, dev(cos), dev(sin), base + 22,
                             dev(cu), dev(np.array(past, np.int32)), dev(slots), n, rows, base, int(half), pk, pv, n_slots,
                             kv_max, nh, nkv, hd, po, q0.shape[1], None)
    lib.tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    got_q, got_k, got_v = dev.read(po, q0), dev.read(pk, k0), dev.read(pv, v0)
    dev.free()
    want_q, want_k, want_v = q0.astype(np.float64), k0.astype(np.float64), v0.astype(np.float64)
    for s in range(n):
        for i in range(lens[s]):
            r, at = cu[s] + i, past[s] + i
            heads = qkv[r, :(nh + 2 * nkv) * hd].reshape(-1, hd)
            q, k = _norm64(heads[:nh], qn, 1e-6), _norm64(heads[nh:nh + nkv], kn, 1e-6)
            if rope:
                q, k = (_rope64(x, cos[base + at], sin[base + at]) for x in (q, k))
            want_q[r, :nh * hd] = q.reshape(-1)
            want_k[slots[s], :, at], want_v[slots[s], :, at] = k, heads[nh + nkv:]
    step = (hd / 2 + 6 + 4) * EPS * 1.5
    cache = step + (2.0 ** -11 if half else 0)
    assert np.all(np.abs(got_q - want_q) <= step * np.abs(want_q).max())
    assert np.all(np.abs(got_k.astype(np.float64) - want_k) <= cache * np.maximum(np.abs(want_k), 0.1 * np.abs(want_k).max()) + step * np.abs(want_k).max())
    assert np.array_equal(got_v, want_v.astype(dtype))     # V is stored, rounded once
    stored = {(slots[s], past[s] + i) for s in range(n) for i in range(lens[s])}
    for a, b in ((got_k, k0), (got_v, v0)):
        for slot in range(n_slots):
            for at in range(kv_max):
                if (slot, at) not in stored:
                    assert np.array_equal(a[slot, :, at], b[slot, :, at]), (slot, at)
    live = np.zeros(rows, bool)
    live[lead:lead + sum(lens)] = True
    assert np.array_equal(got_q[~live], q0[~live]) and np.array_equal(got_q[:, nh * hd:], q0[:, nh * hd:])


def test_append_leaves_out_what_does_not_fit(tg):
    """Sequences with a bad slot or length, rows past the RoPE tables."""
    lib, rng = tg.lib(), np.random.default_rng(0)
    nh, nkv, hd, rows, kv_max = 4, 2, 64, 6, 10
    qkv = rng.standard_normal((rows, (nh + 2 * nkv) * hd)).astype(np.float32)
    cos, sin = _rope_tables(9, hd)
    k0 = np.full((2, nkv, kv_max, hd), 3.0, np.float32)
    for lens, slots, left in (([8, 0], [0, 1], [1, 2]), ([0, 0], [0, 7], [3, 4, 5]), ([0, -2], [1, 0], [3, 4, 5]),
                              ([0, 7], [0, 1], [5])):
        say(f"append left out: kv_len={lens} slots={slots}")
        dev = Dev(tg)
        p, pk, pv, q0 = dev(qkv), dev(k0), dev(k0), np.full((rows, nh * hd), 7.5, np.float32)
        po, w = dev(q0), qkv.shape[1]
        lib.tg_hip_kv_append_dev(p, p + 4 * nh * hd, p + 4 * (nh + nkv) * hd, w, w, None, None, 1e-6, dev(cos), dev(sin), 9,
                                 dev(np.array([0, 3, 6], np.int32)), dev(np.array(lens, np.int32)),
                                 dev(np.array(slots, np.int32)), 2, rows, 0, 0, pk, pv, 2, kv_max, nh, nkv, hd, po,
                                 nh * hd, None)
        lib.tg_hip_synchronize()
        got, gk = dev.read(po, q0), dev.read(pk, k0)
        dev.free()
        same = np.all(got == 7.5, axis=1)
        # kv_len 8 + 3 rows of 10 positions: the whole sequence is left out
        want = np.zeros(rows, bool)
        want[left if lens != [8, 0] else [0, 1, 2]] = True
        assert np.array_equal(same, want), (same, want)
        changed = int(np.any(gk != 3.0, axis=(1, 3)).sum())
        assert changed == rows - int(want.sum())


# ---- the calls together, as a program makes them ----

@pytest.mark.parametrize("half", [False, True])
def test_prompt_then_samples(tg, half):
    """A prompt appended and attended in two chunks, then as the shared prefix
    of five samples that append and attend one token each, twice; against the
    same rows computed in one piece in 64 bits from the rows that were cached."""
    say(f"prompt then samples half={half}")
    lib, rng = tg.lib(), np.random.default_rng(77)
    nh, nkv, hd, n_prompt, kv_max, n = 8, 2, 64, 150, 160, 5
    width, dtype = (nh + 2 * nkv) * hd, np.float16 if half else np.float32
    cos, sin = _rope_tables(200, hd)
    dev = Dev(tg)
    pc, ps = dev(cos), dev(sin)
    pre_k, pre_v = (dev(np.zeros((1, nkv, kv_max, hd), dtype)) for _ in range(2))
    own_k, own_v = (dev(np.zeros((n, nkv, 4, hd), dtype)) for _ in range(2))
    scratch = dev.room(max(lib.tg_hip_attention_prompt_scratch_bytes(100, n, nh, nkv, hd, kv_max, n_prompt), 1 << 20))
    scale = hd ** -0.5
    lib.tg_hip_clear_error()

    def attend(q, k, v, last):
        z = k @ q * scale
        p = np.exp(z[:last + 1] - z[:last + 1].max())
        return (p @ v[:last + 1]) / p.sum()

    def check(got, q, keys, vals, last):
        for h in range(nh):
            k, v = keys[h // 4].astype(np.float64), vals[h // 4].astype(np.float64)
            ref = attend(q[h].astype(np.float64), k, v, last)
            big = (np.abs(k[:last + 1]) @ np.abs(q[h])).max() * scale
            off = (8 * np.sqrt(2 * hd) + 4) * EPS * big + (8 * np.sqrt(last + 1) + 24) * EPS
            assert np.all(np.abs(got[h] - ref) <= 2 * off * np.abs(v).max())

    def step(rows, cu, kv_len, n_seqs, base, caches, slots_max, call):
        qkv = rng.standard_normal((rows, width)).astype(np.float32)
        p = dev(qkv)
        c, l = dev(np.array(cu, np.int32)), dev(np.array(kv_len, np.int32))
        out = dev(np.zeros((rows, nh * hd), np.float32))
        lib.tg_hip_kv_append_dev(p, p + 4 * nh * hd, p + 4 * (nh + nkv) * hd, width, width, None, None, 1e-6, pc, ps, 200,
                                 c, l, None, n_seqs, rows, base, int(half), *caches, n_seqs, slots_max, nh, nkv, hd, p,
                                 width, None)
        front = (p, width, int(half), *caches, n_seqs, slots_max)
        back = (c, l, None, n_seqs, rows, 0, None, nh, nkv, hd, out, nh * hd, scratch, None)
        if call == "prefix":
            lib.tg_hip_attention_prefix_dev(*front, pre_k, pre_v, n_prompt, kv_max, *back)
        else:
            lib.tg_hip_attention_prompt_dev(*front, *back)
        lib.tg_hip_synchronize()
        assert tg.last_error() == "", tg.last_error()
        q = dev.read(p, qkv)[:, :nh * hd].reshape(rows, nh, hd)
        return q, dev.read(out, np.empty((rows, nh, hd), np.float32))

    for first, count in ((0, 90), (90, 60)):
        q, got = step(count, [0, count], [first], 1, 0, (pre_k, pre_v), kv_max, "prompt")
        keys, vals = (dev.read(x, np.empty((nkv, kv_max, hd), dtype)) for x in (pre_k, pre_v))
        for i in range(0, count, 7):
            check(got[i], q[i], keys, vals, first + i)
    for t in range(2):
        q, got = step(n, range(n + 1), [t] * n, n, n_prompt, (own_k, own_v), 4, "prefix")
        ok, ov = (dev.read(x, np.empty((n, nkv, 4, hd), dtype)) for x in (own_k, own_v))
        for s in range(n):
            check(got[s], q[s], np.concatenate([keys[:, :n_prompt], ok[s]], 1), np.concatenate([vals[:, :n_prompt], ov[s]], 1),
                  n_prompt + t)
    dev.free()


def test_one_row_agrees_with_decode_attention(tg):
    """tg_hip_attention_dev's row (its own projections, norm and RoPE) and its
    cache, read back through the packed calls."""
    import oracle as O
    from tests.test_gpu_attention import _case, _gpu
    say("against tg_hip_attention_dev")
    c = _case(5, 512, 8, 2, 64, (O.FMT_Q4K, O.FMT_Q4K, O.FMT_Q4K, O.FMT_Q4K), 64, 40, norms=True, sinks=True, x_scale=0.3)
    _, att, kk, vv = _gpu(tg, c, 0)
    lib, dev = tg.lib(), Dev(tg)
    w, x = [dev(m) for m in c["w"]], dev(c["x"])
    scr = dev.room(lib.tg_hip_matmul_scratch_bytes(1, 512))
    qkv = dev.room(4 * 12 * 64)
    for i, (at, rows) in enumerate(((0, 512), (512, 128), (640, 128))):
        lib.tg_hip_matmul_dev(c["fmts"][i], w[i], None, x, qkv + 4 * at, rows, 512, 1, scr, None)
    pk, pv, cu, past = dev(c["kv_k"]), dev(c["kv_v"]), dev(np.array([0, 1], np.int32)), dev(np.array([40], np.int32))
    lib.tg_hip_kv_append_dev(qkv, qkv + 4 * 512, qkv + 4 * 640, 768, 768, dev(c["qn"]), dev(c["kn"]), ctypes.c_float(1e-6),
                             dev(c["rc"]), dev(c["rs"]), 64, cu, past, None, 1, 1, 0, 0, pk, pv, 1, 64, 8, 2, 64, qkv, 768,
                             None)
    out = dev.room(4 * 512)
    scratch = dev.room(lib.tg_hip_attention_prompt_scratch_bytes(1, 1, 8, 2, 64, 64, 0))
    lib.tg_hip_attention_prompt_dev(qkv, 768, 0, pk, pv, 1, 64, cu, past, None, 1, 1, 0, dev(c["sinks"]), 8, 2, 64, out, 512,
                                    scratch, None)
    lib.tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    got = dev.read(out, np.empty(512, np.float32))
    # the same f32 formulas in another order: tests/test_gpu_attention.py's bars
    assert np.abs(dev.read(pk, kk) - kk).max() <= 2e-5 * np.abs(kk).max()
    assert np.abs(dev.read(pv, vv) - vv).max() <= 2e-5 * np.abs(vv).max()
    assert np.abs(got - att).max() <= 1e-4 * np.abs(att).max()
    dev.free()
