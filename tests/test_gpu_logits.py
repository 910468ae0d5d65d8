"""GPU checks of tg_hip_logits_adjust_dev.  Every step is one f32 operation
rounded to nearest, so numpy's float32 gives the same bits."""

import sys

import numpy as np
import pytest

from tests._packed import Dev, Graph

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _plain(logits, hist=None, lens=None, start=None, pen=None, btok=None, bval=None, blen=None, allow=None):
    k, v = logits.shape
    out = logits.copy()
    with np.errstate(all="ignore"):
        for j in range(k):
            l = out[j]
            if hist is not None:
                h = hist[j, :min(max(lens[j], 0), hist.shape[1])]
                g = 0 if start is None else max(start[j], 0)
                ok = lambda t: t[(t >= 0) & (t < v)]   # noqa: E731
                rep, freq, pres = pen[j]
                t = np.unique(ok(h))
                l[t] = np.where(l[t] > 0, l[t] / rep, l[t] * rep)
                t, c = np.unique(ok(h[g:]), return_counts=True)
                l[t] = (l[t] - freq * c.astype(np.float32)) - pres
            if btok is not None:
                n = btok.shape[1] if blen is None else min(max(blen[j], 0), btok.shape[1])
                last = {int(t): b for t, b in zip(btok[j, :n], bval[j, :n]) if 0 <= t < v}
                for t, b in last.items():
                    l[t] = l[t] + b
            if allow is not None:
                a = allow[j if len(allow) > 1 else 0]
                bits = np.unpackbits(a.view(np.uint8), bitorder="little")[:v]
                l[bits == 0] = -np.inf
    top = np.array([np.nan if np.isnan(r).any() else r.max() for r in out], np.float32)
    arg = np.array([int(np.isnan(r).argmax()) if np.isnan(r).any() else int(r.argmax()) for r in out], np.int32)
    arg[top == -np.inf] = -1
    return out, arg, top


def _run(tg, logits, hist=None, lens=None, start=None, pen=None, btok=None, bval=None, blen=None, allow=None, in_place=False,
         want_out=True, want_arg=True, offset=0, queue=None):
    lib, dev = tg.lib(), Dev(tg)
    k, v = logits.shape
    pl = dev(logits, offset)
    po = pl if in_place else dev(np.full_like(logits, 7.5), offset) if want_out else None
    pa = dev(np.full(k, -77, np.int32)) if want_arg else None
    pm = dev(np.full(k, 7.5, np.float32)) if want_arg else None
    scr = dev.room(lib.tg_hip_logits_scratch_bytes(k, v))
    stride = 0 if allow is None or len(allow) == 1 else allow.shape[1]
    args = (pl, po, k, v, dev(hist), 0 if hist is None else hist.shape[1], dev(lens), dev(start), dev(pen), dev(btok),
            dev(bval), 0 if btok is None else btok.shape[1], dev(blen), dev(allow), stride, pa, pm, scr)
    lib.tg_hip_clear_error()
    if queue:
        queue(lib, args)
    else:
        lib.tg_hip_logits_adjust_dev(*args, None)
    lib.tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    r = (None if po is None else dev.read(po, logits), None if pa is None else dev.read(pa, np.empty(k, np.int32)),
         None if pm is None else dev.read(pm, np.empty(k, np.float32)))
    dev.free()
    return r


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def _inputs(seed, k, v, hist=0, bias=0, mask=False, wild=True):
    rng = np.random.default_rng(seed)
    kw = {}
    logits = (rng.standard_normal((k, v)) * 4).astype(np.float32)
    if hist:
        kw["hist"] = (rng.integers(0, v, (k, hist)) // rng.integers(1, 9, (k, hist))).astype(np.int32)
        kw["hist"][:, hist // 3::5] = kw["hist"][:, :1]     # one token again and again
        if wild:
            kw["hist"][:, ::7] = rng.choice([-1, v, 2 ** 31 - 1, -2 ** 31], kw["hist"][:, ::7].shape)
        kw["lens"] = rng.integers(0, hist + 1, k).astype(np.int32)
        kw["lens"][0] = hist
        kw["start"] = (kw["lens"] * rng.random(k)).astype(np.int32)
        kw["pen"] = np.stack([rng.uniform(0.8, 1.5, k), rng.uniform(-0.5, 1, k), rng.uniform(-0.5, 1, k)], 1).astype(np.float32)
    if bias:
        kw["btok"] = rng.integers(0, v, (k, bias)).astype(np.int32)
        kw["btok"][:, bias // 2:] = kw["btok"][:, :bias - bias // 2][:, ::-1]
        if wild:
            kw["btok"][:, ::6] = rng.choice([-1, v, v + 1, 2 ** 31 - 1], kw["btok"][:, ::6].shape)
        kw["bval"] = (rng.standard_normal((k, bias)) * 5).astype(np.float32)
        kw["blen"] = rng.integers(0, bias + 1, k).astype(np.int32)
        kw["blen"][-1] = bias
    if mask:
        w = (v + 31) // 32
        kw["allow"] = (rng.integers(0, 2 ** 32, (k, w), dtype=np.uint64) & rng.integers(0, 2 ** 32, (k, w), dtype=np.uint64)).astype(np.uint32)
        kw["allow"][:, -1] |= np.uint32(0xFFFFFFFF << (v % 32) & 0xFFFFFFFF) if v % 32 else np.uint32(0)   # bits past the vocabulary
    return logits, kw


@pytest.mark.parametrize("k,v,hist,bias,mask", [
    (1, 1, 1, 1, True), (1, 5, 3, 0, False), (2, 31, 40, 9, True), (3, 33, 0, 5, False), (1, 2047, 100, 0, True),
    (2, 2048, 500, 30, False), (3, 2049, 0, 0, True), (5, 10007, 3000, 700, True), (1, 151936, 700, 0, False),
    (9, 151936, 5000, 300, True), (64, 4099, 64, 8, True), (300, 100, 20, 3, True)])
def test_matches_plain(tg, k, v, hist, bias, mask):
    say(f"logits k={k} v={v} hist={hist} bias={bias} mask={mask}")
    logits, kw = _inputs(k * v + hist, k, v, hist, bias, mask)
    want = _plain(logits, **kw)
    for how in (dict(), dict(in_place=True), dict(offset=4), dict(want_arg=False), dict(want_out=False)):
        got = _run(tg, logits, **kw, **how)
        for g, w in zip(got, want):
            assert g is None or _same(g, w), how


def test_nothing_to_do_copies(tg):
    say("logits without adjustments")
    logits, _ = _inputs(1, 3, 5003)
    out, arg, top = _run(tg, logits)
    assert np.array_equal(out, logits) and np.array_equal(arg, logits.argmax(1)) and np.array_equal(top, logits.max(1))


def test_ties_masks_and_specials(tg):
    """Ties go to the lowest index across slices and lanes, a masked token is
    -inf whatever it was, a row with nothing left is -1, a NaN wins."""
    say("logits ties, masks, specials")
    v = 9000
    logits = np.zeros((8, v), np.float32)
    logits[0, [8999, 4096, 2047, 2048]] = 3                  # a tie over slices
    logits[1] = -np.inf                                      # nothing above -inf
    logits[2, 100] = np.nan                                  # masked away
    logits[3, [5000, 20]] = np.nan                           # seen: the first
    logits[4] = -np.inf
    logits[4, 8999] = np.finfo(np.float32).min               # the type's lowest value counts
    logits[5, :] = -0.0
    logits[5, 77] = 0.0                                      # equal to -0: the first of all
    logits[6, 10] = np.inf
    w = (v + 31) // 32
    allow = np.full((8, w), 0xFFFFFFFF, np.uint32)
    allow[2, 3] &= np.uint32(0xFFFFFFFF ^ (1 << (100 - 96)))
    allow[7] = 0
    want = _plain(logits, allow=allow)
    assert want[1].tolist() == [2047, -1, 0, 20, 8999, 0, 10, -1]
    got = _run(tg, logits, allow=allow)
    assert all(_same(g, x) for g, x in zip(got, want))
    one = allow[2:3]                                         # one mask for all rows
    got = _run(tg, logits, allow=one)
    assert all(_same(g, x) for g, x in zip(got, _plain(logits, allow=one)))


def test_lengths_out_of_range(tg):
    say("logits lengths out of range")
    logits, kw = _inputs(5, 4, 3001, 50, 20)
    kw["lens"] = np.array([-3, 0, 51, 2 ** 31 - 1], np.int32)
    kw["start"] = np.array([0, 5, -9, 2 ** 31 - 1], np.int32)
    kw["blen"] = np.array([-1, 0, 21, 2 ** 31 - 1], np.int32)
    got = _run(tg, logits, **kw)
    assert all(_same(g, x) for g, x in zip(got, _plain(logits, **kw)))
    kw["start"] = kw["blen"] = None
    got = _run(tg, logits, **kw)
    assert all(_same(g, x) for g, x in zip(got, _plain(logits, **kw)))


def test_replayed_graph(tg):
    say("logits graph")
    logits, kw = _inputs(6, 3, 20011, 300, 10, True)

    def queue(lib, args):
        g = Graph(lambda s: lib.tg_hip_logits_adjust_dev(*args, s))
        for _ in range(3):
            g.replay()
            lib.tg_hip_logits_adjust_dev(*args, None)
            lib.tg_hip_synchronize()
        g.replay()
        g.free()

    got = _run(tg, logits, queue=queue, **kw)
    assert all(_same(g, x) for g, x in zip(got, _plain(logits, **kw)))


def test_behind_the_head(tg):
    """The head's logits, adjusted in place, give the token that numpy picks
    from the same logits; without adjustments the head's own argmax."""
    import tinygiant_amd.synth as S
    say("head, then logits")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(8)
    k, v, cols = 5, 4999, 2048
    nbytes = v * lib.tg_row_bytes(tg.FMT_Q6K, cols)
    w = dev.room(nbytes)
    lib.tg_hip_synth_fill(2, S.tensor_seed(8, 0, 0, 3), w, nbytes, None)
    x = dev(rng.standard_normal((k, cols)).astype(np.float32))
    lg, am, mv = dev.room(4 * k * v), dev.room(4 * k), dev.room(4 * k)
    sc, sc2 = dev.room(lib.tg_hip_head_scratch_bytes(k, v, cols)), dev.room(lib.tg_hip_logits_scratch_bytes(k, v))
    lib.tg_hip_clear_error()
    lib.tg_hip_head_argmax_dev(tg.FMT_Q6K, w, x, None, 1e-6, k, v, cols, lg, am, mv, sc, None)
    lib.tg_hip_synchronize()
    logits, first = dev.read(lg, np.empty((k, v), np.float32)), dev.read(am, np.empty(k, np.int32))
    none = (None, 0, None, None, None, None, None, 0, None, None, 0)
    lib.tg_hip_logits_adjust_dev(lg, None, k, v, *none, am, mv, sc2, None)
    lib.tg_hip_synchronize()
    assert np.array_equal(dev.read(am, first), first)
    assert np.array_equal(dev.read(mv, np.empty(k, np.float32)), logits.max(1))
    hist = np.tile(first[:, None], (1, 3)).astype(np.int32)     # each row's favourite three times
    kw = dict(hist=hist, lens=np.full(k, 3, np.int32), pen=np.tile(np.array([[1.3, 50.0, 20.0]], np.float32), (k, 1)))
    lib.tg_hip_logits_adjust_dev(lg, lg, k, v, dev(hist), 3, dev(kw["lens"]), None, dev(kw["pen"]), None, None, 0, None, None,
                                 0, am, mv, sc2, None)
    lib.tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    want = _plain(logits, **kw)
    assert np.array_equal(dev.read(lg, logits), want[0]) and np.array_equal(dev.read(am, first), want[1])
    assert not np.any(want[1] == first)
    dev.free()
