"""GPU checks of rotary positions and of 8-bit caches in pages
(tg_hip_rope_tables_dev, tg_hip_rope_dev, tg_hip_paged_append_dev,
tg_hip_paged_read_dev, tg_hip_attention_paged_dev) against plain
computations in 64 bits; attention's tolerance: tests/_paged.py."""

import ctypes
import math

import numpy as np
import pytest

from tests._packed import EPS, Dev, Graph
from tests._paged import LEAST, MOST, Pages, attend, tables, turn

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def done(tg):
    tg.lib().tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()


# ------------------------------------------------------------------ tables

def _frequencies(rot, theta, scaling, factor, orig, low, high):
    f = []
    for i in range(rot // 2):
        x = theta ** (-2 * i / rot)
        if scaling == 1:
            x /= factor
        elif scaling == 2:
            x = (theta * factor ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif scaling in (3, 4):
            a, b = (rot * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (low, high))
            if scaling == 4:
                a, b = math.floor(a), math.ceil(b)
            a, b = max(a, 0.0), min(b, rot - 1.0)
            w = min(1.0, max(0.0, (i - a) / max(b - a, 1e-3)))
            x = x / factor * w + x * (1 - w)
        elif scaling == 5:
            w = min(1.0, max(0.0, (orig * x / (2 * math.pi) - low) / (high - low)))
            x = x * w + x / factor * (1 - w)
        f.append(x)
    return np.array(f)


@pytest.mark.parametrize("scaling", range(6))
@pytest.mark.parametrize("n,first,rot,theta,factor,m", [
    (1, 0, 8, 1e4, 1.0, 1.0), (77, 0, 128, 1e6, 4.0, 1.0), (300, 131000, 64, 150000.0, 32.0, 1.3465736), (5, 1 << 30, 256, 1e4, 8.0, 0.5),
    (1025, 999, 40, 5e5, 0.5, -1.0)])
def test_tables(tg, scaling, n, first, rot, theta, factor, m):
    """Off by half a step of the value, and by what 64 bits do to the angle: p f of at most A radians is off by a few 2^-53 A
    (the frequency's own roundings among them, eight steps are counted), and that much the cosine."""
    say(f"tables scaling={scaling} {n, first, rot, theta, factor}")
    lib, dev = tg.lib(), Dev(tg)
    low, high = (1.0, 4.0) if scaling == 5 else (32.0, 1.0)
    guard = np.full(n * rot // 2 + 8, 7.0, np.float32)
    cos, sin = dev(guard), dev(guard)
    lib.tg_hip_clear_error()
    lib.tg_hip_rope_tables_dev(cos, sin, n, first, rot, theta, scaling, factor, 4096, low, high, m, None)
    done(tg)
    angle = np.arange(first, first + n)[:, None] * _frequencies(rot, theta, scaling, np.float64(np.float32(factor)), 4096, low, high)
    for ptr, want in ((cos, np.cos(angle)), (sin, np.sin(angle))):
        got = dev.read(ptr, guard)
        assert np.all(got[-8:] == 7.0)
        want = want * np.float64(np.float32(m))
        tol = np.abs(want) * EPS + abs(m) * (8 * 2.0 ** -53 * (angle + 1)) + 1e-45
        assert np.all(np.abs(got[:-8].reshape(n, -1) - want) <= tol)
    dev.free()


# ------------------------------------------------------------------ rows

@pytest.mark.parametrize("inter", [0, 1])
@pytest.mark.parametrize("rows,nh,hd,rot,pad", [
    (1, 1, 8, 8, 0), (3, 5, 16, 8, 1), (40, 36, 128, 128, 0), (9, 18, 80, 40, 3), (130, 2, 1024, 64, 0), (2, 1024, 24, 16, 8), (700, 3, 64, 56, 0)])
def test_rope(tg, inter, rows, nh, hd, rot, pad):
    """Two products and a sum, each rounded once: off by (sqrt 2 + 1) EPS of the pair's length. Rows whose position is in no table stay."""
    say(f"rope {rows, nh, hd, rot} inter={inter}")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(rows + hd)
    stride, n = nh * hd + pad, 50
    x = rng.standard_normal((rows, stride)).astype(np.float32)
    pos = rng.integers(0, n, rows).astype(np.int32)
    pos[::7] = rng.choice([-1, n, 2 ** 31 - 1, -2 ** 31], len(pos[::7])) if rows > 2 else pos[::7]
    cos, sin = tables(n, rot)
    live = (pos >= 0) & (pos < n)
    at = np.where(live, pos, 0)
    v = x[:, :nh * hd].reshape(rows, nh, hd).astype(np.float64)
    c, s = cos[at][:, None].astype(np.float64), sin[at][:, None].astype(np.float64)
    want = turn(v, c, s, rot, inter)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    tol = np.zeros_like(v)
    tol[..., a] = tol[..., b] = 2.5 * EPS * np.hypot(v[..., a], v[..., b])
    args = (dev(pos), dev(cos), dev(sin), n, rot, inter, rows, nh, hd)
    for place in (False, True):
        src = dev(x)
        was = x if place else np.full((rows, stride + 5), 7.0, np.float32)
        dst = src if place else dev(was)
        lib.tg_hip_clear_error()
        lib.tg_hip_rope_dev(src, stride, *args, dst, was.shape[1], None)
        done(tg)
        got = dev.read(dst, was)
        assert np.array_equal(got[~live], was[~live]) and np.array_equal(got[:, nh * hd:], was[:, nh * hd:])
        err = np.abs(got[:, :nh * hd].reshape(rows, nh, hd) - want)[live]
        assert np.all(err <= tol[live]), float(err.max())
    dev.free()


# ------------------------------------------------------------------ append

class Append:
    """A call of tg_hip_paged_append_dev and what it leaves."""

    def __init__(self, seed, nh, nkv, hd, lens, past, size=16, rot=None, inter=0, norm=False, pad=0, lead=0, tail=0, rope_len=None):
        rng = self.rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.hd, self.lens, self.past, self.inter, self.pad = nh, nkv, hd, list(lens), list(past), inter, pad
        self.n, self.rows, self.lead = len(lens), lead + sum(lens) + tail, lead
        self.pages = Pages(rng, self.n, nkv, hd, size, max([1] + [a + b for a, b in zip(lens, past)]))
        for s in range(self.n):
            self.pages.fill(rng, s, past[s])
        self.cu = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
        self.kv_len = np.array(past, np.int32)
        self.x = (rng.standard_normal((self.rows, (nh + 2 * nkv) * hd + pad)) * np.exp2(rng.integers(-3, 4, (self.rows, 1)))).astype(np.float32)
        self.norms = [rng.uniform(0.5, 1.5, hd).astype(np.float32) if norm else None for _ in range(2)]
        self.rot = hd if rot is None else rot
        self.rope_len = rope_len or max([1] + [a + b for a, b in zip(lens, past)])
        self.cos, self.sin = tables(self.rope_len, self.rot) if self.rot else (None, None)

    def want(self):
        """(q in 64 bits with NaN where nothing is written, the pages behind the call)"""
        q, pages = np.full((self.rows, self.nh * self.hd), np.nan), self.pages.copy()
        x = self.x[:, :self.x.shape[1] - self.pad].astype(np.float64).reshape(self.rows, -1, self.hd)
        for s, (n, p) in enumerate(zip(self.lens, self.past)):
            y = x[self.cu[s]:self.cu[s] + n].copy()
            for part, w in ((slice(0, self.nh), self.norms[0]), (slice(self.nh, self.nh + self.nkv), self.norms[1])):
                if w is not None:
                    y[:, part] *= w / np.sqrt((y[:, part] ** 2).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))
            live = np.ones(n, bool)
            if self.rot:
                at = np.arange(p, p + n)
                live = at < self.rope_len
                at = np.minimum(at, self.rope_len - 1)
                y[:, :self.nh + self.nkv] = turn(y[:, :self.nh + self.nkv], self.cos[at][:, None].astype(np.float64),
                                                 self.sin[at][:, None].astype(np.float64), self.rot, self.inter)
            q[self.cu[s]:self.cu[s] + n][live] = y[live, :self.nh].reshape(-1, self.nh * self.hd)
            for which, part in (("k", slice(self.nh, self.nh + self.nkv)), ("v", slice(self.nh + self.nkv, None))):
                pages.store(which, s, p, y[:, part], live)
        return q, pages

    def call(self, dev, stream=None, place=False, q=True):
        p, w = self.pages, self.x.shape[1]
        x = dev(self.x)
        self.ptr = [dev(t) for t in p.arrays()]
        out = (x if place else dev(np.full((self.rows, w), 7.0, np.float32))) if q else None
        qd, kd = 4 * self.nh * self.hd, 4 * self.nkv * self.hd
        self.args = (x if q else None, x + qd, x + qd + kd, w, w, dev(self.norms[0]), dev(self.norms[1]), 1e-6, dev(self.cos), dev(self.sin),
                     self.rope_len, self.rot, self.inter, dev(self.cu), dev(self.kv_len), self.n, self.rows, *self.ptr, p.n_pages,
                     p.size, dev(p.table), p.table.shape[1], self.nh, self.nkv, self.hd, out, w)
        self.out, self.x_ptr = out, x
        self.queue(dev.tg.lib(), stream)

    def queue(self, lib, stream=None):
        lib.tg_hip_paged_append_dev(*self.args, stream)

    def check(self, tg, dev, want=None, place=False):
        q, pages = want or self.want()
        done(tg)
        for got, ptr, name in zip(pages.arrays(), self.ptr, ("pages_k", "pages_v", "exps_k", "exps_v")):
            now = dev.read(ptr, got)
            if name.startswith("exps"):
                assert np.array_equal(now, got), name
                continue
            exps = pages.ek if name == "pages_k" else pages.ev
            same = (now == got) | (np.repeat(exps, 16, 2) == 255)[..., None]   # what a block that is NaN holds means nothing
            assert same.all(), (name, int((~same).sum()))
        if self.out:
            got, qd = dev.read(self.out, self.x), self.nh * self.hd
            was = self.x if place else np.full_like(self.x, 7.0)
            live = ~np.isnan(q[:, 0])
            assert np.array_equal(got[~live], was[~live]) and np.array_equal(got[:, qd:], was[:, qd:])
            # hd products and sums, a root, a division, and the rotation's three steps on values of at most twice the head's largest
            big = np.abs(q[live]).reshape(-1, self.nh, self.hd).max(-1).repeat(self.hd, 1)
            assert np.all(np.abs(got[live, :qd] - q[live]) <= (np.sqrt(self.hd) + 16) * EPS * 2 * big)


LAYOUTS = [(8, 2, 128), (32, 4, 128), (8, 1, 64), (4, 4, 32), (15, 3, 80), (6, 1, 16), (14, 2, 112), (40, 1, 48)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("lens,past,size", [
    ([1], [0], 16), ([1], [15], 16), ([1], [16], 32), ([16], [0], 16), ([17, 0, 1], [15, 3, 31], 64), ([33, 5], [7, 129], 128),
    ([1] * 9, [0, 1, 15, 16, 17, 63, 64, 65, 300], 16), ([130], [1000], 1024)])
def test_append(tg, layout, lens, past, size):
    nh, nkv, hd = layout
    say(f"append {layout} lens={lens} past={past} size={size}")
    for i, kw in enumerate((dict(), dict(rot=hd // 16 * 8, inter=1, norm=True, pad=3, lead=2, tail=1), dict(rot=8, norm=hd == 80), dict(rot=0))):
        a, dev = Append(hd + nh + i, nh, nkv, hd, lens, past, size, **kw), Dev(tg)
        tg.lib().tg_hip_clear_error()
        a.call(dev, place=i == 2)
        a.check(tg, dev, place=i == 2)
        dev.free()


def test_append_again_changes_nothing(tg):
    say("append twice")
    a, dev = Append(1, 8, 2, 64, [5, 40], [9, 30]), Dev(tg)
    a.call(dev)
    want = a.want()
    a.check(tg, dev, want)
    a.queue(tg.lib())
    a.check(tg, dev, want)
    dev.free()


def test_append_only_keys_and_values(tg):
    say("append without q")
    a, dev = Append(2, 8, 2, 128, [20], [5], norm=True), Dev(tg)
    a.call(dev, q=False)
    a.check(tg, dev)
    dev.free()


def test_append_many_sequences(tg):
    for n in (64, 65, 700):
        say(f"append {n} sequences")
        a, dev = Append(n, 4, 2, 32, [i % 3 for i in range(n)], [(7 * i) % 50 for i in range(n)], lead=3), Dev(tg)
        a.call(dev)
        a.check(tg, dev)
        dev.free()


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e10, 127 * 2.0 ** 42, 1e20])
def test_append_ranges(tg, size):
    """Values at and past both ends of the exponents' range, zeros, and halves between two bytes."""
    say(f"append ranges {size}")
    a, dev = Append(3, 4, 2, 64, [35], [20], rot=0), Dev(tg)
    kv = a.x[:, 4 * 64:]
    kv *= np.float32(size)
    kv[:, 64:128] = 0
    kv[:16, :64] = np.float32(size) * (np.arange(64) - 31.5).astype(np.float32)[None]
    a.call(dev)
    a.check(tg, dev)
    dev.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_not_finite(tg, bad):
    """The blocks that take such a value in are NaN, also for what is stored later, until a sequence begins them anew."""
    say(f"append {bad}")
    a, dev = Append(4, 4, 2, 64, [40], [3], rot=16), Dev(tg)
    a.x[9, 4 * 64 + 5] = bad       # K of head 0 at position 12
    a.x[30, (4 + 2 + 1) * 64] = bad   # V of head 1 at position 33
    a.call(dev)
    want = a.want()
    assert (want[1].ek == 255).sum() == 1 and (want[1].ev == 255).sum() == 1
    a.check(tg, dev, want)
    b = Append(5, 4, 2, 64, [4], [10], rot=16)
    b.pages = want[1].copy()
    b.call(dev)
    want = b.want()
    assert (want[1].ek == 255).sum() == 1
    b.check(tg, dev, want)
    c = Append(6, 4, 2, 64, [20], [0], rot=16)
    c.pages = want[1].copy()
    c.call(dev)
    want = c.want()
    assert (want[1].ek == 255).sum() == 0
    c.check(tg, dev, want)
    dev.free()


def test_append_left_out(tg):
    """Rows past the tables, sequences that do not fit, pages that are none: everything of theirs stays."""
    say("append left out")
    a, dev = Append(7, 4, 2, 64, [30, 3], [5, 40], rope_len=20), Dev(tg)
    a.call(dev)
    a.check(tg, dev)
    dev.free()
    for past in (-1, 10 ** 6, 2 ** 31 - 1):
        a, dev = Append(8, 4, 2, 64, [3, 4, 2], [50, 20, 0]), Dev(tg)
        a.kv_len[1] = past
        a.lens = [3, 0, 2]   # as without sequence 1's rows
        want = a.want()
        a.call(dev)
        a.check(tg, dev, want)
        dev.free()
    for page in (-1, 10 ** 6, -2 ** 31):
        a, dev = Append(9, 4, 2, 64, [50], [5]), Dev(tg)
        a.pages.table[0, 2] = page
        a.call(dev)
        a.check(tg, dev)
        dev.free()
    for cu in ([0, 5, 4000], [-7, 3, 6], [4, 2, 1]):   # not specified, but the call ends and stays in bounds
        a, dev = Append(10, 4, 2, 64, [3, 4], [50, 60]), Dev(tg)
        a.cu = np.array(cu, np.int32)
        a.call(dev)
        done(tg)
        dev.free()


def test_a_value_is_off_by_one_step_at_most(tg):
    """Rows of rising magnitude, one a call, each of which may double the unit of those before it."""
    say("append one by one")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(11)
    a = Append(11, 2, 1, 32, [16], [0], rot=0)
    x = (rng.uniform(-1, 1, (16, 4 * 32)) * 1.31 ** np.arange(16)[:, None]).astype(np.float32)
    a.x = x.copy()
    a.call(dev)
    args = list(a.args)
    for i in range(16):
        args[13], args[14], args[16] = dev(np.array([0, 1], np.int32)), dev(np.array([i], np.int32)), 1
        args[1], args[2] = (a.x_ptr + 4 * (i * 128 + o) for o in (64, 96))
        args[0], args[-2] = None, None
        lib.tg_hip_paged_append_dev(*args, None)
    done(tg)
    for name, at, ptr, e in (("k", 64, 0, 2), ("v", 96, 1, 3)):
        bytes_, exps = dev.read(a.ptr[ptr], a.pages.k), dev.read(a.ptr[e], a.pages.ek)
        page = a.pages.table[0, 0]
        unit = 2.0 ** (int(exps[page, 0, 0]) - 127)
        assert unit == 2.0 ** math.ceil(math.log2(np.abs(x[:, at:at + 32].astype(np.float64)).max() / 127))
        err = np.abs(bytes_[page, 0] * unit - x[:, at:at + 32])
        assert err.max() <= unit and err[-1].max() <= unit / 2
    dev.free()


# ------------------------------------------------------------------ read

@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("nkv,hd,lens,size", [(1, 16, [1], 16), (3, 80, [0, 17, 16, 300], 32), (4, 128, [1000, 5], 1024), (8, 64, [33] * 70, 16)])
def test_read(tg, half, nkv, hd, lens, size):
    say(f"read {nkv, hd} half={half}")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(hd)
    n, kv_max = len(lens), max(lens) + 3
    p = Pages(rng, n, nkv, hd, size, max(lens))
    for s in range(n):
        p.fill(rng, s, lens[s], spread=3)
    if n > 2:
        p.ek[p.table[1, 0], 0, 0], p.ev[p.table[1, 0], 1, 0] = 255, 84
        p.table[3, 1] = -5
    slots = rng.permutation(n + 1)[:n].astype(np.int32)
    dtype = np.float16 if half else np.float32
    was = np.full((n + 1, nkv, kv_max, hd), 7.0, dtype)
    k, v = dev(was), dev(was)
    tail = (p.n_pages, size, dev(p.table), p.table.shape[1], dev(np.array(lens, np.int32)), n, nkv, hd, half, k, v, dev(slots), n + 1, kv_max)
    lib.tg_hip_clear_error()
    lib.tg_hip_paged_read_dev(*(dev(t) for t in p.arrays()), *tail, None)
    done(tg)
    for which, ptr in (("k", k), ("v", v)):
        got, want = dev.read(ptr, was), was.copy()
        for s in range(n):
            want[slots[s], :, :lens[s]] = p.values(which, s, lens[s]).astype(dtype)   # exact in f32, nearest in f16
        assert np.array_equal(got, want, equal_nan=True)
    # a slot that is none, a length that does not fit
    for key, vals in (("slot", (-1, n + 1)), ("len", (-1, kv_max + 1, 2 ** 31 - 1))):
        for bad in vals:
            l, sl = np.array(lens, np.int32), slots.copy()
            (l if key == "len" else sl)[0] = bad
            k = dev(was)
            args = list(tail)
            args[4], args[9], args[10], args[11] = dev(l), k, k, dev(sl)
            args[10] = dev(was)
            lib.tg_hip_paged_read_dev(*(dev(t) for t in p.arrays()), *args, None)
            done(tg)
            got = dev.read(k, was)
            assert np.all(got[slots[0]] == 7.0)
    dev.free()


# ------------------------------------------------------------------ attention

class Attend:
    def __init__(self, seed, nh, nkv, hd, lens, past, size=16, window=0, sinks=False, lead=0, tail=0, pad=0, q_scale=2.0, spread=1, room=0):
        rng = self.rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.hd, self.lens, self.past, self.window = nh, nkv, hd, list(lens), list(past), window
        self.n, self.rows, self.pad = len(lens), lead + sum(lens) + tail, pad
        self.longest = max([1] + [a + b for a, b in zip(lens, past)])
        self.max_kv = self.longest + room
        self.pages = Pages(rng, self.n, nkv, hd, size, self.max_kv)
        for s in range(self.n):
            self.pages.fill(rng, s, lens[s] + past[s], spread)
        self.q = (rng.standard_normal((self.rows, nh * hd + pad)) * q_scale).astype(np.float32)
        self.sinks = rng.standard_normal(nh).astype(np.float32) if sinks else None
        self.cu = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
        self.kv_len = np.array(past, np.int32)

    def want(self):
        return attend(self.q[:, :self.nh * self.hd], self.pages, self.cu, self.lens, self.past, self.nh, self.window, self.sinks)

    def call(self, dev, stream=None, place=False):
        p, lib = self.pages, dev.tg.lib()
        q = dev(self.q)
        self.was = self.q if place else np.full_like(self.q, 7.0)
        self.out = q if place else dev(self.was)
        size = lib.tg_hip_attention_paged_scratch_bytes(self.rows, self.n, self.nh, self.nkv, self.hd, self.max_kv)
        self.guard = np.full(64, 0x5A, np.uint8)
        scratch = dev.room(size + 64)
        lib.tg_hip_memcpy_h2d(scratch + size, self.guard.ctypes.data, 64)
        self.after = scratch + size
        self.len_ptr, self.cu_ptr = dev(self.kv_len), dev(self.cu)
        self.args = (q, self.q.shape[1], *(dev(t) for t in p.arrays()), p.n_pages, p.size, dev(p.table), p.table.shape[1], self.cu_ptr,
                     self.len_ptr, self.n, self.rows, self.max_kv, self.window, dev(self.sinks), self.nh, self.nkv, self.hd, self.out,
                     self.q.shape[1], scratch)
        lib.tg_hip_clear_error()
        self.queue(lib, stream)

    def queue(self, lib, stream=None):
        lib.tg_hip_attention_paged_dev(*self.args, stream)

    def check(self, tg, dev, want=None):
        """The worst error, as a part of the tolerance."""
        ref, tol = want or self.want()
        done(tg)
        got, qd = dev.read(self.out, self.q), self.nh * self.hd
        assert np.array_equal(dev.read(self.after, self.guard), self.guard)
        assert np.array_equal(got[:, qd:], self.was[:, qd:])
        mine = np.zeros(self.rows, bool)
        for s in range(self.n):
            mine[self.cu[s]:self.cu[s] + self.lens[s]] = True
        assert np.array_equal(got[~mine], self.was[~mine])
        got, ref, tol = got[mine, :qd], ref[mine], tol[mine]
        assert np.array_equal(np.isnan(got), np.isnan(ref)), (int(np.isnan(got).sum()), int(np.isnan(ref).sum()))
        fine = ~np.isnan(ref)
        err = np.abs(got - ref)[fine]
        assert np.all(err <= tol[fine]), float((err / tol[fine]).max())
        return float((err / np.maximum(tol[fine], 1e-300)).max()) if err.size else 0.0


def _attend(tg, a, **kw):
    dev = Dev(tg)
    a.call(dev, **kw)
    worst = a.check(tg, dev)
    dev.free()
    return worst


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("lens,past,size", [
    ([1], [0], 16), ([1], [1], 32), ([5], [63], 16), ([0, 1, 3], [4, 0, 60], 64), ([33, 0, 64, 1], [0, 5, 1, 130], 16), ([130], [0], 128),
    ([17, 31], [100, 257], 256), ([1] * 9, [0, 1, 15, 16, 31, 32, 65, 127, 300], 16)])
def test_attention(tg, layout, lens, past, size):
    nh, nkv, hd = layout
    say(f"attention {layout} lens={lens} past={past} size={size}")
    a = Attend(nh + hd + sum(lens), nh, nkv, hd, lens, past, size, sinks=nh % 4 != 0, lead=len(lens) % 3, tail=2, pad=4 * (nkv % 2))
    say(f"  worst error / tolerance {_attend(tg, a):.3f}")


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 64, 128, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_windows(tg, window, hd):
    say(f"attention window={window} hd={hd}")
    _attend(tg, Attend(hd, 8, 1, hd, [1, 90, 200], [500, 0, 77], window=window, sinks=hd == 64))
    _attend(tg, Attend(hd + 1, 8, 2, hd, [1, 1, 3], [3000, 2500, 0], 64, window=window))


@pytest.mark.parametrize("nh,nkv,hd,lens,past,size", [
    (32, 4, 128, [9], [4000], 64), (64, 8, 64, [3], [9000], 16), (8, 1, 128, [1], [20011], 128), (8, 2, 128, [600], [700], 16),
    (8, 8, 64, [257, 300], [511, 0], 64), (16, 2, 128, [1] * 12, [37 * i * i % 2900 for i in range(12)], 32), (8, 2, 96, [150, 1, 9], [900, 4100, 37], 16),
    (15, 3, 80, [200], [3], 512)])
def test_attention_long(tg, nh, nkv, hd, lens, past, size):
    say(f"attention long {nh, nkv, hd} lens={lens} past={past[:3]}")
    say(f"  worst error / tolerance {_attend(tg, Attend(sum(lens), nh, nkv, hd, lens, past, size, sinks=hd == 64, spread=4)):.3f}")


@pytest.mark.parametrize("nh,nkv,hd", [(32, 4, 128), (16, 2, 64), (15, 3, 80), (8, 8, 96), (64, 1, 32)])
@pytest.mark.parametrize("lens,past,window", [
    ([1, 200, 9, 0, 1, 40], [900, 0, 2200, 5, 40, 600], 0), ([300, 1], [30, 3500], 0), ([1, 150, 1, 180], [4000, 2500, 0, 0], 0),
    ([17, 16, 130, 1], [1500, 700, 20, 3000], 600), ([1] * 20 + [260], [61 * i for i in range(20)] + [500], 0), ([400, 0, 129], [0, 0, 1400], 0)])
def test_attention_mixed(tg, nh, nkv, hd, lens, past, window):
    """Prompts, chunks, verify passes and single tokens in one call."""
    say(f"attention mixed {nh, nkv, hd} lens={lens} past={past} window={window}")
    a = Attend(sum(lens) + hd, nh, nkv, hd, lens, past, 32, window=window, sinks=nkv != 2, lead=2, tail=1, spread=3)
    say(f"  worst error / tolerance {_attend(tg, a):.3f}")


@pytest.mark.parametrize("nh,nkv,hd,lens,past,window,size", [
    (32, 4, 128, [4100], [20], 0, 64), (28, 2, 112, [4700], [0], 0, 16), (32, 4, 128, [4300], [700], 900, 128), (64, 8, 64, [2200], [33], 0, 32),
    (64, 8, 32, [2100], [0], 300, 1024), (32, 4, 128, [2100, 3, 2500], [100, 4000, 0], 0, 64), (16, 16, 80, [5000], [0], 0, 64)])
def test_attention_of_long_prompts(tg, nh, nkv, hd, lens, past, window, size):
    """Rows all over a call of many, two heads each; all rows are finite and some see a block that is NaN."""
    say(f"attention of long prompts {nh, nkv, hd} lens={lens} past={past} window={window}")
    a, dev = Attend(sum(lens), nh, nkv, hd, lens, past, size, window=window, sinks=hd < 80, lead=1, tail=1, spread=3), Dev(tg)
    at = past[0] + lens[0] // 2
    a.pages.ev[a.pages.table[0, at // size], nkv - 1, at % size // 16] = 255
    rng = np.random.default_rng(1)
    rows = {1, 2, a.rows - 2, 1 + lens[0] // 2, 1 + lens[0] // 2 + 5} | {int(r) for r in rng.integers(1, a.rows - 1, 25)}
    only = {r: [int(h) for h in rng.choice(nh, 2, replace=False)] + [nh - 1] for r in rows}
    ref, tol = attend(a.q, a.pages, a.cu, lens, past, nh, window, a.sinks, only)
    a.call(dev)
    done(tg)
    got = dev.read(a.out, a.q)
    seen = 0
    for r, heads in only.items():
        s = next(i for i in range(a.n) if a.cu[i] <= r < a.cu[i + 1])
        last = past[s] + r - a.cu[s]
        lo = max(0, last + 1 - window) if window else 0
        for h in heads:
            x = slice(h * hd, h * hd + hd)
            nan = s == 0 and h // (nh // nkv) == nkv - 1 and last >= at // 16 * 16 and lo <= at // 16 * 16 + 15
            seen += nan
            if nan:
                assert np.isnan(got[r, x]).all(), (r, h)
            else:
                assert np.all(np.abs(got[r, x] - ref[r, x]) <= tol[r, x]), (r, h)
    assert seen
    assert np.array_equal(got[0], a.was[0]) and np.array_equal(got[-1], a.was[-1])
    heads = got[1:-1].reshape(-1, nh, hd)[:, :(nkv - 1) * (nh // nkv)]
    assert np.isfinite(heads).all()
    dev.free()


def test_mixed_graph(tg):
    """A mixed call captured once, replayed with other lengths: other tiles are cut then."""
    say("mixed graph")
    lib, dev = tg.lib(), Dev(tg)
    a = Attend(33, 16, 2, 64, [200, 1, 9, 1], [100, 2500, 900, 30], size=32, room=1200)
    for s in range(4):
        a.pages.fill(a.rng, s, a.max_kv)
    a.call(dev)
    done(tg)
    g = Graph(lambda stream: a.queue(lib, stream))
    for past in ([100, 2500, 900, 30], [3000, 5, 0, 3500], [0, 0, 3000, 0], [1500, 1500, 1500, 1500]):
        now = np.array(past, np.int32)
        lib.tg_hip_memcpy_h2d(a.len_ptr, now.ctypes.data, now.nbytes)
        lib.tg_hip_memcpy_h2d(a.out, a.was.ctypes.data, a.was.nbytes)
        g.replay()
        a.check(tg, dev, attend(a.q, a.pages, a.cu, a.lens, past, 16))
    g.free()
    dev.free()


def test_attention_mixed_many(tg):
    """More sequences than a wave looks at, and more tiles than are cut."""
    say("attention mixed, many sequences")
    _attend(tg, Attend(31, 8, 2, 32, [40 if i % 3 else 1 for i in range(150)], [(13 * i) % 600 for i in range(150)]))
    say("attention mixed, many tiles")
    _attend(tg, Attend(32, 64, 8, 16, [300] * 7 + [1, 0, 3], [(90 * i) % 500 for i in range(10)], room=200))


@pytest.mark.parametrize("nh,nkv,hd", [(1024, 16, 128), (1024, 1024, 16), (64, 1, 128), (1, 1, 128), (1024, 512, 16)])
def test_ends_of_the_layouts(tg, nh, nkv, hd):
    say(f"attention {nh, nkv, hd}")
    for lens, past in (([2, 1], [70, 0]), ([1], [600]), ([1, 3], [0, 20])):
        _attend(tg, Attend(nh + hd, nh, nkv, hd, lens, past, sinks=True))


def test_attention_many_sequences(tg):
    for n, window in ((200, 0), (700, 0), (700, 16), (3000, 0)):
        say(f"attention {n} sequences window={window}")
        _attend(tg, Attend(n, 4, 2, 32, [i % 3 for i in range(n)], [(7 * i) % 40 + (900 if i == 150 else 0) for i in range(n)], window=window,
                           lead=3 * (n > 200), tail=1))


def test_attention_over_q(tg):
    for lens, past in (([70, 3], [0, 9]), ([2], [3000])):
        say(f"attention over q {lens}")
        _attend(tg, Attend(3, 16, 2, 64, lens, past, lead=1, tail=1), place=True)


def test_attention_with_room(tg):
    """max_kv far above the lengths: another cut, the same rows."""
    for lens, past in (([1, 1], [30, 700]), ([40], [3]), ([300], [20]), ([9, 1], [500, 0])):
        say(f"attention with room {lens}")
        _attend(tg, Attend(4, 16, 2, 128, lens, past, 64, room=30000, sinks=True))


@pytest.mark.parametrize("q_scale", [1e-30, 1e-20, 1e-3, 300.0])
def test_attention_score_ranges(tg, q_scale):
    say(f"attention q_scale={q_scale}")
    for hd in (64, 128):
        _attend(tg, Attend(11, 8, 2, hd, [50, 1, 140], [20, 700, 0], q_scale=q_scale, sinks=True))
        a = Attend(12, 8, 2, hd, [50, 1, 140], [20, 700, 0], q_scale=q_scale)   # the smallest factor that a score can have
        a.pages.ek[:] = 127 + LEAST
        _attend(tg, a)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("lens,past", [([1, 3], [700, 90]), ([140], [60])])
def test_attention_exponents(tg, which, lens, past):
    """Blocks whose exponents are as far apart as they can be: those of V each in turn the largest, those of K small (any
    larger one of them is all that counts)."""
    say(f"attention exponents {which} {lens}")
    for hd in (64, 128):
        a = Attend(13, 8, 2, hd, lens, past, q_scale=0.5)
        exps = a.pages.ev if which == "v" else a.pages.ek
        exps[:] = np.random.default_rng(14).integers(127 + LEAST, (127 + MOST if which == "v" else 124) + 1, exps.shape)
        _attend(tg, a)
        a = Attend(15, 8, 2, hd, lens, past, q_scale=0.5)   # none near 1
        (a.pages.ev if which == "v" else a.pages.ek)[:] = 127 + LEAST
        _attend(tg, a)


def test_attention_zero_values(tg):
    """Blocks of zeros, with the least exponent, count in the sum and nowhere else."""
    say("attention zeros")
    for lens, past in (([1], [900]), ([150], [20])):
        for every in (2, 1):
            a = Attend(16, 8, 2, 64, lens, past, q_scale=0.5)
            blocks = a.pages.v.reshape(a.pages.n_pages, 2, -1, 16, 64)
            blocks[::every] = 0
            a.pages.ev[::every] = 127 + LEAST
            _attend(tg, a)


@pytest.mark.parametrize("lens,past", [([1, 5], [300, 20]), ([150], [16]), ([20, 1], [0, 3000])])
def test_attention_nan(tg, lens, past):
    """Rows that see a block that is NaN, in K or V, or a page that is none are NaN; the others are as they were; and so
    where a query is not finite."""
    for what in ("k", "v", "page", "byte", "q"):
        for window in (0, 20):
            say(f"attention nan {what} {lens} window={window}")
            a = Attend(17, 8, 2, 64, lens, past, size=32, window=window)
            before, tol = a.want()
            s, at = 0, max(0, (lens[0] + past[0]) // 2 - 3)
            page, b = a.pages.table[s, at // 32], at % 32 // 16
            if what in ("k", "v"):
                (a.pages.ek if what == "k" else a.pages.ev)[page, 1, b] = 255
            elif what == "byte":
                a.pages.ek[page, 0, b], a.pages.ev[page, 1, b] = 84, 170
            elif what == "page":
                a.pages.table[s, at // 32] = a.pages.n_pages
            else:
                a.q[0, 3], a.q[-1, -1] = np.nan, -np.inf
            # a row is NaN as a whole where it sees any position of such a block, also one whose weight is 0
            ref = before.copy()
            for s in range(a.n):
                for i in range(lens[s]):
                    lo, hi = max(0, past[s] + i + 1 - window) if window else 0, past[s] + i
                    gone = [np.isnan(a.pages.values(w, s, hi + 1)[:, lo:]).any((1, 2)) for w in "kv"]
                    r = a.cu[s] + i
                    for h in range(8):
                        if gone[0][h // 4] or gone[1][h // 4] or not np.isfinite(a.q[r, 64 * h:64 * h + 64]).all():
                            ref[r, 64 * h:64 * h + 64] = np.nan
            assert window or np.isnan(ref).any()
            dev = Dev(tg)
            a.call(dev)
            a.check(tg, dev, (ref, tol))
            dev.free()


def test_attention_left_out(tg):
    for past in (-1, 10 ** 6, 2 ** 31 - 1):
        say(f"attention left out past={past}")
        a, dev = Attend(18, 8, 2, 64, [3, 4, 2], [50, 60, 70]), Dev(tg)
        want = a.want()
        a.kv_len[1] = past
        a.call(dev)
        done(tg)
        got = dev.read(a.out, a.q)
        gone = slice(a.cu[1], a.cu[2])
        assert np.array_equal(got[gone], a.was[gone])
        keep = np.r_[0:3, 7:9]
        assert np.all(np.abs(got[keep] - want[0][keep]) <= want[1][keep])
        dev.free()
    for cu in ([0, 5, 4000], [-7, 3, 6], [4, 2, 1]):
        say(f"attention offsets {cu}")
        a, dev = Attend(19, 8, 2, 64, [3, 4], [50, 60]), Dev(tg)
        a.cu = np.array(cu, np.int32)
        a.call(dev)
        done(tg)
        dev.free()


def test_shared_pages(tg):
    """Sequences whose tables begin with the same pages, and pages listed twice by one."""
    say("shared pages")
    a = Attend(20, 8, 2, 128, [1, 5, 40], [96, 90, 64], size=32)
    a.pages.table[1, :2] = a.pages.table[2, :2] = a.pages.table[0, :2]
    a.pages.table[2, 1] = a.pages.table[2, 0]
    _attend(tg, a)


def test_null_lengths(tg):
    """Without kv_len every sequence begins at position 0."""
    say("null kv_len")
    lib, dev = tg.lib(), Dev(tg)
    x = Append(34, 8, 2, 64, [20, 3, 40], [0, 0, 0], 32, rot=16)
    x.call(dev)
    args = list(x.args)
    args[14] = None
    for ptr, t in zip(x.ptr, x.pages.arrays()):
        lib.tg_hip_memcpy_h2d(ptr, t.ctypes.data, t.nbytes)
    lib.tg_hip_paged_append_dev(*args, None)
    x.check(tg, dev)
    a = Attend(35, 8, 2, 64, [20, 3, 40], [0, 0, 0], 32)
    a.call(dev)
    args = list(a.args)
    args[11] = None
    lib.tg_hip_memcpy_h2d(a.out, a.was.ctypes.data, a.was.nbytes)
    lib.tg_hip_attention_paged_dev(*args, None)
    a.check(tg, dev)
    dev.free()


@pytest.mark.parametrize("n,nh,nkv,hd", [(128, 32, 4, 128), (100, 64, 8, 64), (300, 8, 1, 96)])
def test_single_tokens_of_many(tg, n, nh, nkv, hd):
    """Single tokens whose lengths lie far apart: the long ones are cut, more sequences than a wave looks at at once."""
    say(f"single tokens of {n} sequences {nh, nkv, hd}")
    past = [(37 * i * i) % 90 for i in range(n)]
    past[n // 2], past[3], past[-1] = 9000, 5000, 7001
    lens = [1] * n
    lens[5] = 0
    a, dev = Attend(n, nh, nkv, hd, lens, past, 64, sinks=hd == 64), Dev(tg)
    rows = [0, 1, 3, 4, 5, n // 2 - 1, n // 2, n - 2] + [int(r) for r in a.rng.integers(0, n - 1, 10)]
    only = {r: [0, nh // 2, nh - 1] for r in rows}
    ref, tol = attend(a.q, a.pages, a.cu, lens, past, nh, 0, a.sinks, only)
    a.call(dev)
    done(tg)
    got = dev.read(a.out, a.q)
    for r, heads in only.items():
        for h in heads:
            x = slice(h * hd, h * hd + hd)
            assert np.all(np.abs(got[r, x] - ref[r, x]) <= tol[r, x]), (r, h)
    assert np.isfinite(got).all()
    dev.free()


# ------------------------------------------------------------------ graphs, streams, together

def test_graph(tg):
    """An append and the attention behind it, captured once and replayed with lengths that the caller advances."""
    say("paged graph")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(21)
    a = Attend(22, 8, 2, 64, [1, 1], [20, 350], size=16, room=8)
    x = Append(23, 8, 2, 64, [1, 1], [20, 350], rope_len=400)
    x.pages = a.pages
    x.call(dev)
    a.q = x.x[:, :8 * 64].copy()
    a.call(dev)
    done(tg)
    # one pool, one table, one array of lengths for both; the append's queries are the attention's
    xa, aa = list(x.args), list(a.args)
    xa[28:30] = aa[:2]
    aa[2:6] = xa[17:21]
    aa[8] = xa[23]
    xa[14] = aa[11]
    for i, t in enumerate(a.pages.arrays()):
        lib.tg_hip_memcpy_h2d(x.ptr[i], t.ctypes.data, t.nbytes)

    def queue(stream):
        lib.tg_hip_paged_append_dev(*xa, stream)
        lib.tg_hip_attention_paged_dev(*aa, stream)
    g = Graph(queue)
    done(tg)
    pages = a.pages.copy()
    for step in range(5):
        x.x = rng.standard_normal(x.x.shape).astype(np.float32)
        x.past = [20 + step, 350 + step]
        now = np.array(x.past, np.int32)
        lib.tg_hip_memcpy_h2d(x.x_ptr, x.x.ctypes.data, x.x.nbytes)
        lib.tg_hip_memcpy_h2d(xa[14], now.ctypes.data, now.nbytes)
        g.replay()
        x.pages = pages
        q, pages = x.want()
        ref, tol = attend(q.astype(np.float32), pages, a.cu, [1, 1], x.past, 8)
        done(tg)
        got = dev.read(a.out, a.q)
        assert np.all(np.abs(got - ref) <= tol + (8 * np.abs(q).max() * 64 ** 0.5 * 8 * EPS) * np.abs(ref).max())
        for t, ptr in zip(pages.arrays(), x.ptr):
            assert np.array_equal(dev.read(ptr, t), t)
    g.free()
    dev.free()


def test_two_streams(tg):
    """Two calls at once, each with scratch of its own."""
    from tests.test_gpu_decode import _hip_runtime
    say("paged on two streams")
    hip, lib, dev = _hip_runtime(), tg.lib(), Dev(tg)
    streams = [ctypes.c_void_p() for _ in range(2)]
    for s in streams:
        assert hip.hipStreamCreate(ctypes.byref(s)) == 0
    calls = [Attend(24, 32, 4, 128, [9], [4000], 64), Attend(25, 8, 2, 64, [1] * 5, [2000, 5, 300, 1, 900])]
    want = [c.want() for c in calls]
    for c, s in zip(calls, streams):
        c.call(dev, s)
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.queue(lib, s)
    for s in streams:
        assert hip.hipStreamSynchronize(s) == 0
    for c, w in zip(calls, want):
        c.check(tg, dev, w)
    for s in streams:
        assert hip.hipStreamDestroy(s) == 0
    dev.free()


def test_offsets_past_32_bits(tg):
    """A pool of more than 4 GiB whose last pages are used."""
    say("pool past 4 GiB")
    lib, dev = tg.lib(), Dev(tg)
    a = Attend(26, 4, 2, 128, [3], [90], size=1024, sinks=True)
    p = a.pages
    want = a.want()
    total = (5 << 30) // (2 * 1024 * 128)
    shift = total - p.n_pages
    a.call(dev)
    done(tg)
    args = list(a.args)
    for i, t in zip(range(2, 6), p.arrays()):
        size = t[0].nbytes
        ptr = dev.room(total * size)
        lib.tg_hip_memcpy_h2d(ptr + shift * size, np.ascontiguousarray(t).ctypes.data, t.nbytes)
        args[i] = ptr
    table = np.where(p.table >= 0, p.table + shift, -1).astype(np.int32)
    args[6], args[8] = total, dev(table)
    a.args = tuple(args)
    lib.tg_hip_memcpy_h2d(a.out, a.was.ctypes.data, a.was.nbytes)
    a.queue(lib)
    a.check(tg, dev, want)
    # an append and a read at the same place
    x = Append(27, 4, 2, 128, [20], [40], size=1024)
    x.pages = p
    q, after = x.want()
    x.call(dev)
    xa = list(x.args)
    xa[17:21], xa[21], xa[23], xa[24] = args[2:6], total, args[8], table.shape[1]
    lib.tg_hip_paged_append_dev(*xa, None)
    out = [dev(np.zeros((1, 2, 64, 128), np.float32)) for _ in range(2)]
    lib.tg_hip_paged_read_dev(*args[2:6], total, 1024, args[8], table.shape[1], dev(np.array([60], np.int32)), 1, 2, 128, 0, *out, None, 1, 64, None)
    done(tg)
    for which, ptr in zip("kv", out):
        got = dev.read(ptr, np.zeros((1, 2, 64, 128), np.float32))
        assert np.array_equal(got[0, :, :60], after.values(which, 0, 60).astype(np.float32)) and not got[0, :, 60:].any()
    dev.free()


@pytest.mark.parametrize("inter", [0, 1])
def test_a_conversation(tg, inter):
    """As a program uses them: tables by parts, a prompt and its answers into pages, attention over them at each step,
    then the pages read into f16 slots, where the packed attention of dense caches goes on."""
    say(f"a conversation inter={inter}")
    lib, dev, rng = tg.lib(), Dev(tg), np.random.default_rng(28 + inter)
    nh, nkv, hd, rot, size, room = 8, 2, 64, 32, 16, 160
    cos, sin = dev(np.zeros((room, rot // 2), np.float32)), dev(np.zeros((room, rot // 2), np.float32))
    lib.tg_hip_clear_error()
    lib.tg_hip_rope_tables_dev(cos, sin, room, 0, rot, 150000.0, tg.ROPE_PARTS, 32.0, 4096, 32.0, 1.0, 1.3465736, None)
    done(tg)
    a = Append(29, nh, nkv, hd, [1, 1], [0, 0], rot=rot, inter=inter)
    a.cos, a.sin = (dev.read(t, np.zeros((room, rot // 2), np.float32)) for t in (cos, sin))
    a.rope_len, a.pages = room, Pages(rng, 2, nkv, hd, size, room)
    ptr = [dev(t) for t in a.pages.arrays()]
    table = dev(a.pages.table)
    scratch = dev.room(lib.tg_hip_attention_paged_scratch_bytes(200, 2, nh, nkv, hd, room))
    past = [0, 0]
    for lens in ([100, 37], [1, 1], [1, 5], [0, 1], [9, 1]):
        a.lens, a.past, a.rows = lens, past, sum(lens)
        a.cu, a.kv_len = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), np.array(past, np.int32)
        a.x = (rng.standard_normal((a.rows, (nh + 2 * nkv) * hd)) * 1.5).astype(np.float32)
        x, w, qd, kd = dev(a.x), a.x.shape[1], 4 * nh * hd, 4 * nkv * hd
        q, out = dev(np.zeros((a.rows, nh * hd), np.float32)), dev(np.zeros((a.rows, nh * hd), np.float32))
        seqs = (dev(a.cu), dev(a.kv_len), 2, a.rows)
        pool = (*ptr, a.pages.n_pages, size, table, a.pages.table.shape[1])
        lib.tg_hip_paged_append_dev(x, x + qd, x + qd + kd, w, w, None, None, 1e-6, cos, sin, room, rot, inter, *seqs, *pool, nh, nkv, hd, q,
                                    nh * hd, None)
        lib.tg_hip_attention_paged_dev(q, nh * hd, *pool, *seqs, room, 0, None, nh, nkv, hd, out, nh * hd, scratch, None)
        done(tg)
        turned, a.pages = a.want()
        got_q = dev.read(q, np.zeros((a.rows, nh * hd), np.float32))
        assert np.abs(got_q - turned).max() <= 8 * EPS * np.abs(turned).max()
        ref, tol = attend(got_q, a.pages, a.cu, lens, past, nh)
        assert np.all(np.abs(dev.read(out, ref.astype(np.float32)) - ref) <= tol)
        for t, p in zip(a.pages.arrays(), ptr):
            assert np.array_equal(dev.read(p, t), t)
        past = [x + y for x, y in zip(past, lens)]
    slots = [dev(np.zeros((2, nkv, room, hd), np.float16)) for _ in range(2)]
    lib.tg_hip_paged_read_dev(*ptr, a.pages.n_pages, size, table, a.pages.table.shape[1], dev(np.array(past, np.int32)), 2, nkv, hd, 1, *slots,
                              None, 2, room, None)
    # the last call's rows again, over the slots: bytes times powers of two near 1 are exact in f16
    more = dev.room(lib.tg_hip_attention_prompt_scratch_bytes(10, 2, nh, nkv, hd, room, 0))
    lib.tg_hip_attention_prompt_dev(q, nh * hd, 1, *slots, 2, room, *seqs[:2], None, 2, a.rows, 0, None, nh, nkv, hd, out, nh * hd, more, None)
    done(tg)
    assert np.all(np.abs(dev.read(out, ref.astype(np.float32)) - ref) <= tol)
    dev.free()
