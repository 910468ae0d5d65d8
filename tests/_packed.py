"""Packed rows of several sequences for the tests of the prompt and batch
path: cases, their plain computation in 64 bits, device copies, HIP graphs."""

import ctypes

import numpy as np

EPS = 2.0 ** -24   # half a step of float32, relative


class Graph:
    """The work that `queue(stream)` queues, captured once."""

    def __init__(self, queue):
        from tests.test_gpu_decode import _hip_runtime
        self.hip, self.s, graph, self.exe = _hip_runtime(), ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamCreate(ctypes.byref(self.s)) == 0
        assert self.hip.hipStreamBeginCapture(self.s, 1) == 0   # thread-local
        queue(self.s)
        assert self.hip.hipStreamEndCapture(self.s, ctypes.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exe), graph, None, None, 0) == 0
        self.hip.hipGraphDestroy(graph)

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exe, self.s) == 0
        assert self.hip.hipStreamSynchronize(self.s) == 0

    def free(self):
        self.hip.hipGraphExecDestroy(self.exe)
        self.hip.hipStreamDestroy(self.s)


class Dev:
    """Device copies of arrays, freed together."""

    def __init__(self, tg):
        self.tg, self.keep = tg, []

    def __call__(self, a, offset=0):
        """The pointer of a copy of `a` (None: a null pointer), `offset` bytes into its allocation."""
        if a is None:
            return None
        a = np.ascontiguousarray(a)
        d = self.tg.DeviceArray(a.nbytes + offset + 16)
        d.upload(a, offset)
        self.keep.append(d)
        return d.ptr + offset

    def room(self, nbytes):
        d = self.tg.DeviceArray(max(int(nbytes), 16))
        self.keep.append(d)
        return d.ptr

    def read(self, ptr, like):
        out = np.empty(like.shape, like.dtype)
        self.tg.lib().tg_hip_memcpy_d2h(out.ctypes.data, ptr, out.nbytes)
        return out

    def free(self):
        for d in self.keep:
            d.free()
        self.keep = []


class Batch:
    """Sequences of `lens` rows behind `past` cached positions, packed, in
    slots of a cache of `n_slots`; prefix > 0: behind that many shared ones.
    What no row may see is NaN: the other slots, and each slot's tail."""

    def __init__(self, seed, nh, nkv, hd, lens, past, half, window=0, sinks=False, prefix=0, lead=0, tail=0, pad=0,
                 q_scale=2.0, hide=np.nan):
        rng = np.random.default_rng(seed)
        self.nh, self.nkv, self.hd, self.window, self.prefix, self.half = nh, nkv, hd, window, prefix, half
        self.lens, self.past = list(lens), list(past)
        self.n, self.lead = len(lens), lead
        self.rows = lead + sum(lens) + tail
        self.dtype = np.float16 if half else np.float32
        self.stride = nh * hd + pad
        self.q = (rng.standard_normal((self.rows, self.stride)) * q_scale).astype(np.float32)
        top = max([a + b for a, b in zip(lens, past)], default=0)
        self.kv_max = max(1, top + int(rng.integers(0, 9)))
        self.n_slots = self.n + 2
        self.slots = rng.permutation(self.n_slots)[:self.n].astype(np.int32)
        self.k = np.full((self.n_slots, nkv, self.kv_max, hd), hide, self.dtype)
        self.v = self.k.copy()
        for s, slot in enumerate(self.slots):
            m = lens[s] + past[s]
            self.k[slot, :, :m] = rng.standard_normal((nkv, m, hd))
            self.v[slot, :, :m] = rng.standard_normal((nkv, m, hd))
        self.pre_max = prefix + 3
        self.pk = np.full((nkv, self.pre_max, hd), hide, self.dtype)
        self.pv = self.pk.copy()
        self.pk[:, :prefix] = rng.standard_normal((nkv, prefix, hd))
        self.pv[:, :prefix] = rng.standard_normal((nkv, prefix, hd))
        self.sinks = rng.standard_normal(nh).astype(np.float32) if sinks else None
        self.cu = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
        self.kv_len = np.array(self.past, np.int32)

    def seen(self, s, i):
        """First and last position (of prefix and slot together) that row i of sequence s sees."""
        last = self.prefix + self.past[s] + i
        return (max(0, last + 1 - self.window) if self.window else 0), last

    def attend(self):
        """(out, tolerance) of every row, NaN rows where no sequence is; 64 bits.

        Tolerance: a score is a sum of hd products, each product and sum
        rounded once, partial sums of at most B = scale * sum |q_d k_d|: off
        by about sqrt(2 hd) EPS B; eight times that and four steps for
        operands split in two halves of 11 bits.  A weight is off by that
        and the exponential's few steps; numerator and denominator are sums
        of n such terms.  All relative to the largest |v|."""
        out = np.full((self.rows, self.nh * self.hd), np.nan)
        tol = np.zeros((self.rows, self.nh * self.hd))
        group, scale = self.nh // self.nkv, self.hd ** -0.5
        for s in range(self.n):
            m = self.past[s] + self.lens[s]
            keys = np.concatenate([self.pk[:, :self.prefix], self.k[self.slots[s], :, :m]], 1).astype(np.float64)
            vals = np.concatenate([self.pv[:, :self.prefix], self.v[self.slots[s], :, :m]], 1).astype(np.float64)
            for i in range(self.lens[s]):
                r = self.cu[s] + i
                lo, hi = self.seen(s, i)
                for h in range(self.nh):
                    q = self.q[r, h * self.hd:(h + 1) * self.hd].astype(np.float64)
                    kk, vv = keys[h // group, lo:hi + 1], vals[h // group, lo:hi + 1]
                    z = (kk @ q) * scale
                    top = z.max()
                    if self.sinks is not None:
                        top = max(top, float(self.sinks[h]))
                    p = np.exp(z - top)
                    den = p.sum() + (np.exp(float(self.sinks[h]) - top) if self.sinks is not None else 0.0)
                    at = slice(h * self.hd, (h + 1) * self.hd)
                    out[r, at] = (p @ vv) / den
                    big = (np.abs(kk) @ np.abs(q)).max() * scale
                    off = (8 * np.sqrt(2 * self.hd) + 4) * EPS * big + (8 * np.sqrt(len(z)) + 24) * EPS
                    tol[r, at] = 2 * off * np.abs(vv).max()
        return out, tol

    def call(self, dev, scratch=None, stream=None, in_place=False):
        """Queues the attention call over device copies; returns (out pointer, what it held before)."""
        lib = dev.tg.lib()
        sentinel = self.q.copy() if in_place else np.full((self.rows, self.stride), 7.5, np.float32)
        q = dev(self.q, 4)   # rows at 4 mod 16 bytes
        out = q if in_place else dev(sentinel, 4)
        self.ptrs = dict(q=q, out=out, k=dev(self.k), v=dev(self.v), cu=dev(self.cu), len=dev(self.kv_len),
                         slots=dev(self.slots), sinks=dev(self.sinks), pk=dev(self.pk), pv=dev(self.pv))
        if scratch is None:
            need = lib.tg_hip_attention_prompt_scratch_bytes(self.rows, self.n, self.nh, self.nkv, self.hd, self.kv_max,
                                                             self.prefix)
            scratch = dev.room(need)
        self.scratch = scratch
        self.queue(lib, stream)
        return out, sentinel

    def queue(self, lib, stream=None):
        p = self.ptrs
        front = (p["q"], self.stride, int(self.half), p["k"], p["v"], self.n_slots, self.kv_max)
        back = (p["cu"], p["len"], p["slots"], self.n, self.rows, self.window, p["sinks"], self.nh, self.nkv, self.hd,
                p["out"], self.stride, self.scratch, stream)
        if self.prefix:
            lib.tg_hip_attention_prefix_dev(*front, p["pk"], p["pv"], self.prefix, self.pre_max, *back)
        else:
            lib.tg_hip_attention_prompt_dev(*front, *back)

    def check(self, got, sentinel, ref=None):
        """Rows of sequences within tolerance, everything else as it was."""
        out, tol = self.attend() if ref is None else ref
        w = self.nh * self.hd
        live = np.zeros(self.rows, bool)
        live[self.lead:self.lead + sum(self.lens)] = True
        assert np.array_equal(got[~live], sentinel[~live]), "rows of no sequence were written"
        assert np.array_equal(got[:, w:], sentinel[:, w:]), "values between the rows were written"
        if not live.any():
            return 0.0
        err = np.abs(got[live, :w] - out[live])
        assert np.all(np.isfinite(got[live, :w])), "not finite"
        worst = float((err / tol[live]).max())
        assert worst <= 1.0, (worst, float(err.max()))
        return worst
