"""Sequences in 8-bit pages for the tests: how rows are held, positions read
back, attention over them, all plain and in 64 bits."""

import numpy as np

from tests._packed import EPS

LEAST, MOST, NAN = -42, 42, 255


def turn(x, cos, sin, rot, inter):
    """x [..., head_dim], cos and sin [..., rot / 2] (broadcast), in 64 bits."""
    y = x.copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    return y


def tables(n, rot, theta=1e4):
    angle = np.arange(n)[:, None] * theta ** (-2 * np.arange(rot // 2) / rot)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def exponent(big):
    """The least e in LEAST .. MOST with big <= 127 2^e; MOST + 1 where there is none."""
    for e in range(LEAST, MOST + 1):
        if big <= 127.0 * 2.0 ** e:
            return e
    return MOST + 1


class Pages:
    """A pool of pages and the tables of n sequences with room for `room` positions each; pages lie anywhere."""

    def __init__(self, rng, n, nkv, hd, size, room, spare=2, more=1):
        self.nkv, self.hd, self.size = nkv, hd, size
        per = -(-room // size)
        self.n_pages = n * per + spare
        self.k, self.v = (rng.integers(-127, 128, (self.n_pages, nkv, size, hd)).astype(np.int8) for _ in range(2))   # stale rows
        self.ek, self.ev = (rng.integers(110, 140, (self.n_pages, nkv, size // 16)).astype(np.uint8) for _ in range(2))
        self.table = np.full((n, per + more), -1, np.int32)
        self.table[:, :per] = rng.permutation(self.n_pages)[:n * per].reshape(n, per)

    def arrays(self):
        return self.k, self.v, self.ek, self.ev

    def copy(self):
        p = object.__new__(Pages)
        p.__dict__.update({a: (b.copy() if isinstance(b, np.ndarray) else b) for a, b in self.__dict__.items()})
        return p

    def fill(self, rng, s, n, spread=1):
        """n positions of sequence s: values of about 1, blocks' exponents within `spread` of each other."""
        for arr, exps in ((self.k, self.ek), (self.v, self.ev)):
            for j in range(-(-n // 16)):
                page, b = self.table[s, 16 * j // self.size], 16 * j % self.size // 16
                x = np.clip(np.rint(rng.standard_normal((self.nkv, 16, self.hd)) * 36), -127, 127)
                arr[page, :, 16 * b:16 * b + 16] = x
                exps[page, :, b] = 127 - 5 + rng.integers(-spread, spread + 1, self.nkv)

    def values(self, which, s, n):
        """Positions 0 .. n - 1 of sequence s [n_kv][n][head_dim]; NaN where there is no page or no such exponent."""
        arr, exps = (self.k, self.ek) if which == "k" else (self.v, self.ev)
        out = np.full((self.nkv, n, self.hd), np.nan)
        for j in range(-(-n // 16)):
            page, b, m = self.table[s, 16 * j // self.size], 16 * j % self.size // 16, min(16, n - 16 * j)
            if 0 <= page < self.n_pages:
                e = exps[page, :, b].astype(int) - 127
                unit = np.where((e >= LEAST) & (e <= MOST), 2.0 ** e, np.nan)
                out[:, 16 * j:16 * j + m] = arr[page, :, 16 * b:16 * b + m] * unit[:, None, None]
        return out

    def store(self, which, s, past, rows, live):
        """rows [n][n_kv][head_dim] in 64 bits at positions past .. of sequence s, of which live[i] are stored."""
        arr, exps = (self.k, self.ek) if which == "k" else (self.v, self.ev)
        n = len(rows)
        for j in range(past // 16, -(-(past + n) // 16) if n else 0):
            page, b = self.table[s, 16 * j // self.size], 16 * j % self.size // 16
            at = [p for p in range(max(past, 16 * j), min(past + n, 16 * j + 16)) if live[p - past]]
            if not 0 <= page < self.n_pages or not at:
                continue
            held = min(16, max(0, past - 16 * j))
            for h in range(self.nkv):
                new = np.array([rows[p - past, h] for p in at])
                e = exponent(np.abs(new).max()) if np.all(np.isfinite(new)) else MOST + 1
                old = int(exps[page, h, b]) - 127
                if held:
                    e = max(e, old) if LEAST <= old <= MOST else MOST + 1
                if e > MOST:
                    exps[page, h, b] = NAN
                    continue
                block = arr[page, h, 16 * b:16 * b + 16]
                if held and e > old:
                    block[:held] = np.rint(block[:held] * 2.0 ** (old - e))
                for p, x in zip(at, new):
                    block[p - 16 * j] = np.rint(x * 2.0 ** -e)
                exps[page, h, b] = e + 127


def attend(q, pages, cu, lens, past, nh, window=0, sinks=None, only=None):
    """(out, tolerance) of every packed row (`only`: of these rows, a dict of row: heads), NaN where no sequence is;
    q [rows][nh * hd].

    Tolerance, in natural units of a score, all relative to the largest |v|.
    q is held to half a step of 2^-22 of its head's largest value Q, times the
    sum of |k|: 2^-22.9 Q sum |k| / sqrt(hd).  Joining the digits, the
    factor's constants and products and the exponent's sum round six times a score
    of at most B, and once a number of at most B and what the exponents add
    (64).  Each counts for numerator and denominator.  Weights in two f16 are
    off by 2^-22, the exponential by a few steps; sums of n terms by
    about sqrt(n) of them, times eight; what f16 cannot hold of a weight is below
    2^-33 of a reference that is less than twice the largest weight times unit, of
    which values are at most 127, and the largest value at least 63: n 2^-31."""
    rows, hd, nkv = len(q), pages.hd, pages.nkv
    out, tol = np.full((rows, nh * hd), np.nan), np.zeros((rows, nh * hd))
    group, scale = nh // nkv, hd ** -0.5
    for s, (n, p) in enumerate(zip(lens, past)):
        keys, vals = pages.values("k", s, p + n), pages.values("v", s, p + n)
        for i in range(n) if only is None else [r - cu[s] for r in only if 0 <= r - cu[s] < n]:
            last = p + i
            lo = max(0, last + 1 - window) if window else 0
            for h in range(nh) if only is None else only[cu[s] + i]:
                k, v = keys[h // group, lo:last + 1], vals[h // group, lo:last + 1]
                x = q[cu[s] + i, h * hd:(h + 1) * hd].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    z = k @ x * scale
                    m = max(z.max(), -np.inf if sinks is None else float(sinks[h]))
                    w = np.exp(z - m)
                    total = w.sum() + (0 if sinks is None else np.exp(float(sinks[h]) - m))
                    y = w @ v / total
                    big = scale * (np.abs(k) @ np.abs(x)).max()
                    off = 2.0 ** -22.9 * np.abs(x).max() * np.abs(k).sum(1).max() * scale + (7 * big + 64) * EPS
                    t = (2 * off + (8 * np.sqrt(len(z)) + 24) * EPS + len(z) * 2.0 ** -31) * np.abs(v).max()
                out[cu[s] + i, h * hd:(h + 1) * hd] = y
                tol[cu[s] + i, h * hd:(h + 1) * hd] = t
    return out, tol
