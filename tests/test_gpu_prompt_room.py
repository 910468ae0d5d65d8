"""GPU checks of packed attention where caches have room for much more than is
in them, and of what a call leaves alone when its offsets are wrong."""

import sys

import numpy as np
import pytest

from tests._packed import Batch, Dev

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def _roomy(b, kv_max):
    """The batch's caches with room for kv_max positions, NaN behind those in use."""
    for name in "kv":
        t = getattr(b, name)
        big = np.full((b.n_slots, b.nkv, kv_max, b.hd), np.nan, b.dtype)
        big[:, :, :t.shape[2]] = t
        setattr(b, name, big)
    b.kv_max = kv_max
    return b


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,lens,past,prefix,window", [
    (32, 4, 128, [16], [0], 0, 0), (32, 4, 128, [128], [0], 0, 0), (64, 8, 64, [300], [0], 0, 0), (64, 8, 64, [600], [3], 0, 0),
    (32, 4, 128, [9], [1000], 0, 0), (32, 4, 128, [1] * 8, [300, 0, 1, 63, 64, 65, 127, 2], 0, 0),
    (8, 2, 64, [40, 0, 1, 200], [0, 3, 700, 11], 0, 0), (64, 8, 64, [150, 160], [0, 40], 0, 100),
    (32, 4, 128, [1] * 20, [3 * i for i in range(20)], 500, 0), (8, 2, 64, [1, 30, 2], [0, 5, 64], 200, 0)])
def test_short_sequences_in_large_caches(tg, nh, nkv, hd, lens, past, prefix, window, half):
    """The host cuts a call by kv_max, the device by what is there: shapes and
    spans that are made for long sequences, on short ones."""
    say(f"large caches {nh, nkv, hd} lens={lens[:4]} past={past[:4]} prefix={prefix} window={window} half={half}")
    b = Batch(nh + len(lens), nh, nkv, hd, lens, past, half, window=window, prefix=prefix, sinks=hd == 64, lead=1, tail=1)
    _roomy(b, 32768)
    dev = Dev(tg)
    tg.lib().tg_hip_clear_error()
    out, was = b.call(dev)
    tg.lib().tg_hip_synchronize()
    assert tg.last_error() == "", tg.last_error()
    got = dev.read(out, b.q)
    dev.free()
    say(f"  worst error / tolerance {b.check(got, was):.3f}")


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("past", [50, 3000])
@pytest.mark.parametrize("half", [False, True])
def test_wrong_offsets_write_nothing_else(tg, half, past, prefix):
    """Offsets past the rows, negative ones and decreasing ones: rows that lie
    between no offset and the next, the values between rows, and the memory
    around the output and the scratch stay as they were."""
    lib = tg.lib()
    for cu in ([0, 5, 4000], [-7, 3, 6], [4, 2, 1], [2, 2 ** 31 - 1, 5], [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1]):
        say(f"wrong offsets {cu} half={half} past={past} prefix={prefix}")
        b = Batch(2, 8, 2, 64, [3, 4], [past, 60], half, prefix=prefix, pad=4)
        dev = Dev(tg)
        lib.tg_hip_clear_error()
        b.call(dev)
        lib.tg_hip_synchronize()
        need = lib.tg_hip_attention_prompt_scratch_bytes(b.rows, b.n, b.nh, b.nkv, b.hd, b.kv_max, prefix)
        guard = 1 << 16
        outs = np.full(guard // 2 + b.rows * b.stride, 7.5, np.float32)
        scratch = np.full(2 * guard + need, 0x5A, np.uint8)
        po, ps = dev(outs), dev(scratch)
        b.ptrs["out"], b.scratch = po + guard, ps + guard
        b.ptrs["cu"] = dev(np.array(cu, np.int32))
        b.queue(lib)
        lib.tg_hip_synchronize()
        assert tg.last_error() == "", tg.last_error()
        got, after = dev.read(po, outs), dev.read(ps, scratch)
        dev.free()
        assert np.all(after[:guard] == 0x5A) and np.all(after[guard + need:] == 0x5A)
        first, last = guard // 4, guard // 4 + b.rows * b.stride
        assert np.all(got[:first] == 7.5) and np.all(got[last:] == 7.5)
        rows = got[first:last].reshape(b.rows, b.stride)
        assert np.all(rows[:, b.nh * b.hd:] == 7.5)
        r = np.arange(b.rows)
        held = np.any([(lo <= r) & (r < hi) for lo, hi in zip(cu, cu[1:])], axis=0)
        assert np.all(rows[~held] == 7.5)
