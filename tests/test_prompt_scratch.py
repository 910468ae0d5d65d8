"""The scratch of packed attention: one allocation for a program's largest
sizes has to serve its smaller calls, which may need more than large ones."""

import numpy as np
import pytest

P = 1 << 20   # stands for a device pointer that must not be followed


def _draw(rng):
    nkv = int(rng.choice([1, 2, 3, 4, 8, 16]))
    nh = nkv * int(rng.choice([1, 2, 4, 5, 8, 16]))
    prefix = int(rng.choice([0, 1])) * int(2 ** rng.uniform(0, 15))
    return nh, nkv, int(rng.choice([8, 64, 80, 128])), int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 9)), int(
        2 ** rng.uniform(0, 18)), prefix


def _smaller(rng, n):
    return int(rng.choice([n, max(1, n // 2), max(1, int(n ** rng.uniform(0, 1)))]))


def _need(tg, half, n_rows, n_seqs, nh, nkv, hd, kv_max, prefix, window, p=P, cu=P):
    """What a call says it needs, given none."""
    lib = tg.lib()
    front = (p, nh * hd, half, p, p, 1, kv_max)
    back = (cu, cu, None, n_seqs, n_rows, window, None, nh, nkv, hd, p, nh * hd, None, None)
    lib.tg_hip_clear_error()
    if prefix:
        lib.tg_hip_attention_prefix_dev(*front, p, p, prefix, prefix, *back)
    else:
        lib.tg_hip_attention_prompt_dev(*front, *back)
    e = tg.last_error()
    lib.tg_hip_clear_error()
    return int(e.split("needs ")[1].split()[0]) if e else 0


def test_the_size_of_a_prompt_holds_its_decode_steps(tg):
    size = tg.lib().tg_hip_attention_prompt_scratch_bytes
    last = 0
    for rows in (1, 2, 4, 9, 17, 60, 128, 129, 300, 512, 1024, 2000, 4096, 8192):
        got = size(rows, 1, 32, 4, 128, 8192, 0)
        assert got >= last, (rows, got, last)
        last = got
    assert last <= 64 << 20


def test_sizes_rise_with_every_argument(tg):
    size, rng = tg.lib().tg_hip_attention_prompt_scratch_bytes, np.random.default_rng(1)
    for _ in range(20000):
        nh, nkv, hd, n_rows, n_seqs, kv_max, prefix = _draw(rng)
        a, b, c = (_smaller(rng, x) for x in (n_rows, n_seqs, kv_max))
        d = _smaller(rng, prefix) if prefix else 0
        most, less = size(n_rows, n_seqs, nh, nkv, hd, kv_max, prefix), size(a, b, nh, nkv, hd, c, d)
        assert less <= most, (nh, nkv, hd, (n_rows, n_seqs, kv_max, prefix, most), (a, b, c, d, less))


def test_smaller_calls_behind_a_prefix(tg):
    """These always need scratch, so the call is refused and no device is asked."""
    size, rng = tg.lib().tg_hip_attention_prompt_scratch_bytes, np.random.default_rng(2)
    for _ in range(4000):
        nh, nkv, hd, n_rows, n_seqs, kv_max, prefix = _draw(rng)
        prefix = max(prefix, 1)
        most = size(n_rows, n_seqs, nh, nkv, hd, kv_max, prefix)
        a, b, c, d = (_smaller(rng, x) for x in (n_rows, n_seqs, kv_max, prefix))
        for half in (0, 1):
            window = int(rng.choice([0, int(2 ** rng.uniform(0, 18))]))
            need = _need(tg, half, a, b, nh, nkv, hd, c, d, window)
            assert 0 < need <= most, (nh, nkv, hd, (n_rows, n_seqs, kv_max, prefix, most), (a, b, c, d, window, half, need))


@pytest.mark.gpu
def test_smaller_calls(tg):
    """The calls have no rows on the device: those that need nothing run."""
    from tests._packed import Dev
    print("scratch of smaller calls", flush=True)
    size, rng, dev, seen = tg.lib().tg_hip_attention_prompt_scratch_bytes, np.random.default_rng(3), Dev(tg), 0
    p, cu = dev(np.zeros(1 << 16, np.float32)), dev(np.zeros(1 << 14, np.int32))
    for _ in range(4000):
        nh, nkv, hd, n_rows, n_seqs, kv_max, prefix = _draw(rng)
        most = size(n_rows, n_seqs, nh, nkv, hd, kv_max, prefix)
        a, b, c = (_smaller(rng, x) for x in (n_rows, n_seqs, kv_max))
        d = _smaller(rng, prefix) if prefix else 0
        half, window = int(rng.integers(2)), int(rng.choice([0, int(2 ** rng.uniform(0, 18))]))
        need = _need(tg, half, a, b, nh, nkv, hd, c, d, window, p, cu)
        assert need <= most, (nh, nkv, hd, (n_rows, n_seqs, kv_max, prefix, most), (a, b, c, d, window, half, need))
        seen += need > 0
    tg.lib().tg_hip_synchronize()
    dev.free()
    assert seen > 1000
