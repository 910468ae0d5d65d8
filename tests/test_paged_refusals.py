"""Arguments that the calls of paged caches and rotary positions refuse, calls
with nothing to do, and scratch sizes: no device work, so no GPU."""

import math

import numpy as np
import pytest

P = 1 << 20   # stands for a device pointer that must not be followed


def _tables(**kw):
    a = dict(cos=P, sin=P, len=10, first=0, rot=64, theta=1e4, scaling=0, factor=1.0, orig=4096, low=32.0, high=1.0, m=1.0, stream=None)
    a.update(kw)
    return list(a.values())


def _rope(**kw):
    a = dict(x=P, x_stride=512, pos=P, cos=P, sin=P, len=10, rot=64, inter=0, rows=3, nh=8, hd=64, out=2 * P, out_stride=512, stream=None)
    a.update(kw)
    return list(a.values())


PAGES = dict(pk=P, pv=P, ek=P, ev=P, n_pages=4, size=16, table=P, stride=8)


def _append(**kw):
    a = dict(q=P, k=P, v=P, q_stride=512, kv_stride=128, qn=None, kn=None, eps=1e-6, cos=P, sin=P, len=10, rot=64, inter=0, cu=P,
             past=P, n=1, rows=3, **PAGES, nh=8, nkv=2, hd=64, qo=2 * P, qo_stride=512, stream=None)
    a.update(kw)
    return list(a.values())


def _read(**kw):
    a = dict(**PAGES, len=P, n=1, nkv=2, hd=64, type=0, k=P, v=P, slots=None, n_slots=2, kv_max=64, stream=None)
    a.update(kw)
    return list(a.values())


def _attend(**kw):
    a = dict(q=P, q_stride=512, **PAGES, cu=P, past=P, n=1, rows=3, max_kv=128, window=0, sinks=None, nh=8, nkv=2, hd=64, out=2 * P,
             out_stride=512, scratch=P, stream=None)
    a.update(kw)
    return list(a.values())


def _refused(tg, name, args, word):
    lib = tg.lib()
    lib.tg_hip_clear_error()
    getattr(lib, name)(*args)
    assert word in tg.last_error() and name in tg.last_error(), tg.last_error()
    lib.tg_hip_clear_error()


@pytest.mark.parametrize("kw,word", [
    (dict(len=-1), "rope_len"), (dict(len=(1 << 20) + 1), "rope_len"), (dict(first=-1), "first"), (dict(first=(1 << 30) + 1), "first"),
    (dict(rot=4), "rot_dim"), (dict(rot=60), "rot_dim"), (dict(rot=264), "rot_dim"), (dict(theta=1.0), "theta"),
    (dict(theta=math.nan), "theta"), (dict(theta=1e31), "theta"), (dict(scaling=6), "scaling"), (dict(scaling=-1), "scaling"),
    (dict(m=math.inf), "mscale"), (dict(m=math.nan), "mscale"), (dict(scaling=1, factor=0.0), "factor"),
    (dict(scaling=2, factor=math.nan), "factor"), (dict(scaling=3, low=1.0, high=32.0), "low"), (dict(scaling=5), "low"),
    (dict(scaling=4, orig=0), "orig_len"), (dict(scaling=3, high=0.0), "low"), (dict(cos=None), "null"), (dict(sin=P + 2), "4-byte")])
def test_tables_refuse(tg, kw, word):
    _refused(tg, "tg_hip_rope_tables_dev", _tables(**kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "n_rows"), (dict(nh=0), "n_heads"), (dict(nh=1025), "n_heads"), (dict(hd=60), "head_dim"), (dict(hd=1032), "head_dim"),
    (dict(rows=1 << 22, nh=1024, hd=128, x_stride=1 << 17, out_stride=1 << 17), "2^24"),
    (dict(x_stride=511), "stride"), (dict(out_stride=100), "stride"), (dict(out=P, out_stride=600), "stride"), (dict(x=None), "null"),
    (dict(out=P + 1), "4-byte"), (dict(pos=None), "null"), (dict(cos=None), "null"), (dict(sin=None), "tables"), (dict(rot=0), "rot_dim"),
    (dict(rot=72), "rot_dim"), (dict(rot=20), "rot_dim"), (dict(len=0), "rope_len")])
def test_rope_refuses(tg, kw, word):
    _refused(tg, "tg_hip_rope_dev", _rope(**kw), word)


PAGES_REFUSED = [
    (dict(size=8), "page_size"), (dict(size=2048), "page_size"), (dict(size=48), "page_size"), (dict(size=0), "page_size"),
    (dict(n_pages=0), "n_pages"), (dict(stride=0), "table_stride"), (dict(stride=1 << 27), "table_stride"), (dict(nkv=0), "n_kv_heads"),
    (dict(hd=40), "head_dim"), (dict(hd=144), "head_dim"), (dict(n=-1), "n_seqs"), (dict(n=1 << 17), "n_seqs"),
    (dict(n_pages=1 << 30), "too many"), (dict(n=1 << 16, nkv=32, nh=32), "too many"), (dict(pk=None), "null"), (dict(pv=P + 8), "16-byte"), (dict(ek=None), "null"),
    (dict(table=None), "null"), (dict(table=P + 2), "null")]


@pytest.mark.parametrize("kw,word", PAGES_REFUSED + [
    (dict(rows=-1), "n_rows"), (dict(rows=1 << 23), "n_rows"), (dict(nh=9), "integral"), (dict(nh=130, nkv=1), "integral"),
    (dict(rows=1 << 22, nh=64), "n_rows * n_heads"), (dict(cu=None), "cu_rows"), (dict(q=None), "q_out"), (dict(q_stride=8), "q_out"),
    (dict(qo_stride=8), "q_out"), (dict(qo=P, q_stride=600), "q_out"), (dict(kv_stride=127), "kv_stride"), (dict(cos=None), "tables"),
    (dict(rot=68), "rot_dim"), (dict(rot=12), "rot_dim"), (dict(len=0), "rope_len"), (dict(k=None), "null k"), (dict(v=P + 1), "4-byte")])
def test_append_refuses(tg, kw, word):
    _refused(tg, "tg_hip_paged_append_dev", _append(**kw), word)


@pytest.mark.parametrize("kw,word", [(k, w) for k, w in PAGES_REFUSED if "nh" not in k] + [
    (dict(type=2), "kv_type"), (dict(n_slots=0), "n_slots"), (dict(kv_max=0), "kv_max"), (dict(kv_max=1 << 21), "kv_max"),
    (dict(len=None), "null"), (dict(k=None), "null"), (dict(v=P + 4), "16-byte")])
def test_read_refuses(tg, kw, word):
    _refused(tg, "tg_hip_paged_read_dev", _read(**kw), word)


@pytest.mark.parametrize("kw,word", PAGES_REFUSED + [
    (dict(rows=-1), "n_rows"), (dict(nh=9), "integral"), (dict(cu=None), "cu_rows"), (dict(max_kv=0), "max_kv"),
    (dict(max_kv=129), "max_kv"), (dict(max_kv=(1 << 20) + 1, stride=1 << 17), "max_kv"), (dict(window=-1), "window"),
    (dict(q_stride=511), "stride"), (dict(out_stride=511), "stride"), (dict(q_stride=(1 << 21) + 1), "stride"), (dict(q=None), "null"),
    (dict(out=P + 2), "4-byte"), (dict(out=P, out_stride=600), "same stride"), (dict(scratch=None, max_kv=4096, stride=256), "scratch"),
    (dict(scratch=P + 8, max_kv=4096, stride=256), "scratch")])
def test_attention_refuses(tg, kw, word):
    _refused(tg, "tg_hip_attention_paged_dev", _attend(**kw), word)


def test_nothing_to_do(tg):
    lib = tg.lib()
    lib.tg_hip_clear_error()
    lib.tg_hip_rope_tables_dev(*_tables(len=0, cos=None, sin=None))
    lib.tg_hip_rope_dev(*_rope(rows=0, x=None, out=None))
    for kw in (dict(n=0), dict(rows=0), dict(n=0, rows=0, cu=None, k=None, v=None, q=None, qo=None, pk=None, table=None)):
        lib.tg_hip_paged_append_dev(*_append(**kw))
    lib.tg_hip_paged_read_dev(*_read(n=0, len=None, k=None, table=None))
    for kw in (dict(n=0), dict(rows=0), dict(n=0, rows=0, cu=None, pk=None, q=None, out=None, table=None)):
        lib.tg_hip_attention_paged_dev(*_attend(**kw))
    assert tg.last_error() == ""


def test_scratch_sizes(tg):
    f = tg.lib().tg_hip_attention_paged_scratch_bytes
    for bad in ((0, 1, 8, 2, 64, 64), (1, 0, 8, 2, 64, 64), (1, 1, 9, 2, 64, 64), (1, 1, 8, 2, 64, 0), (1, 1, 8, 2, 200, 64),
                (1 << 23, 1, 8, 2, 64, 64), (1, 1 << 17, 8, 2, 64, 64), (1, 1, 2048, 1024, 64, 64), (1, 1, 8, 2, 64, 1 << 21)):
        assert f(*bad) == 0
    assert f(1, 1, 8, 2, 64, 128) == 0      # one span
    assert 0 < f(1, 1, 8, 2, 64, 100000) <= f(100, 1, 8, 2, 64, 100000) <= f(100, 7, 8, 2, 64, 100000)


def draw_sizes(rng):
    nkv = int(rng.choice([1, 2, 3, 4, 8, 16]))
    nh = nkv * int(rng.choice([1, 2, 4, 5, 8, 16, 64]))
    return int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 9)), nh, nkv, int(rng.choice([16, 64, 80, 128])), int(2 ** rng.uniform(0, 18))


def smaller(rng, n):
    return int(rng.choice([n, max(1, n // 2), max(1, int(n ** rng.uniform(0, 1)))]))


def test_sizes_rise_with_every_argument(tg):
    size, rng = tg.lib().tg_hip_attention_paged_scratch_bytes, np.random.default_rng(1)
    for _ in range(20000):
        rows, n, nh, nkv, hd, kv = draw_sizes(rng)
        a, b, c = (smaller(rng, x) for x in (rows, n, kv))
        assert size(a, b, nh, nkv, hd, c) <= size(rows, n, nh, nkv, hd, kv), (rows, n, nh, nkv, hd, kv, a, b, c)


def test_scratch_serves_mixed_calls(tg):
    """Calls that always need scratch, so that they are refused and no device is asked: some many rows and some few behind long
    contexts."""
    lib, rng, seen = tg.lib(), np.random.default_rng(5), 0
    for _ in range(3000):
        nkv = int(rng.choice([1, 2, 4, 8]))
        nh = nkv * int(rng.choice([1, 2, 4, 8, 16]))
        hd, n, kv = int(rng.choice([16, 64, 80, 128])), int(rng.integers(2, 12)), int(rng.integers(8192, 100000))
        rows = int(rng.integers(600, 4000))
        size = lib.tg_hip_attention_paged_scratch_bytes(rows, n, nh, nkv, hd, kv)
        for a, b, c in ((rows, n, kv), (rows, smaller(rng, n), kv), (max(600, smaller(rng, rows)), n, max(8192, smaller(rng, kv)))):
            if (a * nh // nkv // 128 + b) * nkv > 1000 or a * nh // nkv < 600 or b < 2:
                continue
            lib.tg_hip_clear_error()
            lib.tg_hip_attention_paged_dev(*_attend(rows=a, n=b, max_kv=c, nh=nh, nkv=nkv, hd=hd, q_stride=nh * hd, out_stride=nh * hd,
                                                    stride=1 << 14, scratch=P + 4))
            said = tg.last_error()
            assert "needs" in said and int(said.split("needs ")[1].split()[0]) <= size, (rows, n, nh, nkv, hd, kv, a, b, c, said, size)
            seen += 1
    lib.tg_hip_clear_error()
    assert seen > 3000


def test_scratch_of_a_chunk_among_single_tokens(tg):
    """Single tokens have no tiles of 128 m-rows. Of 599 rows of 32 + 4 heads, 4,792 m-rows, at most 37 sequences have more than
    128, in at most 37 + 37 tiles; 128 spans a KV head may be added by cuts. Tiles of 16: 299 + 100, and 128. A record is
    16 bytes and a head; a tile's entry 16 bytes, at 37 + 100 places and 8 of each sequence; six roundings to 256."""
    lib = tg.lib()
    lib.tg_hip_clear_error()
    lib.tg_hip_attention_paged_dev(*_attend(rows=599, n=100, max_kv=9000, nh=32, nkv=4, hd=128, q_stride=4096, out_stride=4096, stride=1024,
                                            scratch=None))
    said = tg.last_error()
    lib.tg_hip_clear_error()
    most = 4 * (128 * (37 + 37 + 128) + 16 * (299 + 100 + 128)) * (16 + 4 * 128) + (37 + 100 + 800) * 16 + 6 * 256
    assert "needs" in said and int(said.split("needs ")[1].split()[0]) <= most, (said, most)


@pytest.mark.gpu
def test_scratch_serves_smaller_calls(tg):
    """Given scratch at an odd place a call says how much it needs; its rows are none, so one that needs nothing runs."""
    from tests._packed import Dev
    print("scratch of smaller paged calls", flush=True)
    lib, rng, dev, seen = tg.lib(), np.random.default_rng(3), Dev(tg), 0
    zeros = dev(np.zeros(1 << 16, np.float32))
    for _ in range(4000):
        rows, n, nh, nkv, hd, kv = draw_sizes(rng)
        most = lib.tg_hip_attention_paged_scratch_bytes(rows, n, nh, nkv, hd, kv)
        a, b, c = (smaller(rng, x) for x in (rows, n, kv))
        z = dict(q=zeros, pk=zeros, pv=zeros, ek=zeros, ev=zeros, table=zeros, cu=zeros, past=zeros, out=zeros, scratch=zeros + 4)
        lib.tg_hip_clear_error()
        lib.tg_hip_attention_paged_dev(*_attend(**z, rows=a, n=b, max_kv=c, window=int(rng.choice([0, int(2 ** rng.uniform(0, 18))])), nh=nh,
                                                nkv=nkv, hd=hd, q_stride=nh * hd, out_stride=nh * hd, n_pages=1, stride=1 << 14))
        said = tg.last_error()
        if said:
            seen += 1
            assert int(said.split("needs ")[1].split()[0]) <= most, (rows, n, nh, nkv, hd, kv, a, b, c, said)
    lib.tg_hip_clear_error()
    lib.tg_hip_synchronize()
    dev.free()
    assert seen > 500


def test_names(tg):
    assert (tg.ROPE_PLAIN, tg.ROPE_LINEAR, tg.ROPE_BASE, tg.ROPE_PARTS, tg.ROPE_PARTS_WHOLE, tg.ROPE_SMOOTH) == tuple(range(6))
