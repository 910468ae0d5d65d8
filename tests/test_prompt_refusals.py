"""Arguments that the prompt and batch path refuses, and calls with nothing to
do: both return before any device work, so they run without a GPU."""

import numpy as np
import pytest

P = 1 << 20   # stands for a device pointer that must not be followed


def _attention(**kw):
    a = dict(q=P, q_stride=512, kv_type=0, k=P, v=P, n_slots=2, kv_max=64, cu=P, len=P, slots=P, n_seqs=1, n_rows=3, window=0,
             sinks=None, nh=8, nkv=2, hd=64, out=2 * P, out_stride=512, scratch=P, stream=None)
    pre = dict(pk=P, pv=P, plen=10, pmax=20)
    prefix = any(x in kw for x in pre)
    for x, y in kw.items():
        (pre if x in pre else a)[x] = y
    v = list(a.values())
    return prefix, v[:7] + (list(pre.values()) if prefix else []) + v[7:]


def _append(**kw):
    a = dict(q=P, k=P, v=P, q_stride=512, kv_stride=128, qn=None, kn=None, eps=1e-6, cos=P, sin=P, rope_len=10, cu=P, len=P,
             slots=P, n_seqs=1, n_rows=3, base=0, kv_type=0, kk=P, kv=P, n_slots=2, kv_max=64, nh=8, nkv=2, hd=64, qo=P,
             qo_stride=512, stream=None)
    a.update(kw)
    return list(a.values())


def _logits(**kw):
    a = dict(logits=P, out=P, k=2, nrows=100, hist=P, hist_stride=5, hist_len=P, start=None, pen=P, btok=P, bval=P, bstride=3,
             blen=None, allow=P, allow_stride=4, arg=P, top=P, scratch=P, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,word", [
    (dict(kv_type=2), "kv_type"), (dict(kv_type=-1), "kv_type"), (dict(n_seqs=-1), "n_seqs"), (dict(n_rows=-5), "n_rows"),
    (dict(n_rows=1 << 23), "n_rows"), (dict(n_slots=0), "n_slots"), (dict(kv_max=0), "kv_max"), (dict(kv_max=(1 << 20) + 1), "kv_max"),
    (dict(hd=60), "shape"), (dict(hd=0), "shape"), (dict(hd=136), "shape"), (dict(nh=9), "shape"), (dict(nkv=0), "shape"),
    (dict(nh=130, nkv=1), "shape"), (dict(nh=2048, nkv=1024), "shape"), (dict(cu=None), "cu_rows"), (dict(k=None), "cache"),
    (dict(v=P + 4), "16-byte"), (dict(window=-1), "window"), (dict(q_stride=511), "stride"), (dict(out_stride=100), "stride"), (dict(q_stride=(1 << 21) + 1), "stride"),
    (dict(q=None), "q or out"), (dict(out=None), "q or out"), (dict(q=P + 2), "q or out"),
    (dict(out=P, out_stride=600), "same stride"), (dict(plen=21), "prefix_len"), (dict(plen=-1), "prefix_len"),
    (dict(n_rows=1 << 22, nh=64, nkv=8, q_stride=4096, out_stride=4096), "too many"), (dict(n_seqs=1 << 16, nkv=32, nh=32), "too many"),
    (dict(pk=None), "prefix_k"), (dict(pv=P + 8), "prefix_k"), (dict(pmax=1 << 21), "prefix_len")])
def test_attention_refuses(tg, kw, word):
    lib = tg.lib()
    prefix, args = _attention(**kw)
    lib.tg_hip_clear_error()
    (lib.tg_hip_attention_prefix_dev if prefix else lib.tg_hip_attention_prompt_dev)(*args)
    assert word in tg.last_error() and "tg_hip_attention_pr" in tg.last_error()
    lib.tg_hip_clear_error()


@pytest.mark.parametrize("kw,word", [
    (dict(kv_type=7), "kv_type"), (dict(hd=12), "shape"), (dict(kk=P + 2), "16-byte"), (dict(cu=None), "cu_rows"),
    (dict(q=None), "q_out"), (dict(q_stride=8), "q_out"), (dict(qo_stride=8), "q_out"), (dict(qo=P, q_stride=600), "same stride"),
    (dict(kv_stride=127), "kv_stride"), (dict(base=-1), "base_pos"), (dict(cos=None), "tables"), (dict(sin=None), "tables"),
    (dict(rope_len=0), "tables"), (dict(k=None), "null k"), (dict(v=None), "null k"), (dict(k=P + 1), "4-byte")])
def test_append_refuses(tg, kw, word):
    lib = tg.lib()
    lib.tg_hip_clear_error()
    lib.tg_hip_kv_append_dev(*_append(**kw))
    assert word in tg.last_error() and "tg_hip_kv_append_dev" in tg.last_error()
    lib.tg_hip_clear_error()


@pytest.mark.parametrize("kw,word", [
    (dict(k=-1), "k <="), (dict(k=70000), "k <="), (dict(nrows=0), "nrows"), (dict(nrows=(1 << 24) + 1), "nrows"),
    (dict(hist_stride=-1), "strides"), (dict(bstride=-1), "strides"), (dict(logits=None), "null logits"),
    (dict(out=None, arg=None, top=None), "no output"), (dict(scratch=None), "scratch"), (dict(scratch=P + 4), "scratch"),
    (dict(hist_len=None), "history"), (dict(pen=None), "history"), (dict(bval=None), "bias"), (dict(btok=None), "bias"),
    (dict(allow_stride=3), "allow_stride"), (dict(allow_stride=-4), "allow_stride"),
    (dict(logits=P + 2), "4-byte"), (dict(out=P + 1), "4-byte"), (dict(hist=P + 2), "4-byte")])
def test_logits_refuses(tg, kw, word):
    lib = tg.lib()
    lib.tg_hip_clear_error()
    lib.tg_hip_logits_adjust_dev(*_logits(**kw))
    assert word in tg.last_error() and "tg_hip_logits_adjust_dev" in tg.last_error()
    lib.tg_hip_clear_error()


def test_nothing_to_do(tg):
    lib = tg.lib()
    lib.tg_hip_clear_error()
    for kw in (dict(n_seqs=0), dict(n_rows=0), dict(n_seqs=0, n_rows=0, cu=None, k=None, v=None, q=None, out=None)):
        lib.tg_hip_attention_prompt_dev(*_attention(**kw)[1])
    lib.tg_hip_attention_prefix_dev(*_attention(n_rows=0, plen=3)[1])
    for kw in (dict(n_seqs=0), dict(n_rows=0)):
        lib.tg_hip_kv_append_dev(*_append(**kw))
    lib.tg_hip_logits_adjust_dev(*_logits(k=0))
    assert tg.last_error() == ""


def test_scratch_sizes(tg):
    lib = tg.lib()
    assert lib.tg_hip_logits_scratch_bytes(0, 5) == 0 and lib.tg_hip_logits_scratch_bytes(5, 0) == 0
    assert lib.tg_hip_logits_scratch_bytes(1, 1) >= 8
    for bad in ((0, 1, 8, 2, 64, 64, 0), (1, 0, 8, 2, 64, 64, 0), (1, 1, 9, 2, 64, 64, 0), (1, 1, 8, 2, 64, 0, 0),
                (1, 1, 8, 2, 200, 64, 0), (1, 1, 8, 2, 64, 64, -1), (1 << 23, 1, 8, 2, 64, 64, 0),
                (1, 1 << 17, 8, 2, 64, 64, 0), (1, 1, 2048, 1024, 64, 64, 0), (1, 1, 8, 2, 64, 1 << 21, 0)):
        assert lib.tg_hip_attention_prompt_scratch_bytes(*bad) == 0


def test_kv_codes(tg):
    assert (tg.KV_F32, tg.KV_F16) == (0, 1)
    assert np.dtype(np.float16).itemsize == 2
