"""The operators of the prompt and batch path, measured: rows appended to the caches, attention of packed sequences
over them, attention behind a shared prefix, and the adjustments of logits before a token is chosen.

  append   tg_hip_kv_append_dev: QK norm, RoPE and the K/V stores of packed rows
  prompt   tg_hip_attention_prompt_dev: causal grouped attention of packed sequences over their cache slots
  prefix   tg_hip_attention_prefix_dev: the same for a batch whose sequences share a prefix that is held once
  logits   tg_hip_logits_adjust_dev: penalties, biases and a grammar's mask, with the argmax of the result

Head layouts are those of the two models the package names (Qwen3-30B-A3B: 32 query and 4 KV heads of 128, QK norm;
gpt-oss-120b: 64 and 8 of 64, sinks, every other layer with a window of 128) and, among the drawn cases, others.
The library runs on a stream of its own; whoever times or reads waits for the device.
"""

import math

import numpy as np
import torch

own = False

LAYOUTS = {   # query heads, KV heads, head size, QK norm, sinks
    "qwen3": (32, 4, 128, True, False),
    "gptoss": (64, 8, 64, False, True),
    "even": (8, 8, 96, False, False),     # a KV head for every query head
    "odd": (15, 3, 80, True, True),       # groups and sizes that fill no tile
    "wide": (28, 2, 112, False, False),   # many query heads on a KV head
    "small": (6, 2, 32, False, True),
}
VOCAB = 151936
EPS = 1e-6


# ------------------------------------------------------------------ the cases
# lens and past: each sequence's rows in the call and its positions cached before them, in words

def listed():
    return [
        # eight conversations decode a token each: the smallest call, latency
        dict(name="append decode batch", kind="append", layout="qwen3", lens="1 " * 8, past="700 " * 8, half=True),
        # a long prompt enters an f32 cache
        dict(name="append gptoss prompt", kind="append", layout="gptoss", lens="4001", past="0", half=False),
        # requests of very different lengths, packed into one pass, over the cache that decode attention reads
        dict(name="prompt qwen3 packed", kind="prompt", layout="qwen3", lens="1 17 300 509 64 1000 129", past="0 " * 7,
             half=False, window=0),
        # one long document
        dict(name="prompt qwen3 long", kind="prompt", layout="qwen3", lens="8192", past="0", half=True, window=0),
        # the same of the other model: a sliding layer, then a chunk of a prompt deep in a full layer
        dict(name="prompt gptoss window", kind="prompt", layout="gptoss", lens="4096", past="0", half=True, window=128),
        dict(name="prompt gptoss chunk", kind="prompt", layout="gptoss", lens="500", past="30001", half=False, window=0),
        # the verify pass of eight drafts in a conversation of a few thousand tokens
        dict(name="prompt qwen3 verify", kind="prompt", layout="qwen3", lens="9", past="4000", half=False, window=0),
        # a token of each of many conversations
        dict(name="prompt qwen3 decode batch", kind="prompt", layout="qwen3", lens="1 " * 32,
             past=" ".join(str(61 + 131 * i) for i in range(32)), half=True, window=0),
        # many samples of one long prompt, and a few answers behind a short one
        dict(name="prefix qwen3 samples", kind="prefix", layout="qwen3", prefix=8000, lens="1 " * 48,
             past=" ".join(str(37 * i % 500) for i in range(48)), half=True, window=0),
        dict(name="prefix gptoss few", kind="prefix", layout="gptoss", prefix=1500, lens="1 1 1 1 1", past="3 40 0 77 12",
             half=False, window=0),
        # the next token of one conversation with a repetition penalty; a batch under grammars
        dict(name="logits one row", kind="logits", vocab=VOCAB, k=1, hist=700, bias=0, mask=False),
        dict(name="logits batch", kind="logits", vocab=VOCAB, k=64, hist=4000, bias=300, mask=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _words(v):
    return " ".join(map(str, v))


def draw(rng):
    kind = rng.choice(["append", "prompt", "prompt", "prompt", "prompt", "prefix", "prefix", "logits"])
    layout = rng.choice(["qwen3", "qwen3", "gptoss", "gptoss", "even", "odd", "wide", "small"])
    half, window = rng.random() < 0.5, rng.choice([0, 0, 128, _log_int(rng, 1, 4000)])
    if kind == "logits":
        return dict(kind=kind, vocab=rng.choice([VOCAB, _log_int(rng, 1000, VOCAB)]), k=_log_int(rng, 1, 64),
                    hist=_log_int(rng, 1, 16000), bias=rng.choice([0, _log_int(rng, 1, 1000)]), mask=rng.random() < 0.6)
    if kind == "prefix":
        n = _log_int(rng, 1, 64)
        return dict(kind=kind, layout=layout, prefix=_log_int(rng, 1, 8000), lens=_words([rng.choice([1, 1, 1, rng.randint(0, 9)]) for _ in range(n - 1)] + [1]),
                    past=_words(rng.randint(0, 400) for _ in range(n)), half=half, window=window)
    if kind == "append":
        n = _log_int(rng, 1, 16)
        return dict(kind=kind, layout=layout, lens=_words(_log_int(rng, 1, 4000 // n) for _ in range(n)),
                    past=_words(rng.choice([0, _log_int(rng, 1, 4000)]) for _ in range(n)), half=half)
    way = rng.choice(["whole", "whole", "chunk", "decode"])
    if way == "whole":
        n = rng.choice([1, _log_int(rng, 2, 12)])
        lens, past = [_log_int(rng, 1, 5000 // n) for _ in range(n)], [0] * n
    elif way == "chunk":
        n = rng.choice([1, 1, 3])
        lens, past = [_log_int(rng, 2, 500) for _ in range(n)], [_log_int(rng, 1, 30000 // n) for _ in range(n)]
    else:
        n = _log_int(rng, 1, 48)
        lens, past = [1] * n, [_log_int(rng, 1, 8000) for _ in range(n)]
    return dict(kind="prompt", layout=layout, lens=_words(lens), past=_words(past), half=half, window=window)


# ------------------------------------------------------------------ inputs

class State:
    pass


def _lens(case):
    return [int(w) for w in case["lens"].split()], [int(w) for w in case["past"].split()]


def _ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    s = State()
    s.kind, s.scratch = case["kind"], None
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if s.kind == "logits":
        _prepare_logits(s, case, g)
    else:
        _prepare_rows(s, case, g)
    torch.cuda.synchronize()   # the library's stream reads what torch's wrote
    return s


def _prepare_rows(s, case, g):
    normal = lambda *shape, scale=1.0: torch.randn(*shape, generator=g, device="cuda") * scale   # noqa: E731
    s.nh, s.nkv, s.hd, norm, sinks = LAYOUTS[case["layout"]]
    lens, past = _lens(case)
    s.n, s.rows, s.most = len(lens), sum(lens), max(lens)
    s.total = max(a + b for a, b in zip(lens, past))             # the longest sequence
    s.kv_max = 256 * (s.total // 256 + 1)
    s.cu, s.kv_len = _ints(np.concatenate([[0], np.cumsum(lens)])), _ints(past)
    s.slots = _ints(reversed(range(s.n)))                        # any order of the cache's slots
    s.kv_type, dtype = (1, torch.float16) if case["half"] else (0, torch.float32)
    s.cache = [torch.empty(s.n, s.nkv, s.kv_max, s.hd, device="cuda", dtype=dtype) for _ in range(2)]
    for t in s.cache:   # stale rows of earlier sequences behind the live ones
        t.copy_(normal(s.n, s.nkv, s.kv_max, s.hd))
    s.prefix = case.get("prefix", 0)
    s.window = case.get("window", 0)
    s.sinks = normal(s.nh) if sinks else None
    if s.kind == "append":
        s.base, top = 0, s.total
        s.qkv = normal(s.rows, (s.nh + 2 * s.nkv) * s.hd, scale=1.5)   # the projections, side by side
        s.norms = [torch.empty(s.hd, device="cuda").uniform_(0.5, 1.5, generator=g) for _ in range(2)] if norm else [None] * 2
        angle = torch.arange(top, device="cuda")[:, None].double() / 1e6 ** (torch.arange(s.hd // 2, device="cuda").double() / (s.hd // 2))
        s.cos, s.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        s.out = torch.empty(s.rows, s.nh * s.hd, device="cuda")
        return
    s.q = normal(s.rows, s.nh * s.hd, scale=2.0)                 # scores of a trained model's spread
    s.out = torch.zeros(s.rows, s.nh * s.hd, device="cuda")
    if s.kind == "prefix":
        s.common = [normal(s.nkv, s.prefix, s.hd).to(dtype) for _ in range(2)]


def _prepare_logits(s, case, g):
    k, s.vocab, n = case["k"], case["vocab"], case["hist"]
    s.k = k
    s.logits = torch.randn(k, s.vocab, generator=g, device="cuda") * 3
    # a history's tokens repeat: low ranks of a permutation more often
    u = torch.rand(k, n, generator=g, device="cuda")
    rank = ((s.vocab ** u - 1) / (s.vocab - 1) * s.vocab).long().clamp(0, s.vocab - 1)
    s.hist = ((rank * 7919 + 13) % s.vocab).int()
    s.hist_len = (n - torch.randint(0, n // 2 + 1, (k,), generator=g, device="cuda")).int()
    s.gen_start = (s.hist_len.float() * torch.rand(k, generator=g, device="cuda")).int()   # the prompt's part
    s.pen = torch.stack([1 + torch.rand(k, generator=g, device="cuda") * 0.5, torch.rand(k, generator=g, device="cuda"),
                         torch.rand(k, generator=g, device="cuda")], 1).contiguous()
    s.nb = case["bias"]
    s.bias_tok = s.bias_val = s.bias_len = s.allow = None
    if s.nb:
        s.bias_tok = torch.randint(0, s.vocab, (k, s.nb), generator=g, device="cuda", dtype=torch.int32)
        s.bias_tok[:, s.nb // 2:] = s.bias_tok[:, :s.nb - s.nb // 2].flip(1)   # some are listed again: the last holds
        s.bias_val = torch.randn(k, s.nb, generator=g, device="cuda") * 4
        s.bias_len = torch.full((k,), s.nb, device="cuda", dtype=torch.int32)
    s.words = (s.vocab + 31) // 32
    if case["mask"]:
        a, b = (torch.randint(-2 ** 31, 2 ** 31, (k, s.words), generator=g, device="cuda", dtype=torch.int32) for _ in range(2))
        s.allow = a & b
        s.allow[0] = 0 if k > 2 else s.allow[0]   # a grammar that has ended
    s.out = torch.empty_like(s.logits)
    s.arg = torch.empty(k, dtype=torch.int32, device="cuda")
    s.top = torch.empty(k, device="cuda")


# ------------------------------------------------------------------ one pass

def _ptr(t):
    return None if t is None else t.data_ptr()


def run(s):
    if own:
        return _run_own(s)
    if s.kind == "append":
        return _plain_append(s)
    if s.kind == "logits":
        return _plain_logits(s)
    return _plain_attention(s)


def _workspace(s, lib):
    """The call's scratch, which a program allocates once."""
    if s.kind == "logits":
        need = lib.tg_hip_logits_scratch_bytes(s.k, s.vocab)
    else:
        need = lib.tg_hip_attention_prompt_scratch_bytes(s.rows, s.n, s.nh, s.nkv, s.hd, s.kv_max, s.prefix)
    return torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)


def _run_own(s):
    import tinygiant_amd as tg
    lib = tg.lib()
    if s.scratch is None:
        s.scratch = _workspace(s, lib)
    if s.kind == "append":
        p, qd, kd, st = s.qkv.data_ptr(), s.nh * s.hd, s.nkv * s.hd, (s.nh + 2 * s.nkv) * s.hd
        lib.tg_hip_kv_append_dev(p, p + 4 * qd, p + 4 * (qd + kd), st, st, _ptr(s.norms[0]), _ptr(s.norms[1]), EPS,
                                 s.cos.data_ptr(), s.sin.data_ptr(), len(s.cos), s.cu.data_ptr(), s.kv_len.data_ptr(),
                                 s.slots.data_ptr(), s.n, s.rows, s.base, s.kv_type, s.cache[0].data_ptr(),
                                 s.cache[1].data_ptr(), s.n, s.kv_max, s.nh, s.nkv, s.hd, s.out.data_ptr(), qd, None)
        return dict(q=s.out, k=s.cache[0], v=s.cache[1])
    if s.kind == "logits":
        lib.tg_hip_logits_adjust_dev(s.logits.data_ptr(), s.out.data_ptr(), s.k, s.vocab, s.hist.data_ptr(), s.hist.shape[1],
                                     s.hist_len.data_ptr(), s.gen_start.data_ptr(), s.pen.data_ptr(), _ptr(s.bias_tok),
                                     _ptr(s.bias_val), s.nb, _ptr(s.bias_len), _ptr(s.allow), s.words, s.arg.data_ptr(),
                                     s.top.data_ptr(), s.scratch.data_ptr(), None)
        return dict(logits=s.out, argmax=s.arg, maxval=s.top)
    qd = s.nh * s.hd
    rows = (s.q.data_ptr(), qd, s.kv_type, s.cache[0].data_ptr(), s.cache[1].data_ptr(), s.n, s.kv_max)
    seqs = (s.cu.data_ptr(), s.kv_len.data_ptr(), s.slots.data_ptr(), s.n, s.rows, s.window, _ptr(s.sinks), s.nh, s.nkv, s.hd,
            s.out.data_ptr(), qd, s.scratch.data_ptr(), None)
    if s.kind == "prefix":
        lib.tg_hip_attention_prefix_dev(*rows, s.common[0].data_ptr(), s.common[1].data_ptr(), s.prefix, s.prefix, *seqs)
    else:
        lib.tg_hip_attention_prompt_dev(*rows, *seqs)
    return s.out


def _places(s):
    """Of every packed row: its sequence, and its place in it."""
    r = torch.arange(s.rows, device="cuda")
    seq = (r[:, None] >= s.cu[None, 1:]).sum(1)
    return seq, r - s.cu[seq]


def _norm(x, w):
    return x if w is None else x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w


def _turn(x, c, sn):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _plain_append(s):
    seq, i = _places(s)
    at = s.kv_len[seq] + i
    q, k, v = s.qkv.view(s.rows, -1, s.hd).split([s.nh, s.nkv, s.nkv], 1)
    c, sn = s.cos[s.base + at][:, None], s.sin[s.base + at][:, None]
    q, k = _turn(_norm(q, s.norms[0]), c, sn), _turn(_norm(k, s.norms[1]), c, sn)
    for cache, new in zip(s.cache, (k, v)):
        cache[s.slots[seq].long(), :, at.long()] = new.to(cache.dtype)
    return dict(q=q.reshape(s.rows, -1), k=s.cache[0], v=s.cache[1])


def _plain_attention(s):
    """Sequences padded to the longest, scores of all heads at once."""
    seq, i = _places(s)
    group, scale = s.nh // s.nkv, s.hd ** -0.5
    q = torch.zeros(s.n, s.nkv, group, s.most, s.hd, device="cuda")
    q[seq, :, :, i] = s.q.view(s.rows, s.nkv, group, s.hd)
    keys, vals = (t[s.slots.long(), :, :s.total].float() for t in s.cache)
    z = torch.matmul(q.view(s.n, s.nkv, -1, s.hd), keys.transpose(2, 3).contiguous()).view(s.n, s.nkv, group, s.most, s.total)
    place = torch.arange(s.most, device="cuda")[None, :, None] + s.kv_len[:, None, None]   # of a row, in its own cache
    key = torch.arange(s.total, device="cuda")
    see = key <= place
    if s.window:
        see = see & (key > place - s.window)
    if s.prefix:
        first_k, first_v = (t.float() for t in s.common)
        y = torch.matmul(q.view(s.n, s.nkv, -1, s.hd), first_k.transpose(1, 2).contiguous()[None])
        key = torch.arange(s.prefix, device="cuda")
        saw = (key > place + s.prefix - s.window) if s.window else (key >= 0).expand(s.n, s.most, s.prefix)
        z = torch.cat([y.view(s.n, s.nkv, group, s.most, s.prefix), z], -1)
        see = torch.cat([saw, see], -1)
    z.mul_(scale).masked_fill_(~see[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    if s.sinks is not None:
        sink = s.sinks.view(1, s.nkv, group, 1, 1)
        m = torch.maximum(m, sink)
    p = z.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + (sink - m).exp()
    p = p.view(s.n, s.nkv, group * s.most, -1)
    o = torch.matmul(p[..., s.prefix:].contiguous() if s.prefix else p, vals)
    if s.prefix:
        o = o + torch.matmul(p[..., :s.prefix].contiguous(), first_v[None])
    o = o.view(s.n, s.nkv, group, s.most, s.hd) / total
    return o[seq, :, :, i].reshape(s.rows, -1)


def _plain_logits(s):
    n, token = s.hist.shape[1], torch.arange(s.vocab, device="cuda")
    at = torch.arange(n, device="cuda")
    live = at < s.hist_len[:, None]
    made = (live & (at >= s.gen_start[:, None])).float()
    seen, count = (torch.zeros(s.k, s.vocab, device="cuda").scatter_add_(1, s.hist.long(), x) for x in (live.float(), made))
    rep, freq, pres = s.pen[:, :1], s.pen[:, 1:2], s.pen[:, 2:]
    l = torch.where(seen > 0, torch.where(s.logits > 0, s.logits / rep, s.logits * rep), s.logits)
    l = torch.where(count > 0, l - freq * count - pres, l)
    if s.nb:
        order = torch.arange(1, s.nb + 1, device="cuda").expand(s.k, -1)
        order = torch.where(order <= s.bias_len[:, None], order, 0)
        last = torch.zeros(s.k, s.vocab, dtype=torch.long, device="cuda").scatter_reduce_(1, s.bias_tok.long(), order, "amax")
        l = torch.where(last > 0, l + s.bias_val.gather(1, (last - 1).clamp(min=0)), l)
    if s.allow is not None:
        bit = (s.allow[:, token >> 5] >> (token & 31).int()) & 1
        l = torch.where(bit == 1, l, -math.inf)
    m = l.amax(1)
    first = torch.where(l == m[:, None], token, s.vocab).amin(1)
    return dict(logits=l, argmax=torch.where(m == -math.inf, -1, first).int(), maxval=m)


# ------------------------------------------------------------------ the work of a pass

def work(case):
    if case["kind"] == "logits":
        k, v = case["k"], case["vocab"]
        return dict(bytes=k * (8 * v + 4 * case["hist"] + 8 * case["bias"] + (v // 8 if case["mask"] else 0)), flops=4 * k * v)
    nh, nkv, hd, _, _ = LAYOUTS[case["layout"]]
    lens, past = _lens(case)
    size, rows, window, prefix = 2 if case["half"] else 4, sum(lens), case.get("window", 0), case.get("prefix", 0)
    if case["kind"] == "append":
        return dict(bytes=rows * hd * (8 * nh + 2 * nkv * (4 + size) + 4), flops=rows * hd * (nh + nkv) * 8)
    pairs, seen, first = 0, 0, prefix
    for n, p in zip(lens, past):
        ends = np.arange(n) + p + 1 + prefix                      # positions that each row could see
        pairs += int(np.minimum(ends, window).sum() if window else ends.sum())
        if n:
            low = max(0, p + prefix + 1 - window) if window else 0   # the first position that any of its rows sees
            seen += n + p - max(0, low - prefix)
            first = min(first, low)
    seen += prefix - first
    return dict(bytes=2 * nkv * hd * size * seen + 8 * rows * nh * hd, flops=4 * nh * hd * pairs)


# ------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "logits":
        return _exact_logits(s)
    lens, past = _lens(case)
    if s.kind == "append":
        return _exact_append(s, lens, past)
    group, out, r = s.nh // s.nkv, [], 0
    heads = s.q.double().view(s.rows, s.nkv, group, s.hd)
    for b, (n, p) in enumerate(zip(lens, past)):
        slot, ends = s.n - 1 - b, torch.arange(p, p + n, device="cuda") + s.prefix   # the last position a row sees
        mine = torch.empty(n, s.nkv, group, s.hd, device="cuda", dtype=torch.float64)
        for h in range(s.nkv if n else 0):
            keys, vals = (t[slot, h, :p + n].double() for t in s.cache)
            if s.prefix:
                keys, vals = (torch.cat([c[h].double(), t]) for c, t in zip(s.common, (keys, vals)))
            where = torch.arange(len(keys), device="cuda")
            hide = where[None] > ends[:, None]
            if s.window:
                hide |= where[None] <= ends[:, None] - s.window
            for j in range(group):
                z = heads[r:r + n, h, j] @ keys.T / math.sqrt(s.hd)
                z[hide] = -math.inf
                top = z.max(1, keepdim=True).values
                extra = 0
                if s.sinks is not None:
                    sink = s.sinks[h * group + j].double()
                    top = torch.clamp(top, min=sink)
                    extra = torch.exp(sink - top)
                w = torch.exp(z - top)
                mine[:, h, j] = (w @ vals) / (w.sum(1, keepdim=True) + extra)
        out.append(mine.view(n, -1))
        r += n
    return torch.cat(out)


def _exact_append(s, lens, past):
    x = s.qkv.double().view(s.rows, -1, s.hd)
    k, v = (t.double() for t in s.cache)
    q_out, r, half = [], 0, s.hd // 2
    for b, (n, p) in enumerate(zip(lens, past)):
        y = x[r:r + n].clone()
        for part, w in ((slice(0, s.nh), s.norms[0]), (slice(s.nh, s.nh + s.nkv), s.norms[1])):
            if w is not None:
                y[:, part] *= w.double() / torch.sqrt(y[:, part].pow(2).sum(-1, keepdim=True) / s.hd + EPS)
        c, sn = (t[p:p + n].double()[:, None] for t in (s.cos, s.sin))
        a, d = y[..., :half].clone(), y[..., half:].clone()
        turned = torch.cat([a * c - d * sn, d * c + a * sn], -1)
        q_out.append(turned[:, :s.nh].reshape(n, -1))
        k[s.n - 1 - b, :, p:p + n] = turned[:, s.nh:s.nh + s.nkv].transpose(0, 1)
        v[s.n - 1 - b, :, p:p + n] = y[:, s.nh + s.nkv:].transpose(0, 1)
        r += n
    return dict(q=torch.cat(q_out), k=k, v=v)


def _exact_logits(s):
    """Row by row from the lists; which index is largest may hang on a 32-bit rounding, so it has no value here."""
    rows = []
    for j in range(s.k):
        l = s.logits[j].double().cpu().numpy()
        rep, freq, pres = (float(x) for x in s.pen[j])
        seen = s.hist[j, :int(s.hist_len[j])].cpu().numpy()
        t = np.unique(seen)
        l[t] = np.where(l[t] > 0, l[t] / rep, l[t] * rep)
        t, c = np.unique(seen[int(s.gen_start[j]):], return_counts=True)
        l[t] -= freq * c + pres
        if s.nb:
            held = dict(zip(s.bias_tok[j].tolist(), s.bias_val[j].tolist()))   # a later entry replaces an earlier one
            l[list(held)] += np.array(list(held.values()))
        if s.allow is not None:
            bits = np.unpackbits(s.allow[j].cpu().numpy().view(np.uint8), bitorder="little")[:s.vocab]
            l[bits == 0] = -np.inf
        rows.append(l)
    l = torch.from_numpy(np.stack(rows)).cuda()
    return dict(logits=l, argmax=None, maxval=l.max(1).values)
