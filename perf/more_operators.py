"""The operators of paged 8-bit caches and of rotary positions, measured.

  tables   tg_hip_rope_tables_dev: cosines and sines of positions, frequencies scaled for long contexts
  rope     tg_hip_rope_dev: rows rotated, half or interleaved pairs, part of the head
  append   tg_hip_paged_append_dev: QK norm, rotation, and K/V of packed rows into 8-bit pages
  read     tg_hip_paged_read_dev: positions of paged sequences as values, in dense cache slots
  attend   tg_hip_attention_paged_dev: causal grouped attention of packed sequences over their pages

Pages hold `page` positions of every KV head as signed bytes, [n_pages][KV heads][page][head size]; a block of 16 positions
of a head has one power of two, held as a byte b for 2^(b - 127). A sequence's pages are those of its row of a table,
in order. Head layouts are those of the two models the package names (Qwen3-30B-A3B: 32 query and 4 KV heads of 128, QK
norm; gpt-oss-120b: 64 and 8 of 64, sinks, every other layer with a window of 128, positions scaled by parts) and, among
the drawn cases, others. The library runs on a stream of its own; whoever times or reads waits for the device.
"""

import math

import numpy as np
import torch

own = False

LAYOUTS = {   # query heads, KV heads, head size, rotated part, QK norm, sinks
    "qwen3": (32, 4, 128, 128, True, False),
    "gptoss": (64, 8, 64, 64, False, True),
    "even": (8, 8, 96, 96, False, False),     # a KV head for every query head
    "odd": (15, 3, 80, 40, True, True),       # groups and sizes that fill no tile, half of the head rotated
    "wide": (28, 2, 112, 64, False, False),   # many query heads on a KV head
    "small": (6, 2, 32, 32, False, True),
}
EPS = 1e-6
BLOCK = 16                 # positions that share a power of two
LEAST, MOST = -42, 42      # its exponents
SCALINGS = ["plain", "linear", "base", "parts", "parts whole", "smooth"]   # in the order of the library's numbers


# ------------------------------------------------------------------ the cases
# lens and past: each sequence's rows in the call and its positions cached before them, in words

def listed():
    return [
        # the tables of a chat's context, when a program starts
        dict(name="tables short", kind="tables", first=0, len=4096, rot=128, scaling="plain", factor=1.0),
        # those of gpt-oss at its full context
        dict(name="tables long by parts", kind="tables", first=0, len=131072, rot=64, scaling="parts", factor=32.0),
        # a token of each of eight conversations, in front of an append that does not rotate
        dict(name="rope decode batch", kind="rope", layout="qwen3", rows=8, far=4000, interleaved=False),
        # a prompt of a model with interleaved pairs on half of its head
        dict(name="rope interleaved prompt", kind="rope", layout="odd", rows=4001, far=4001, interleaved=True),
        # 32 conversations decode a token each into 8-bit pages
        dict(name="append decode batch", kind="append", layout="qwen3", lens="1 " * 32,
             past=" ".join(str(61 + 131 * i) for i in range(32)), page=64, interleaved=False),
        # a long prompt enters the cache
        dict(name="append gptoss prompt", kind="append", layout="gptoss", lens="4001", past="0", page=64, interleaved=False),
        # a conversation leaves its pages for a slot
        dict(name="read one", kind="read", layout="qwen3", lens="700", page=16, half=False),
        # a batch moves from pages to f16 slots
        dict(name="read batch", kind="read", layout="gptoss", lens="4001 17 9000 2500", page=256, half=True),
        # the next token of one long conversation
        dict(name="attend one deep", kind="attend", layout="gptoss", lens="1", past="30001", page=64, window=0),
        # a token of each of many conversations
        dict(name="attend decode batch", kind="attend", layout="qwen3", lens="1 " * 64,
             past=" ".join(str(61 + 131 * i) for i in range(64)), page=64, window=0),
        # requests of very different lengths in one pass: whole prompts, chunks, a verify pass, single tokens
        dict(name="attend mixed", kind="attend", layout="qwen3", lens="1 17 300 9 1000 1 129", past="900 0 512 4000 0 2500 77",
             page=16, window=0),
        # one long document
        dict(name="attend long", kind="attend", layout="qwen3", lens="8192", past="0", page=128, window=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _words(v):
    return " ".join(map(str, v))


def draw(rng):
    kind = rng.choice(["tables", "rope", "append", "append", "read", "attend", "attend", "attend", "attend"])
    layout, page = rng.choice(["qwen3", "qwen3", "gptoss", "gptoss", "even", "odd", "wide", "small"]), 16 << rng.randint(0, 4)
    if kind == "tables":
        return dict(kind=kind, first=rng.choice([0, _log_int(rng, 1, 1000000)]), len=_log_int(rng, 1, 131072),
                    rot=8 * rng.randint(2, 8), scaling=rng.choice(SCALINGS), factor=float(rng.choice([2, 4, 8, 32])))
    if kind == "rope":
        return dict(kind=kind, layout=layout, rows=_log_int(rng, 1, 4001), far=_log_int(rng, 1, 100000),
                    interleaved=rng.random() < 0.5)
    if kind == "append":
        n = _log_int(rng, 1, 32)
        return dict(kind=kind, layout=layout, lens=_words(_log_int(rng, 1, 4000 // n) for _ in range(n)),
                    past=_words(rng.choice([0, _log_int(rng, 1, 4000)]) for _ in range(n)), page=page, interleaved=rng.random() < 0.5)
    if kind == "read":
        n = _log_int(rng, 1, 16)
        return dict(kind=kind, layout=layout, lens=_words(_log_int(rng, 1, 15000 // n) for _ in range(n)), page=page,
                    half=rng.random() < 0.5)
    window = rng.choice([0, 0, 128, _log_int(rng, 1, 4000)])
    way = rng.choice(["whole", "chunk", "decode", "decode"])
    if way == "whole":
        n = rng.choice([1, _log_int(rng, 2, 12)])
        lens, past = [_log_int(rng, 1, 5000 // n) for _ in range(n)], [0] * n
    elif way == "chunk":
        n = rng.choice([1, 1, 3])
        lens, past = [_log_int(rng, 2, 500) for _ in range(n)], [_log_int(rng, 1, 30000 // n) for _ in range(n)]
    else:
        n = _log_int(rng, 1, 64)
        lens, past = [1] * n, [_log_int(rng, 1, 8000) for _ in range(n)]
    return dict(kind=kind, layout=layout, lens=_words(lens), past=_words(past), page=page, window=window)


# ------------------------------------------------------------------ inputs

class State:
    pass


def _lens(case):
    lens = [int(w) for w in case["lens"].split()]
    return lens, [int(w) for w in case.get("past", "0 " * len(lens)).split()]


def _ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    s = State()
    s.kind, s.scratch = case["kind"], None
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if s.kind == "tables":
        _prepare_tables(s, case, seed)
    elif s.kind == "rope":
        _prepare_rope(s, case, g)
    else:
        _prepare_pages(s, case, g)
    torch.cuda.synchronize()   # the library's stream reads what torch's wrote
    return s


def _prepare_tables(s, case, seed):
    s.first, s.len, s.rot, s.scaling, s.factor = (case[k] for k in ("first", "len", "rot", "scaling", "factor"))
    s.theta = 150000.0 + 1000.0 * (seed % 97)
    s.original = 4096
    s.low, s.high = (1.0, 4.0) if s.scaling == "smooth" else (32.0, 1.0)
    s.times = 1.0 if s.factor == 1 else 0.1 * math.log(s.factor) + 1.0
    s.cos, s.sin = (torch.empty(s.len, s.rot // 2, device="cuda") for _ in range(2))


def _prepare_rope(s, case, g):
    nh, nkv, s.hd, s.rot, _, _ = LAYOUTS[case["layout"]]
    s.heads, s.rows, s.interleaved = nh + nkv, case["rows"], case["interleaved"]   # queries and keys side by side
    s.table = case["far"]
    s.x = torch.randn(s.rows, s.heads * s.hd, generator=g, device="cuda")
    s.y = torch.empty_like(s.x)
    s.pos = torch.randint(0, s.table, (s.rows,), generator=g, device="cuda", dtype=torch.int32)
    s.cos, s.sin = _angles(s.table, s.rot)


def _angles(n, rot):
    angle = torch.arange(n, device="cuda")[:, None].double() / 1e6 ** (torch.arange(rot // 2, device="cuda").double() / (rot // 2))
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _prepare_pages(s, case, g):
    normal = lambda *shape, scale=1.0: torch.randn(*shape, generator=g, device="cuda") * scale   # noqa: E731
    s.nh, s.nkv, s.hd, s.rot, norm, sinks = LAYOUTS[case["layout"]]
    lens, past = _lens(case)
    s.n, s.rows, s.most, s.page = len(lens), sum(lens), max(lens), case["page"]
    s.total = max(a + b for a, b in zip(lens, past))             # the longest sequence
    need = [-(-(a + b) // s.page) for a, b in zip(lens, past)]
    s.stride = max(need) + 3                                     # the table has room for more
    s.n_pages = sum(need) + 5
    order = torch.randperm(s.n_pages, generator=g, device="cuda").int()
    s.table = torch.full((s.n, s.stride), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):   # pages of a sequence lie anywhere
        s.table[i, :m] = order[at:at + m]
        at += m
    s.cu, s.kv_len = _ints(np.concatenate([[0], np.cumsum(lens)])), _ints(past)
    # every page is full of some sequence's rows, stale ones among them
    s.pages, s.exps = [], []
    for _ in range(2):
        x = torch.randn(s.n_pages, s.nkv, s.page // BLOCK, BLOCK, s.hd, generator=g, device="cuda")
        x *= torch.exp2(normal(s.n_pages, s.nkv, s.page // BLOCK, 1, 1, scale=0.5))
        e = _exponent(x.abs().amax((3, 4)).double())
        s.pages.append(torch.round(x * _power(-e, torch.float32)[..., None, None]).to(torch.int8).view(s.n_pages, s.nkv, s.page, s.hd))
        s.exps.append((e + 127).to(torch.uint8))
    if s.kind == "read":
        s.after, s.half = _ints(lens), case["half"]
        s.kv_max = 64 * (s.total // 64 + 1)
        s.slots = _ints(reversed(range(s.n)))
        s.out = [torch.zeros(s.n, s.nkv, s.kv_max, s.hd, device="cuda", dtype=torch.float16 if s.half else torch.float32) for _ in range(2)]
        return
    if s.kind == "append":
        s.interleaved = case["interleaved"]
        s.after = _ints(a + b for a, b in zip(lens, past))
        s.kv_max, s.slots, s.half = s.total, None, False
        s.values = [torch.zeros(s.n, s.nkv, s.kv_max, s.hd, device="cuda") for _ in range(2)]
        s.qkv = normal(s.rows, (s.nh + 2 * s.nkv) * s.hd, scale=1.5)   # the projections, side by side
        s.norms = [torch.empty(s.hd, device="cuda").uniform_(0.5, 1.5, generator=g) for _ in range(2)] if norm else [None] * 2
        s.cos, s.sin = _angles(s.total, s.rot)
        s.out = torch.empty(s.rows, s.nh * s.hd, device="cuda")
        return
    s.window = case["window"]
    s.sinks = normal(s.nh) if sinks else None
    s.q = normal(s.rows, s.nh * s.hd, scale=2.0)                 # scores of a trained model's spread
    s.out = torch.zeros(s.rows, s.nh * s.hd, device="cuda")


# ------------------------------------------------------------------ one pass

def _ptr(t):
    return None if t is None else t.data_ptr()


def run(s):
    if own:
        return _run_own(s)
    return {"tables": _plain_tables, "rope": _plain_rope, "append": _plain_append, "read": _plain_read,
            "attend": _plain_attend}[s.kind](s)


def _run_own(s):
    import tinygiant_amd as tg
    lib = tg.lib()
    if s.kind == "tables":
        lib.tg_hip_rope_tables_dev(s.cos.data_ptr(), s.sin.data_ptr(), s.len, s.first, s.rot, s.theta, SCALINGS.index(s.scaling),
                                   s.factor, s.original, s.low, s.high, s.times, None)
        return dict(cos=s.cos, sin=s.sin)
    if s.kind == "rope":
        lib.tg_hip_rope_dev(s.x.data_ptr(), s.heads * s.hd, s.pos.data_ptr(), s.cos.data_ptr(), s.sin.data_ptr(), s.table, s.rot,
                            s.interleaved, s.rows, s.heads, s.hd, s.y.data_ptr(), s.heads * s.hd, None)
        return s.y
    pages = (*(t.data_ptr() for t in s.pages), *(t.data_ptr() for t in s.exps), s.n_pages, s.page, s.table.data_ptr(), s.stride)
    if s.kind == "read":
        lib.tg_hip_paged_read_dev(*pages, s.after.data_ptr(), s.n, s.nkv, s.hd, int(s.half), *(t.data_ptr() for t in s.out),
                                  s.slots.data_ptr(), s.n, s.kv_max, None)
        return dict(k=s.out[0], v=s.out[1])
    if s.kind == "append":
        p, qd, kd, st = s.qkv.data_ptr(), s.nh * s.hd, s.nkv * s.hd, (s.nh + 2 * s.nkv) * s.hd
        lib.tg_hip_paged_append_dev(p, p + 4 * qd, p + 4 * (qd + kd), st, st, _ptr(s.norms[0]), _ptr(s.norms[1]), EPS,
                                    s.cos.data_ptr(), s.sin.data_ptr(), len(s.cos), s.rot, s.interleaved, s.cu.data_ptr(),
                                    s.kv_len.data_ptr(), s.n, s.rows, *pages, s.nh, s.nkv, s.hd, s.out.data_ptr(), qd, None)
        # the bytes that the sequences now hold, as values
        lib.tg_hip_paged_read_dev(*pages, s.after.data_ptr(), s.n, s.nkv, s.hd, 0, *(t.data_ptr() for t in s.values), None, s.n,
                                  s.kv_max, None)
        return dict(q=s.out, k=s.values[0], v=s.values[1])
    if s.scratch is None:   # a program allocates it once
        need = lib.tg_hip_attention_paged_scratch_bytes(s.rows, s.n, s.nh, s.nkv, s.hd, s.total)
        s.scratch = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)
    qd = s.nh * s.hd
    lib.tg_hip_attention_paged_dev(s.q.data_ptr(), qd, *pages, s.cu.data_ptr(), s.kv_len.data_ptr(), s.n, s.rows, s.total,
                                   s.window, _ptr(s.sinks), s.nh, s.nkv, s.hd, s.out.data_ptr(), qd, s.scratch.data_ptr(), None)
    return s.out


def _plain_tables(s):
    """In 64 bits: angles of far positions."""
    i = torch.arange(s.rot // 2, device="cuda").double()
    theta = s.theta * s.factor ** (s.rot / (s.rot - 2)) if s.scaling == "base" else s.theta
    f = torch.exp(-math.log(theta) * 2 * i / s.rot)
    if s.scaling == "linear":
        f = f / s.factor
    elif s.scaling.startswith("parts"):
        # the pair that turns `low` (`high`) times in the original context, as a place among the pairs
        a, b = (s.rot * math.log(s.original / (turns * 2 * math.pi)) / (2 * math.log(s.theta)) for turns in (s.low, s.high))
        if s.scaling == "parts whole":
            a, b = math.floor(a), math.ceil(b)
        a, b = max(a, 0.0), min(b, s.rot - 1.0)
        ramp = ((i - a) / max(b - a, 0.001)).clamp(0, 1)
        f = f / s.factor * ramp + f * (1 - ramp)
    elif s.scaling == "smooth":
        share = ((s.original * f / (2 * math.pi) - s.low) / (s.high - s.low)).clamp(0, 1)
        f = f / s.factor * (1 - share) + f * share
    angle = (torch.arange(s.len, device="cuda") + s.first).double()[:, None] * f
    return dict(cos=(angle.cos() * s.times).float(), sin=(angle.sin() * s.times).float())


def _turn(x, c, sn, rot, interleaved):
    """The first `rot` values of every head: pairs (i, i + rot / 2), or neighbours."""
    y, c, sn = x.clone(), c[:, None], sn[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * sn, b * c + a * sn
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * sn, b * c + a * sn
    return y


def _plain_rope(s):
    at = s.pos.long()
    return _turn(s.x.view(s.rows, s.heads, s.hd), s.cos[at], s.sin[at], s.rot, s.interleaved).view(s.rows, -1)


def _exponent(big):
    """The least e of LEAST .. MOST with big <= 127 2^e."""
    m, k = torch.frexp(big)
    e = k - 7 + (m > 127 / 128)
    return torch.where(big > 0, e, LEAST).clamp(LEAST, MOST)


def _power(e, dtype):
    """2^e exactly, where exp2 may be off by its last bit."""
    return torch.ldexp(torch.ones(e.shape, device="cuda", dtype=dtype), e.int())


def _places(s):
    """Of every packed row: its sequence, and its place in it."""
    r = torch.arange(s.rows, device="cuda")
    seq = (r[:, None] >= s.cu[None, 1:]).sum(1)
    return seq, r - s.cu[seq]


def _norm(x, w):
    return x if w is None else x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w


def _gather(s, which, n):
    """Positions 0 .. n - 1 of every sequence as values [n_seqs][KV heads][n][head size], 0 where it has no page."""
    t = s.table[:, :-(-n // s.page)].long()
    v = s.pages[which][t.clamp(min=0)].float().view(s.n, t.shape[1], s.nkv, s.page // BLOCK, BLOCK, s.hd)
    v = v * _power(s.exps[which][t.clamp(min=0)].int() - 127, torch.float32)[..., None, None]
    v = torch.where((t >= 0)[:, :, None, None, None, None], v, 0)
    return v.view(s.n, t.shape[1], s.nkv, s.page, s.hd).transpose(1, 2).reshape(s.n, s.nkv, -1, s.hd)[:, :, :n]


def _plain_append(s):
    """K and V in 64 bits up to the rounding: a value next to the border of two bytes."""
    seq, i = _places(s)
    at = (s.kv_len[seq] + i).long()
    q, k, v = s.qkv.view(s.rows, -1, s.hd).split([s.nh, s.nkv, s.nkv], 1)
    q = _turn(_norm(q, s.norms[0]), s.cos[at], s.sin[at], s.rot, s.interleaved)
    k = _turn(_norm(k.double(), s.norms[1]), s.cos[at].double(), s.sin[at].double(), s.rot, s.interleaved)
    blocks = s.page // BLOCK
    block = s.table[seq, at // s.page].long() * blocks + at % s.page // BLOCK      # the row's block, of all pages'
    kept = s.kv_len[seq] > at - at % BLOCK                                        # it holds earlier rows
    for which, new in ((0, k), (1, v.double())):
        exps = s.exps[which].transpose(1, 2).reshape(-1, s.nkv)                   # [pages and blocks][KV heads]
        big = torch.zeros(exps.shape, device="cuda", dtype=torch.float64)
        big.scatter_reduce_(0, block[:, None].expand(-1, s.nkv), new.abs().amax(-1), "amax")
        touched, holds = (torch.zeros(len(exps), device="cuda", dtype=torch.bool) for _ in range(2))
        touched[block] = True
        holds[block[kept]] = True
        old = exps.int() - 127
        e = torch.where(holds[:, None], torch.maximum(_exponent(big), old), _exponent(big))
        e = torch.where(touched[:, None], e, old)
        # rows that a block held before, in its new unit
        moved = torch.nonzero(holds)[:, 0]
        p, b = moved // blocks, moved % blocks
        pages = s.pages[which].view(s.n_pages, s.nkv, blocks, BLOCK, s.hd)
        pages[p, :, b] = torch.round(pages[p, :, b].float() * _power((old - e)[moved], torch.float32)[..., None, None]).to(torch.int8)
        pages = s.pages[which]
        pages[block // blocks, :, at % s.page] = torch.round(new * _power(-e[block], torch.float64)[..., None]).to(torch.int8)
        s.exps[which].copy_((e + 127).to(torch.uint8).view(s.n_pages, blocks, s.nkv).transpose(1, 2))
    live = (torch.arange(s.total, device="cuda") < s.after[:, None])[:, None, :, None]
    for which in range(2):
        s.values[which].copy_(torch.where(live, _gather(s, which, s.total), s.values[which]))
    return dict(q=q.reshape(s.rows, -1), k=s.values[0], v=s.values[1])


def _plain_read(s):
    live = (torch.arange(s.total, device="cuda") < s.after[:, None])[:, None, :, None]
    for which in range(2):
        to = s.out[which][s.slots.long(), :, :s.total]
        s.out[which][s.slots.long(), :, :s.total] = torch.where(live, _gather(s, which, s.total).to(to.dtype), to)
    return dict(k=s.out[0], v=s.out[1])


def _plain_attend(s):
    """Sequences padded to the longest, scores of all heads at once."""
    seq, i = _places(s)
    group, scale = s.nh // s.nkv, s.hd ** -0.5
    q = torch.zeros(s.n, s.nkv, group, s.most, s.hd, device="cuda")
    q[seq, :, :, i] = s.q.view(s.rows, s.nkv, group, s.hd)
    keys, vals = (_gather(s, which, s.total) for which in range(2))
    z = torch.matmul(q.view(s.n, s.nkv, -1, s.hd), keys.transpose(2, 3).contiguous()).view(s.n, s.nkv, group, s.most, s.total)
    place = torch.arange(s.most, device="cuda")[None, :, None] + s.kv_len[:, None, None]
    key = torch.arange(s.total, device="cuda")
    see = key <= place
    if s.window:
        see = see & (key > place - s.window)
    z.mul_(scale).masked_fill_(~see[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    if s.sinks is not None:
        sink = s.sinks.view(1, s.nkv, group, 1, 1)
        m = torch.maximum(m, sink)
    p = z.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + (sink - m).exp()
    o = torch.matmul(p.view(s.n, s.nkv, group * s.most, -1), vals.contiguous()).view(s.n, s.nkv, group, s.most, s.hd) / total
    return o[seq, :, :, i].reshape(s.rows, -1)


# ------------------------------------------------------------------ the work of a pass

def work(case):
    if case["kind"] == "tables":
        return dict(bytes=4 * case["len"] * case["rot"], flops=24 * case["len"] * case["rot"])
    nh, nkv, hd, rot, _, _ = LAYOUTS[case["layout"]]
    if case["kind"] == "rope":
        rows, heads = case["rows"], nh + nkv
        return dict(bytes=rows * (8 * heads * hd + 4 * rot + 4), flops=3 * rows * heads * rot)
    lens, past = _lens(case)
    rows, held = sum(lens), 1 + 1 / (BLOCK * hd)                  # bytes of a value in a page
    if case["kind"] == "read":
        return dict(bytes=int(2 * nkv * hd * rows * (held + (2 if case["half"] else 4))), flops=2 * nkv * hd * rows)
    if case["kind"] == "append":
        live = rows + sum(past)
        return dict(bytes=int(rows * hd * (8 * nh + 2 * nkv * (4 + held)) + 4 * rows * rot + 2 * nkv * hd * live * (held + 4)),
                    flops=rows * hd * (nh + nkv) * 8)
    pairs, seen, window = 0, 0, case["window"]
    for n, p in zip(lens, past):
        ends = np.arange(n) + p + 1                               # positions that each row could see
        pairs += int(np.minimum(ends, window).sum() if window else ends.sum())
        seen += n + p - (max(0, p + 1 - window) if window else 0)
    return dict(bytes=int(2 * nkv * hd * held * seen) + 8 * rows * nh * hd, flops=4 * nh * hd * pairs)


# ------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "tables":
        return _exact_tables(s)
    if s.kind == "rope":
        return _exact_turn(s.x.double().view(s.rows, s.heads, s.hd), s.pos.tolist(), s).view(s.rows, -1)
    lens, past = _lens(case)
    if s.kind == "read":
        out = [t.double() for t in s.out]
        for b, n in enumerate(lens):
            for which in range(2):
                out[which][s.n - 1 - b, :, :n] = _exact_held(s, which, b, n)
        return dict(k=out[0], v=out[1])
    if s.kind == "append":
        return _exact_append(s, lens, past)
    group, out, r = s.nh // s.nkv, [], 0
    heads = s.q.double().view(s.rows, s.nkv, group, s.hd)
    for b, (n, p) in enumerate(zip(lens, past)):
        keys, vals = (_exact_held(s, which, b, p + n) for which in range(2))
        ends, where = torch.arange(p, p + n, device="cuda"), torch.arange(p + n, device="cuda")
        hide = where[None] > ends[:, None]
        if s.window:
            hide |= where[None] <= ends[:, None] - s.window
        mine = torch.empty(n, s.nkv, group, s.hd, device="cuda", dtype=torch.float64)
        for h in range(s.nkv):
            for j in range(group):
                z = heads[r:r + n, h, j] @ keys[h].T / math.sqrt(s.hd)
                z[hide] = -math.inf
                top = z.max(1, keepdim=True).values
                extra = 0
                if s.sinks is not None:
                    sink = s.sinks[h * group + j].double()
                    top = torch.clamp(top, min=sink)
                    extra = torch.exp(sink - top)
                w = torch.exp(z - top)
                mine[:, h, j] = (w @ vals[h]) / (w.sum(1, keepdim=True) + extra)
        out.append(mine.view(n, -1))
        r += n
    return torch.cat(out)


def _exact_tables(s):
    f = np.empty(s.rot // 2)
    for i in range(s.rot // 2):
        if s.scaling == "base":
            f[i] = (s.theta * s.factor ** (s.rot / (s.rot - 2))) ** (-2 * i / s.rot)
            continue
        f[i] = s.theta ** (-2 * i / s.rot)
        if s.scaling == "linear":
            f[i] /= s.factor
        elif s.scaling == "smooth":   # pairs by how often they turn in the original context
            turns = s.original * f[i] / (2 * math.pi)
            if turns < s.low:
                f[i] /= s.factor
            elif turns < s.high:
                share = (turns - s.low) / (s.high - s.low)
                f[i] = share * f[i] + (1 - share) * f[i] / s.factor
        elif s.scaling != "plain":
            a, b = (s.rot / 2 * (math.log(s.original) - math.log(2 * math.pi * t)) / math.log(s.theta) for t in (s.low, s.high))
            if s.scaling == "parts whole":
                a, b = math.floor(a), math.ceil(b)
            a, b = max(a, 0), min(b, s.rot - 1)
            ramp = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            f[i] *= ramp / s.factor + 1 - ramp
    angle = torch.from_numpy(np.outer(np.arange(s.first, s.first + s.len, dtype=np.float64), f))
    return dict(cos=(torch.cos(angle) * s.times).cuda(), sin=(torch.sin(angle) * s.times).cuda())


def _exact_turn(x, pos, s):
    """As products of complex numbers."""
    at = torch.tensor(pos, device="cuda")
    unit = torch.complex(s.cos[at].double(), s.sin[at].double())[:, None]
    y, half = x.clone(), s.rot // 2
    first, second = ((slice(0, s.rot, 2), slice(1, s.rot, 2)) if s.interleaved else (slice(0, half), slice(half, s.rot)))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_held(s, which, b, n):
    """Positions 0 .. n - 1 of sequence b: [KV heads][n][head size]."""
    parts = []
    for j in range(-(-n // s.page)):
        page = int(s.table[b, j])
        unit = torch.from_numpy(np.ldexp(1.0, s.exps[which][page].int().cpu().numpy() - 127)).cuda()   # [KV heads][blocks]
        parts.append(s.pages[which][page].double() * unit.repeat_interleave(BLOCK, 1)[..., None])
    return torch.cat(parts, 1)[:, :n] if n else torch.zeros(s.nkv, 0, s.hd, device="cuda", dtype=torch.float64)


def _exact_append(s, lens, past):
    x = s.qkv.double().view(s.rows, -1, s.hd)
    out, q_out, r = [t.double() for t in s.values], [], 0
    for b, (n, p) in enumerate(zip(lens, past)):
        y = x[r:r + n].clone()
        for part, w in ((slice(0, s.nh), s.norms[0]), (slice(s.nh, s.nh + s.nkv), s.norms[1])):
            if w is not None:
                y[:, part] *= w.double() / torch.sqrt(y[:, part].pow(2).sum(-1, keepdim=True) / s.hd + EPS)
        y[:, :s.nh + s.nkv] = _exact_turn(y[:, :s.nh + s.nkv], list(range(p, p + n)), s)
        q_out.append(y[:, :s.nh].reshape(n, -1))
        first = p // BLOCK * BLOCK                                # the first block that the rows touch
        for which in range(2):
            new = y[:, s.nh + which * s.nkv:s.nh + (which + 1) * s.nkv].transpose(0, 1)
            held = _exact_held(s, which, b, p)
            rows = torch.cat([held[:, first:], new], 1)
            pad = torch.nn.functional.pad(rows, (0, 0, 0, -rows.shape[1] % BLOCK)).view(s.nkv, -1, BLOCK, s.hd)
            fresh = torch.nn.functional.pad(new, (0, 0, p - first, -rows.shape[1] % BLOCK)).view(s.nkv, -1, BLOCK, s.hd)
            e = torch.ceil(torch.log2(fresh.abs().amax((2, 3)) / 127)).clamp(LEAST, MOST)
            if p > first:   # a block's unit never shrinks while it holds rows
                page, block = int(s.table[b, first // s.page]), first % s.page // BLOCK
                e[:, 0] = torch.maximum(e[:, 0], s.exps[which][page, :, block].double() - 127)
            unit = torch.from_numpy(np.ldexp(1.0, e.int().cpu().numpy())).cuda()
            pad = torch.round(pad / unit[..., None, None]) * unit[..., None, None]
            out[which][b, :, :first] = held[:, :first]
            out[which][b, :, first:p + n] = pad.view(s.nkv, -1, s.hd)[:, :p + n - first]
        r += n
    return dict(q=torch.cat(q_out), k=out[0], v=out[1])
