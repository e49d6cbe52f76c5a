"""Cases of the decode-step operators around the quantised products: the norm, the rotary append to the 8-bit cache,
attention over that cache, and sampling. `own` chooses between the plain torch forms and the library's kernels.

The 8-bit cache: pages of `page` tokens; codes uint8 [pages][kv_heads][page][dim], stored as code + 128 (-127..127),
one fp32 scale per page and head for K and for V; value = code * scale. A sequence's token p is in slot p % page of
page table[seq][p / page].
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _vkb():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "volta-kernel-bakeoff_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import vkb
    return vkb


# ---- the cases -------------------------------------------------------------------------------------------------------

def _attn(name, batch, longest, new, q_heads, kv_heads, dim, page, dtype="f16", window=0, spread=0):
    c = dict(op="attention", batch=batch, longest=longest, new=new, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
             page=page, dtype=dtype, window=window, spread=spread)
    return dict(c, name=name) if name else c


def _append(name, batch, longest, new, q_heads, kv_heads, dim, rot, page, layout, stretch=1.0, dtype="f16", spread=0):
    c = dict(op="append", batch=batch, longest=longest, new=new, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rot=rot,
             page=page, layout=layout, stretch=stretch, dtype=dtype, spread=spread)
    return dict(c, name=name) if name else c


def _norm(name, tokens, width, dtype, res, q8):
    c = dict(op="norm", tokens=tokens, width=width, dtype=dtype, res=res, q8=q8)
    return dict(c, name=name) if name else c


def _sample(name, rows, vocab, dtype, top_k, top_p, min_p):
    c = dict(op="sample", rows=rows, vocab=vocab, dtype=dtype, top_k=top_k, top_p=top_p, min_p=min_p)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one layer between two GEMVs: fp16 GEMV output added to an fp32 residual stream
        _norm("norm_token", 1, 2048, "f16", "f32", False),
        # a prompt's norm with the 8-bit copy for a transfer or an 8-bit consumer
        _norm("norm_prompt_q8", 8191, 2560, "bf16", "bf16", True),
        # one decode step of eight sequences, grown to different lengths, idle ones among them
        _append("append_step", 8, 4000, 1, 32, 8, 128, 128, 64, "half", spread=5),
        # ragged prompts entering the cache, part of each head rotated, positions stretched for a long context
        _append("append_prompts", 6, 3500, 3500, 16, 4, 256, 64, 16, "interleaved", 4.0, "bf16", spread=11),
        # the smallest attention: a short chat's next token
        _attn("attn_short", 1, 777, 1, 32, 8, 128, 64),
        # a serving batch: 64 sequences of very different lengths, one token each
        _attn("attn_serve", 64, 8192, 1, 32, 8, 128, 64, spread=3),
        # one long document, one token, few kv heads: the split over the long axis
        _attn("attn_long", 1, 131073, 1, 24, 4, 128, 128, "bf16"),
        # checking drafted tokens: a few query tokens per sequence, small heads
        _attn("attn_drafted", 16, 3001, 5, 16, 16, 64, 32, spread=9),
        # a prompt chunk behind a long prefix: tensor-core work
        _attn("attn_chunk", 1, 16384, 4096, 32, 8, 128, 64, "bf16"),
        # ragged prompts through a sliding window, wide heads
        _attn("attn_prompts_window", 5, 2500, 2500, 16, 2, 256, 16, "f16", window=1024, spread=21),
        # a single user's next token
        _sample("sample_one", 1, 32000, "f16", 40, 0.95, 0.0),
        # a serving batch over a large vocabulary with mixed settings
        _sample("sample_serve", 256, 151936, "f32", 1000, 0.9, 0.02),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attention", "attention", "attention", "sample"])
    if op == "norm":
        width = rng.choice([2048, 2560, 6144]) if rng.random() < 0.5 else 32 * _log(rng, 1, 256)
        q8 = rng.random() < 0.5
        if not q8 and rng.random() < 0.4:
            width = _log(rng, 1, 8191)
        return _norm(None, _log(rng, 1, max(1, min(8192, (1 << 24) // width))), width,
                     rng.choice(["f16", "bf16", "f32"]), rng.choice(["f16", "bf16", "f32", "none"]), q8)
    if op == "sample":
        vocab = _log(rng, 100, 200000)
        return _sample(None, _log(rng, 1, max(1, min(256, (256 * 140000) // vocab))), vocab,
                       rng.choice(["f16", "bf16", "f32"]), rng.choice([0, 1, 20, _log(rng, 2, 5000)]),
                       rng.choice([1.0, 0.95, 0.8, round(rng.uniform(0.1, 1.0), 3)]), rng.choice([0.0, 0.05, 0.01]))
    kv, group, dim = rng.choice([(8, 4, 128), (4, 6, 128), (2, 8, 256), (8, 5, 128), (1, 16, 64), (16, 1, 64),
                                 (3, 3, 80), (2, 7, 192), (4, 1, 96)])
    page, dtype, spread = rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16", "f32"]), rng.randrange(1, 1 << 20)
    kind = rng.choice(["token", "token", "drafted", "prompt"])
    if op == "append":
        batch = _log(rng, 1, 64) if kind != "prompt" else _log(rng, 1, 8)
        longest = _log(rng, 2, 20000 // batch if kind == "prompt" else 8000)
        rot = rng.choice([dim, dim // 2, 0])
        return _append(None, batch, longest, 1 if kind == "token" else rng.randint(2, 9) if kind == "drafted" else longest,
                       kv * group, kv, dim, rot, page, rng.choice(["half", "interleaved"]), rng.choice([1.0, 2.0, 8.0]),
                       dtype, spread)
    window = rng.choice([0, 0, 0, _log(rng, 1, 4000)])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "prompt":
        batch = _log(rng, 1, 6)
        longest = _log(rng, 2, 16384 // batch)
        c = _attn(None, batch, longest, _log(rng, 2, min(longest, 4096)), kv * group, kv, dim, page, dtype, window, spread)
        while work(c)["flops"] > 9e11:
            c["new"] //= 2
        return c
    batch = _log(rng, 1, 100)
    longest = _log(rng, 1, min(40000, 400000 // (batch * max(1, kv * dim // 1024))))
    return _attn(None, batch, longest, 1 if kind == "token" else rng.randint(2, 9), kv * group, kv, dim, page, dtype,
                 window, spread)


def _lengths(case):
    """(lens, news): each sequence's length with its new tokens, and how many of them are new. From the case alone."""
    b, longest, new = case["batch"], case["longest"], case["new"]
    if not case["spread"]:
        return [longest] * b, [min(new, longest)] * b
    r = random.Random(case["spread"])
    lens = [longest] + [0 if r.random() < 0.06 else r.randint(1, longest) for _ in range(b - 1)]
    if new == 1:
        return lens, [1] * b          # one query token per sequence; a sequence of length 0 is an idle one
    news = [min(n, new) if r.random() < 0.5 else r.randint(0, min(n, new)) for n in lens]
    news[0] = max(1, news[0])
    return lens, news


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _cache(case, g, lens):
    """A filled cache in pages of random order: codes of roughly normal values, scales that differ by page and head."""
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    per = [(n + page - 1) // page for n in lens]
    total, width = sum(per) + 3, max(max(per), 1)
    dev = "cuda"

    def codes():
        t = torch.empty((total, h, page, d), dtype=torch.uint8, device=dev)
        rows = max(1, (1 << 27) // (h * page * d))
        for i in range(0, total, rows):
            n = min(rows, total - i)
            t[i:i + n] = torch.randn((n, h, page, d), generator=g, device=dev).mul_(34).round_().clamp_(-127, 127).add_(128).to(torch.uint8)
        return t
    k, v = codes(), codes()
    ks = torch.rand((total, h), generator=g, device=dev) * 0.04 + 0.02
    vs = torch.rand((total, h), generator=g, device=dev) * 0.04 + 0.01
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((len(lens), width), dtype=torch.int32, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=dev), torch.tensor(per, device=dev), output_size=sum(per))
    first = torch.tensor([sum(per[:i]) for i in range(len(per))], device=dev)
    at = torch.arange(sum(per), device=dev)
    table[seq, at - first[seq]] = order[:sum(per)]
    return k, v, ks, vs, table


def _turns(case):
    """Turns per position of each rotated pair, as 64-bit fractions of a turn (base 10000, positions divided by stretch)."""
    n = case["rot"] // 2
    f = [10000.0 ** (-i / n) / case["stretch"] / (2 * math.pi) for i in range(n)]
    whole = [int(x * 2.0 ** 64) & ((1 << 64) - 1) for x in f]
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in whole], dtype=torch.int64, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dev = case["op"], "cuda"

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)
    st = {"case": case}
    if op == "norm":
        t, d, dt = case["tokens"], case["width"], _DT[case["dtype"]]
        st["x"] = randn(t, d).to(dt)
        st["weight"] = (1 + 0.2 * randn(d)).to(dt)
        if case["res"] != "none":   # a residual stream grows to several times its branches, a few channels far more
            st["res"] = (randn(t, d) * 4 * (1 + 20 * (torch.rand(d, generator=g, device=dev) < 0.01))).to(_DT[case["res"]])
        return st
    if op == "sample":
        b, v = case["rows"], case["vocab"]
        peak = 1.0 + 3.0 * torch.rand((b, 1), generator=g, device=dev)       # confident and undecided rows
        st["logits"] = (randn(b, v) * peak).to(_DT[case["dtype"]])
        banned = torch.rand((b, v), generator=g, device=dev) < 0.02           # tokens a grammar forbids
        banned[:, 0] = False
        st["logits"][banned] = float("-inf")
        st["u"] = torch.rand(b, generator=g, device=dev)
        st["temperature"] = 0.5 + torch.rand(b, generator=g, device=dev)
        st["temperature"][3::7] = 0.0                                          # greedy rows among them
        st["top_k"] = torch.full((b,), case["top_k"], dtype=torch.int32, device=dev)
        st["top_p"] = torch.full((b,), case["top_p"], device=dev)
        st["min_p"] = torch.full((b,), case["min_p"], device=dev)
        st["top_k"][5::6] = 0                                                  # rows without a top-k
        return st
    lens, news = _lengths(case)
    hq, h, d, dt = case["q_heads"], case["kv_heads"], case["dim"], _DT[case["dtype"]]
    t = sum(news)
    st["k"], st["v"], st["ks"], st["vs"], st["table"] = _cache(case, g, lens)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    ends = [sum(news[:i]) for i in range(len(news) + 1)]
    st["cu"] = torch.tensor(ends, dtype=torch.int32, device=dev)
    st["one"] = case["new"] == 1
    qkv = (randn(t, hq + 2 * h, d) * 1.3).to(dt)          # the fused projection's output: q, k and v are views of it
    if op == "attention":
        st["q"] = qkv[:, :hq]
    else:
        st["q"], st["kn"], st["vn"] = qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:]
        st["turns"] = _turns(case) if case["rot"] else None
        # the tokens of every page the call touches, for reading the cache back
        page, seq, pos = case["page"], [], []
        for b, (n, m) in enumerate(zip(lens, news)):
            first = max(0, (n - m) // page * page) if m else n
            pos += range(first, n)
            seq += [b] * (n - first)
        st["seq"] = torch.tensor(seq, dtype=torch.int32, device=dev)
        st["pos"] = torch.tensor(pos, dtype=torch.int32, device=dev)
    if own:   # the handle and the workspace that a serving program keeps beside its cache
        vkb = _vkb()
        st["cache"] = vkb.KvCache(st["k"], st["v"], st["ks"], st["vs"])
        if op == "attention":
            st["work"] = vkb.attention_workspace(st["cache"])
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    return (_OWN if own else _PLAIN)[op](state)


def _own_norm(st):
    vkb = _vkb()
    y, res, q, s = vkb.rms_norm(st["x"], st["weight"], st.get("res"), q8=st["case"]["q8"])
    out = {"y": y, "res": res}
    if q is not None:
        out["q8"] = vkb.dequant(vkb.FMT_Q8, q, s, q.shape[0], q.shape[1])
    return out


def _own_append(st):
    vkb = _vkb()
    q = vkb.rope_append(st["cache"], st["table"], st["lens"], st["q"], st["kn"], st["vn"], turns=st["turns"],
                        cu=None if st["one"] else st["cu"], layout=st["case"]["layout"])
    k, v = vkb.kv_read(st["cache"], st["table"], st["seq"], st["pos"])
    return {"q": q, "k": k, "v": v}


def _own_attention(st):
    return _vkb().attention(st["cache"], st["table"], st["lens"], st["q"], cu=None if st["one"] else st["cu"],
                            window=st["case"]["window"], work=st["work"])


def _own_sample(st):
    token, prob = _vkb().sample(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
    return {"token": token, "prob": prob}


def _plain_norm(st):
    x = st["x"].float()
    if "res" in st:
        x = x + st["res"].float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * st["weight"].float()
    out = {"y": y.to(st["x"].dtype), "res": x.to(st["res"].dtype) if "res" in st else None}
    if st["case"]["q8"]:
        b = y.reshape(y.shape[0], -1, 32)
        s = (b.abs().amax(-1, keepdim=True) / 127).half().float()
        code = torch.where(s > 0, b / s, torch.zeros_like(b)).round().clamp(-127, 127)
        out["q8"] = (code * s).reshape(y.shape).half()
    return out


def _plain_places(st):
    """(seq, position) of every new token, in order."""
    cu, lens = st["cu"].long(), st["lens"].long()
    t = st["q"].shape[0]
    at = torch.arange(t, device=cu.device)
    seq = torch.searchsorted(cu, at, right=True) - 1
    return seq, at - cu[seq + 1] + lens[seq]


def _plain_rotate(x, pos, turns, layout):
    if turns is None:
        return x
    n = turns.numel()
    angle = ((pos[:, None] * turns[None, :]) >> 40).float() * (2 * math.pi / (1 << 24))
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., :2 * n:2], x[..., 1:2 * n:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_append(st):
    case, page = st["case"], st["case"]["page"]
    seq, pos = _plain_places(st)
    q = _plain_rotate(st["q"].float(), pos, st["turns"], case["layout"])
    kn = _plain_rotate(st["kn"].float(), pos, st["turns"], case["layout"])
    live = torch.nonzero(pos >= 0).flatten()
    seq_l, pos_l = seq[live], pos[live]
    blk, slot = st["table"][seq_l, pos_l // page].long(), pos_l % page
    first = torch.zeros(st["k"].shape[0], dtype=torch.int64, device=blk.device) + page  # first new slot of each page
    first.scatter_reduce_(0, blk, slot, "amin")
    touched = torch.unique(blk)
    old = torch.arange(page, device=blk.device)[None, :] < first[touched][:, None]       # [touched][page] held before
    out = {"q": q.to(st["q"].dtype)}
    rs, rp = st["seq"].long(), st["pos"].long()
    rb = st["table"][rs, rp // page].long()
    for name, codes, scale, new in (("k", st["k"], st["ks"], kn), ("v", st["v"], st["vs"], st["vn"].float())):
        new = new[live]
        before = torch.where(first[touched][:, None] > 0, scale[touched], torch.zeros_like(scale[touched]))
        most = torch.zeros_like(scale).scatter_reduce_(0, blk[:, None].expand(-1, new.shape[1]), new.abs().amax(-1), "amax")
        after = torch.maximum(before, most[touched] / 127)
        held = codes[touched].float() - 128
        kept = torch.where(after > 0, before / after, torch.ones_like(after))[:, :, None, None]
        held = torch.where(old[:, None, :, None], (held * kept).round(), held)
        codes[touched] = (held + 128).to(torch.uint8)
        scale[touched] = after
        s = scale[blk][:, :, None]
        codes[blk, :, slot] = (torch.where(s > 0, new / s, torch.zeros_like(new)).round().clamp(-127, 127) + 128).to(torch.uint8)
        out[name] = ((codes[rb, :, rp % page].float() - 128) * scale[rb][:, :, None]).half()
    return out


def _plain_attention(st):
    case, page = st["case"], st["case"]["page"]
    b, hq, h, d = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    group = hq // h
    lens, cu, table = st["lens"].long(), st["cu"].long(), st["table"].long()
    news = _lengths(case)[1]
    widest = max(news)
    seq, pos = _plain_places(st)
    at = torch.arange(seq.numel(), device=seq.device) - cu[seq]

    def values(codes, scale):   # [b][h][longest][d]
        x = (codes[table].float() - 128) * scale[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    k = values(st["k"], st["ks"])
    q = torch.zeros((b, widest, hq, d), device=k.device)
    q[seq, at] = st["q"].float()
    where = torch.full((b, widest), -1, dtype=torch.int64, device=k.device)
    where[seq, at] = pos
    q = q.reshape(b, widest, h, group, d).permute(0, 2, 3, 1, 4).reshape(b, h, group * widest, d)
    s = (q * d ** -0.5) @ k.transpose(-1, -2)
    del k
    s = s.reshape(b, h, group, widest, -1)
    j = torch.arange(s.shape[-1], device=s.device)
    seen = (j <= where[..., None]) & (j < lens[:, None, None])
    if case["window"]:
        seen &= j > where[..., None] - case["window"]
    seen = seen[:, None, None]
    s = s.masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    s = s / torch.where(total > 0, total, torch.ones_like(total))
    o = s.reshape(b, h, group * widest, -1) @ values(st["v"], st["vs"])
    o = o.reshape(b, h, group, widest, d).permute(0, 3, 1, 2, 4).reshape(b, widest, hq, d)
    return o[seq, at].to(st["q"].dtype)


def _plain_sample(st):
    z = st["logits"].float()
    n = z.shape[1]
    cold = st["temperature"] <= 0
    z, order = torch.sort(z, dim=-1, descending=True, stable=True)
    d = (z - z[:, :1]) / torch.where(cold, torch.ones_like(st["temperature"]), st["temperature"])[:, None]
    w = torch.exp(d)
    rank = torch.arange(n, device=z.device)[None]
    k = torch.where((st["top_k"] <= 0) | (st["top_k"] > n), torch.full_like(st["top_k"], n), st["top_k"])
    k = torch.where(cold, torch.ones_like(k), k)
    w = torch.where(rank < k[:, None], w, torch.zeros_like(w))
    c = torch.cumsum(w, -1)
    keep = ((c - w) < st["top_p"][:, None] * c[:, -1:]) & (w >= st["min_p"][:, None]) | (rank == 0)
    w = torch.where(keep, w, torch.zeros_like(w))
    p = torch.zeros_like(w).scatter_(1, order, w)
    c = torch.cumsum(p, -1)
    total = c[:, -1:]
    past = (c > st["u"][:, None] * total) & (p > 0)
    past[:, -1] |= ~past.any(-1)
    token = torch.where(past, rank, torch.full_like(rank, n)).amin(-1)
    prob = p.gather(1, token[:, None]) / total
    return {"token": token.to(torch.int32), "prob": prob[:, 0]}


_OWN = {"norm": _own_norm, "append": _own_append, "attention": _own_attention, "sample": _own_sample}
_PLAIN = {"norm": _plain_norm, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4, "none": 0}
    op = case["op"]
    if op == "norm":
        n = case["tokens"] * case["width"]
        # the 8-bit copy is read back as fp16 values in the pass
        q8 = n * (1 + 2 / 32) * 2 + 2 * n if case["q8"] else 0
        return {"bytes": 2 * n * size[case["dtype"]] + 2 * n * size[case["res"]] + q8 + case["width"] * size[case["dtype"]], "flops": 4 * n}
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["dtype"]] + case["rows"] * 28, "flops": 3 * n}
    lens, news = _lengths(case)
    hq, h, d, e = case["q_heads"], case["kv_heads"], case["dim"], size[case["dtype"]]
    t = sum(news)
    if op == "append":
        page = case["page"]
        back = sum(n - (n - m) // page * page for n, m in zip(lens, news) if m and n)
        # q in and out, k and v in, their codes out; the touched pages read back as codes and written as fp16 values
        return {"bytes": t * d * (2 * hq * e + 2 * h * e + 2 * h) + back * 2 * h * d * 3,
                "flops": 3 * t * case["rot"] * (hq + h) + 4 * t * h * d}
    w = case["window"]
    pairs = held = 0
    for n, m in zip(lens, news):
        first = n - m                     # query tokens at positions first..n - 1 see first + 1..n keys, at most w
        if not w or n <= w:
            pairs += m * first + m * (m + 1) // 2 if n else 0
        else:
            grow = max(0, min(n, w) - first)     # query tokens that see less than the window
            pairs += grow * first + grow * (grow + 1) // 2 + (m - grow) * w
        held += n if not w else min(n, w + m - 1)
    return {"bytes": 2 * held * h * d + 2 * t * hq * d * e, "flops": 4 * pairs * hq * d}


# ---- the definition in 64 bits, sequence by sequence -----------------------------------------------------------------

def _exact_rows(st, seq):
    """K and V of one sequence as float64 [len][kv_heads][dim]."""
    page, n = st["case"]["page"], int(st["lens"][seq])
    at = torch.arange(n, device="cuda")
    blk, slot = st["table"][seq].long()[at // page], at % page
    return [(c[blk, :, slot].double() - 128.0) * s[blk].double().unsqueeze(-1) for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"]))]


def _exact_turn(x, pos, case):
    if not case["rot"]:
        return x
    n = case["rot"] // 2
    i = torch.arange(n, dtype=torch.float64, device=x.device)
    angle = torch.outer(pos.double(), 10000.0 ** (-i / n) / case["stretch"])[:, None, :]
    z = torch.polar(torch.ones_like(angle), angle)
    out = x.clone()
    first, second = (slice(0, n), slice(n, 2 * n)) if case["layout"] == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    w = torch.complex(x[..., first], x[..., second]) * z
    out[..., first], out[..., second] = w.real, w.imag
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        r = st["x"].double() + (st["res"].double() if "res" in st else 0.0)
        y = r / torch.sqrt(r.square().mean(1, keepdim=True) + 1e-6) * st["weight"].double()
        out = {"y": y, "res": r if "res" in st else None}
        if case["q8"]:
            b = y.view(-1, 32)
            s = (b.abs().max(1, keepdim=True).values / 127).half().double()
            out["q8"] = ((b / s.clamp_min(1e-300)).round().clamp(-127, 127) * s).view(y.shape)
        return out
    if op == "sample":
        probs = []
        for r in range(case["rows"]):
            z = st["logits"][r].double()
            t, k, p, m = (float(st[x][r]) for x in ("temperature", "top_k", "top_p", "min_p"))
            if t <= 0:
                probs.append(1.0)
                continue
            z, order = z.sort(descending=True, stable=True)
            w = ((z - z[0]) / t).exp()
            if 0 < k < w.numel():
                w, order = w[:int(k)], order[:int(k)]
            before = torch.cumsum(w, 0) - w
            n = max(1, int(((before < p * w.sum()) & (w >= m)).sum()))
            order, at = order[:n].sort()
            w = w[:n][at]
            c = torch.cumsum(w, 0)
            i = min(int(torch.searchsorted(c, float(st["u"][r]) * c[-1], right=True)), n - 1)
            probs.append(float(w[i] / c[-1]))
        return {"token": None, "prob": torch.tensor(probs, dtype=torch.float64)}
    lens, news = _lengths(case)
    ends = [sum(news[:i]) for i in range(len(news) + 1)]
    if op == "attention":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        h, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
        for b, (n, m) in enumerate(zip(lens, news)):
            if not n or not m:
                continue
            k, v = _exact_rows(st, b)
            pos = torch.arange(n - m, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = (j > pos) | ((j <= pos - case["window"]) if case["window"] else False)
            for q in range(case["q_heads"]):
                s = st["q"][ends[b]:ends[b + 1], q].double() @ k[:, q // group].T / math.sqrt(case["dim"])
                out[ends[b]:ends[b + 1], q] = torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ v[:, q // group]
        return out
    q_out, kept = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda"), {"k": [], "v": []}
    page = case["page"]
    for b, (n, m) in enumerate(zip(lens, news)):
        a, z = ends[b], ends[b + 1]
        pos = torch.arange(n - m, n, device="cuda")
        q_out[a:z] = _exact_turn(st["q"][a:z].double(), pos, case)
        if not n or not m:
            continue
        new = {"k": _exact_turn(st["kn"][a:z].double(), pos, case), "v": st["vn"][a:z].double()}
        for name in ("k", "v"):
            codes, scales = st[name], st[name + "s"]
            for blk in range((n - m) // page, (n - 1) // page + 1):
                lo, hi = max(n - m, blk * page), min(n, blk * page + page)     # its new tokens
                at, held = int(st["table"][b, blk]), lo - blk * page
                x = new[name][lo - (n - m):hi - (n - m)].transpose(0, 1)       # [heads][new][dim]
                was = scales[at].double() if held else torch.zeros_like(scales[at].double())
                s = torch.maximum(was, x.abs().amax((1, 2)) / 127).float().double()[:, None, None]
                back = (codes[at, :, :held].double() - 128) * was[:, None, None]
                x = torch.cat([back, x], 1)
                kept[name].append(((x / s.clamp_min(1e-300)).round().clamp(-127, 127) * s).transpose(0, 1))
    empty = torch.zeros((0, case["kv_heads"], case["dim"]), dtype=torch.float64, device="cuda")
    return {"q": q_out, "k": torch.cat(kept["k"] + [empty]), "v": torch.cat(kept["v"] + [empty])}
