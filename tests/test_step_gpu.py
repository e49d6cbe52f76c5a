"""GPU tests of the decode-step operators against plain implementations in 64 bits, one token and row at a time where that
is the definition. Tolerances come from the roundings that each operator's formula has (stated where they are used):
u16 = 2^-11 and ubf = 2^-8 are the half-ulp bounds of fp16 and bf16, u32 = 2^-24 of fp32."""
import math

import numpy as np
import pytest

import vkb

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def dt(name):
    import torch
    return getattr(torch, name)


def ulp(t):
    return U[str(t.dtype).split(".")[1]]


def tiny(t):   # the spacing of the type's subnormal numbers
    return {"float16": 2.0 ** -24, "bfloat16": 2.0 ** -133, "float32": 2.0 ** -149}[str(t.dtype).split(".")[1]]


def gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---- norm ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,d", [(1, 1), (3, 7), (1, 2048), (5, 32), (33, 96), (9, 2560), (2, 8191), (2, 16384), (3, 16392), (130, 64)])
@pytest.mark.parametrize("x_dt,res_dt", [("float16", "float32"), ("bfloat16", "bfloat16"), ("float32", None), ("float16", "float16")])
def test_rms_norm(cuda, T, d, x_dt, res_dt):
    import torch
    g = gen(T * 131 + d)
    x = torch.randn((T, d), generator=g, device="cuda").to(dt(x_dt))
    w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt(x_dt))
    res = None if res_dt is None else (4 * torch.randn((T, d), generator=g, device="cuda")).to(dt(res_dt))
    y, r, q, s = vkb.rms_norm(x, w, res, eps=1e-5)
    assert q is None and s is None and (r is None) == (res is None)
    R = x.double() + (res.double() if res is not None else 0)
    Y = R / torch.sqrt(R.square().mean(1, keepdim=True) + 1e-5) * w.double()
    # r: one fp32 addition and one rounding. y: the addition, the sum of squares (relative error at most (d / 1024 + 40) u32
    # for sums over lanes, warps and a thread's share, halved by the root), four more roundings, and the output's
    rel = (d / 1024 + 60) * U["float32"]
    if res is not None:
        assert bool(((r.double() - R).abs() <= (ulp(r) + U["float32"]) * 1.01 * R.abs() + tiny(r)).all())
    assert bool(((y.double() - Y).abs() <= (ulp(y) * 1.01 + rel) * Y.abs() + tiny(y)).all())


@pytest.mark.parametrize("T,d,x_dt", [(1, 32, "float16"), (7, 96, "float32"), (33, 2560, "bfloat16"), (4, 16416, "float16"), (3, 2080, "float16")])
def test_rms_norm_q8(cuda, T, d, x_dt):
    """The Q8 copy follows vkb_quantize's rule on the unrounded y: half a code step of the exact y, plus the fp16 scale."""
    import torch
    g = gen(d)
    x = torch.randn((T, d), generator=g, device="cuda").to(dt(x_dt))
    x[0, :32] = 0                       # a group of zeros: scale 0, codes 0
    w = torch.ones(d, device="cuda").to(dt(x_dt))
    y, _, q, s = vkb.rms_norm(x, w, q8=True)
    X = x.double()
    Y = X / torch.sqrt(X.square().mean(1, keepdim=True) + 1e-6)
    B = Y.view(T, -1, 32)
    amax = B.abs().amax(-1)
    assert bool(((s.double() - amax / 127).abs() <= amax / 127 * (2.0 ** -11 + 1e-5) + 2.0 ** -24).all())
    assert int(q.view(T, -1, 32)[0, 0].abs().max()) == 0 and float(s[0, 0]) == 0.0
    val = vkb.dequant(vkb.FMT_Q8, q, s, T, d).double().view(T, -1, 32)
    step = s.double()[..., None]
    # half a step from rounding, the clamp at 127 of a scale rounded down (127 u16 steps), the fp16 of the value
    assert bool(((val - B).abs() <= step * (0.5 + 127 * 2.0 ** -11 + 1e-3) + 2.0 ** -11 * B.abs() + 2.0 ** -24).all())


def test_rms_norm_strides_in_place_and_empty(cuda):
    import torch
    g = gen(5)
    wide = torch.randn((6, 300), generator=g, device="cuda").half()
    w = torch.ones(256, device="cuda").half()
    for off in (0, 3):                  # aligned and odd rows of a wider tensor
        x = wide[:, off:off + 256]
        y, *_ = vkb.rms_norm(x, w)
        z, *_ = vkb.rms_norm(x.contiguous(), w)
        assert float((y.double() - z.double()).abs().max()) <= 2 * 2.0 ** -11 * float(z.abs().max())
    res = torch.randn((6, 256), generator=g, device="cuda")
    want_y, want_r, *_ = vkb.rms_norm(wide[:, :256], w, res)
    y, r, *_ = vkb.rms_norm(wide[:, :256], w, res, residual_out=res)
    assert r is res and torch.equal(r, want_r) and torch.equal(y, want_y)
    assert vkb.rms_norm(wide[:0, :256], w)[0].shape == (0, 256)
    big = torch.full((1, 64), float("inf"), device="cuda").half()
    assert bool(torch.isnan(vkb.rms_norm(big, w[:64])[0]).all())       # inf / inf, as the formula says


# ---- the cache -------------------------------------------------------------------------------------------------------

def make_cache(lens, heads, dim, page, seed=1, spare=2):
    """A filled cache whose pages lie in random order, and its values as [seq][len][heads][dim] in 64 bits."""
    import torch
    g = gen(seed)
    per = [-(-n // page) for n in lens]
    total = sum(per) + spare
    code = torch.randn((2, total, heads, page, dim), generator=g, device="cuda").mul_(40).round_().clamp_(-127, 127).add_(128).to(torch.uint8)
    scale = torch.rand((2, total, heads), generator=g, device="cuda") * 0.04 + 0.01
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(1, max(per, default=1))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    cache = vkb.KvCache(code[0].contiguous(), code[1].contiguous(), scale[0].contiguous(), scale[1].contiguous())
    return cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def values(cache, table, b, n):
    import torch
    at = torch.arange(n, device="cuda")
    blk = table[b].long()[at // cache.page]
    return [(c[blk, :, at % cache.page].double() - 128) * s[blk].double()[..., None] for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


def offsets(news):
    import torch
    return torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device="cuda")


def turned(x, pos, turns, layout, mscale=1.0):
    """R(pos) x in 64 bits; the angle from the exact fraction of a turn."""
    import torch
    if turns is None or not pos:
        return x.clone()
    n = turns.numel()
    f = [int(t) % (1 << 64) for t in turns.cpu()]
    ang = torch.tensor([[2 * math.pi * ((int(p) * v) % (1 << 64)) / 2.0 ** 64 for v in f] for p in pos], dtype=torch.float64, device="cuda")
    c, s = (ang.cos() * mscale)[:, None], (ang.sin() * mscale)[:, None]
    out = x.clone()
    a, b = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return out


@pytest.mark.parametrize("lens,news,heads,hq,dim,rot,page,layout,x_dt", [
    ([5], [5], 2, 4, 64, 64, 16, "half", "float16"),
    ([1, 17, 0, 64, 65], [1, 1, 1, 1, 1], 2, 6, 128, 128, 64, "half", "float16"),
    ([40, 3, 0, 130], [40, 2, 0, 7], 3, 3, 80, 40, 32, "interleaved", "bfloat16"),
    ([300, 129], [171, 1], 1, 8, 256, 64, 128, "half", "float32"),
    ([33], [33], 2, 2, 16, 6, 16, "half", "float32"),
    ([33], [20], 2, 2, 48, 10, 16, "interleaved", "float16"),
    ([70, 20], [70, 20], 1, 2, 96, 0, 64, "half", "bfloat16"),
])
def test_rope_append(cuda, lens, news, heads, hq, dim, rot, page, layout, x_dt):
    import torch
    g = gen(sum(lens) + dim)
    cache, table, ln = make_cache(lens, heads, dim, page, seed=dim)
    T = sum(news)
    qkv = (torch.randn((T, hq + 2 * heads, dim), generator=g, device="cuda") * 2).to(dt(x_dt))
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + heads], qkv[:, hq + heads:]
    turns, ms = vkb.rope_turns(rot, scaling="parts", factor=4.0) if rot else (None, 1.0)
    one = all(n == 1 for n in news)
    before = [values(cache, table, b, n) for b, n in enumerate(lens)]
    scales = [cache.k_scale.double().clone(), cache.v_scale.double().clone()]
    out = vkb.rope_append(cache, table, ln, q, k, v, turns=turns, cu=None if one else offsets(news), layout=layout, mscale=ms)
    torch.cuda.synchronize()
    assert vkb.device_status() == 0
    at = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        pos = list(range(n - m, n))
        rows = slice(at, at + m)
        Q, K, V = turned(q[rows].double(), pos, turns, layout, ms), turned(k[rows].double(), pos, turns, layout, ms), v[rows].double()
        big = qkv[rows].double().abs().amax() if m else 0
        # q: cos and sin within 2^-22 (the 32-bit turn, cospi, the factor), two products and a sum, the output's rounding
        assert bool(((out[rows].double() - Q).abs() <= ulp(out) * 1.01 * Q.abs() + 2.0 ** -20 * big + tiny(out)).all())
        at += m
        if not n or not m:
            continue
        have = values(cache, table, b, n)
        for which, (new, held) in enumerate(((K, before[b][0]), (V, before[b][1]))):
            for blk in range((n - m) // page, (n - 1) // page + 1):
                lo, hi = max(n - m, blk * page), min(n, (blk + 1) * page)
                pg = int(table[b, blk])
                x = new[lo - (n - m):hi - (n - m)]                       # [tokens][heads][dim]
                was = scales[which][pg] if lo > blk * page else torch.zeros(heads, dtype=torch.float64, device="cuda")
                s = torch.maximum(was, x.abs().amax((0, 2)) / 127)
                got_s = (cache.k_scale, cache.v_scale)[which][pg].double()
                assert bool(((got_s - s).abs() <= 1e-5 * s).all())
                # half a step, and the fp32 turn's error; codes held before: half a step of the new scale
                got = have[which][lo:hi]
                assert bool(((got - x).abs() <= s[:, None] * 0.5001 + 2.0 ** -20 * big).all())
                old = held[blk * page:lo]
                grown = (s > was * (1 + 1e-6))[None, :, None]
                d = (have[which][blk * page:lo] - old).abs()
                assert bool((d <= torch.where(grown, s[:, None] * 0.5001, torch.zeros_like(d))).all())
    # a second call finds the scales it made: nothing changes
    snap = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    vkb.rope_append(cache, table, ln, q, k, v, turns=turns, cu=None if one else offsets(news), layout=layout, mscale=ms)
    assert all(torch.equal(a, b) for a, b in zip(snap, (cache.k, cache.v, cache.k_scale, cache.v_scale)))


def test_rope_append_positions_in_place_and_specials(cuda):
    import torch
    g = gen(3)
    cache, table, ln = make_cache([4], 1, 64, 16)
    q = torch.randn((4, 2, 64), generator=g, device="cuda")
    k = torch.randn((4, 1, 64), generator=g, device="cuda")
    v = torch.randn((4, 1, 64), generator=g, device="cuda")
    turns, _ = vkb.rope_turns(64)
    pos = torch.tensor([0, 1 << 20, (1 << 31) - 1, -5], dtype=torch.int32, device="cuda")   # angles stay exact far out
    cu = offsets([4])
    want = turned(q.double(), pos.tolist(), turns, "half")
    out = vkb.rope_append(cache, table, ln, q, k, v, turns=turns, cu=cu, pos=pos)
    assert float((out.double() - want).abs().max()) <= 2.0 ** -20 * float(q.abs().max())
    same = q.clone()
    assert vkb.rope_append(cache, table, ln, same, k, v, turns=turns, cu=cu, pos=pos, q_out=same) is same and torch.equal(same, out)
    for rot in (64, 6):                 # in place also where the pairs are not whole vectors
        t2, _ = vkb.rope_turns(rot)
        a = vkb.rope_append(cache, table, ln, q, k, v, turns=t2, cu=cu)
        b = q.clone()
        vkb.rope_append(cache, table, ln, b, k, v, turns=t2, cu=cu, q_out=b)
        assert torch.equal(a, b)
    # infinities saturate and stay out of the scale, NaN is held as zero, zeros make a zero scale
    v2 = v.clone()
    v2[1, 0, 3], v2[2, 0, 5], v2[3, 0, 7] = float("inf"), float("-inf"), float("nan")
    vkb.rope_append(cache, table, ln, None, k * 0, v2, cu=cu)
    kk, vv = values(cache, table, 0, 4)
    s = float(cache.v_scale[int(table[0, 0]), 0])
    finite = torch.where(torch.isfinite(v2), v2, torch.zeros_like(v2))
    assert abs(s - float(finite.abs().max()) / 127) < 1e-6 * s
    assert abs(float(vv[1, 0, 3]) - 127 * s) < 1e-9 and abs(float(vv[2, 0, 5]) + 127 * s) < 1e-9 and float(vv[3, 0, 7]) == 0.0
    assert float(cache.k_scale[int(table[0, 0]), 0]) == 0.0 and float(kk.abs().max()) == 0.0
    # an empty call, and rows that belong to no sequence's span
    assert vkb.rope_append(cache, table, ln, q[:0], k[:0], v[:0], cu=offsets([0])).shape == (0, 2, 64)


def test_bad_indices_are_reported(cuda):
    """Lengths, offsets and pages outside their arrays: skipped, bit 16 of the device status, no fault."""
    import torch
    cache, table, ln = make_cache([20, 20], 1, 64, 16)
    q = torch.zeros((2, 1, 64), device="cuda").half()
    work = vkb.attention_workspace(cache)
    bad = table.clone()
    bad[1, 1] = 1 << 20
    vkb.rope_append(cache, bad, ln, q, q, q)
    assert vkb.device_status() == 16
    vkb.attention(cache, bad, ln, q, work=work)
    assert vkb.device_status() == 16
    vkb.attention(cache, table, ln + 1000, q, work=work)
    assert vkb.device_status() == 16
    many = torch.zeros((2 * 40, 4, 64), device="cuda").half()
    vkb.attention(cache, bad, ln, many, cu=offsets([40, 40]), work=work)
    assert vkb.device_status() == 16
    wide = torch.zeros((2 * 40, 64, 64), device="cuda").half()
    vkb.attention(cache, bad, ln, wide, cu=offsets([40, 40]), work=work)
    assert vkb.device_status() == 16
    k, v = vkb.kv_read(cache, table, torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.tensor([99, 0], dtype=torch.int32, device="cuda"))
    assert float(k.abs().max()) == 0.0 and vkb.device_status() == 16
    out = vkb.attention(cache, table, ln, q, work=work)      # and the workspace is ready for the next call
    torch.cuda.synchronize()
    assert vkb.device_status() == 0 and bool(torch.isfinite(out).all())


# ---- attention -------------------------------------------------------------------------------------------------------

def attention_ref(cache, table, lens, news, q, window=0, scale=None):
    """(o, error bound) in 64 bits. The kernels round p once to fp16 (relative 2^-11) and sum in fp32; a score's fp32 sum of dim
    products has an error of at most 2 dim u32 (the tensor cores truncate) times the sum of its terms' magnitudes, which
    moves p by that factor, twice (in the sum of p too); 2^-21 covers the exponential and the scale's logarithm."""
    import torch
    T, hq, dim = q.shape
    grp = hq // cache.heads
    scale = dim ** -0.5 if scale is None else scale
    o = torch.zeros((T, hq, dim), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    at = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        if n and m:
            k, v = values(cache, table, b, n)
            pos = torch.arange(n - m, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            seen = (j <= pos) & (j > pos - window if window else j >= 0)
            for h in range(hq):
                x, kh, vh = q[at:at + m, h].double(), k[:, h // grp], v[:, h // grp]
                s = (x @ kh.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)
                o[at:at + m, h] = p @ vh
                terms = (x.abs() @ kh.abs().T * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                tol[at:at + m, h] = (p @ vh.abs()) * (2.0 ** -11 + 2 * terms * 2 * dim * 2.0 ** -24 + 2.0 ** -21 * 8)
        at += m
    u = U[str(q.dtype).split(".")[1]]
    return o, tol * (1 + u) + o.abs() * u * 1.01 + 1e-6


def check_attention(cache, table, lens, news, q, window=0, scale=None, cu="auto", work=None):
    import torch
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    one = all(n == 1 for n in news)
    out = vkb.attention(cache, table, ln, q, cu=None if one and cu == "auto" else offsets(news), window=window, scale=scale, work=work)
    torch.cuda.synchronize()
    assert vkb.device_status() == 0
    o, tol = attention_ref(cache, table, lens, news, q, window, scale)
    bad = (out.double() - o).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float((out.double() - o).abs().max()))
    return out


CASES = [   # lens, news, kv heads, q heads, dim, page, window
    ([1], [1], 1, 1, 64, 16, 0),
    ([63, 64, 65, 0, 1, 777], [1] * 6, 2, 8, 128, 64, 0),
    ([129, 2, 16, 17], [1] * 4, 2, 14, 256, 16, 0),
    ([300, 45], [1, 1], 1, 16, 64, 32, 7),            # 16 rows
    ([300, 45, 5], [5, 3, 5], 4, 4, 80, 128, 0),      # dimension inside a padded tile
    ([200, 90], [6, 2], 2, 10, 128, 32, 33),          # 30 rows
    ([257], [9], 3, 9, 192, 64, 0),                   # 27 rows: prompt kernel at dimension 256
    ([40, 500, 0, 64], [40, 130, 0, 1], 2, 8, 128, 16, 0),
    ([333, 70], [333, 64], 2, 16, 256, 32, 50),
    ([260, 1, 2], [200, 1, 2], 1, 71, 64, 64, 0),     # 71 heads on one
    ([129], [129], 2, 2, 96, 128, 1),                 # a window of one: its own value
    ([100, 30], [130, 30], 1, 8, 48, 16, 0),          # more new tokens than the sequence is long: the first rows see nothing
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("x_dt", ["float16", "bfloat16"])
def test_attention(cuda, case, x_dt):
    import torch
    lens, news, heads, hq, dim, page, window = case
    cache, table, _ = make_cache(lens, heads, dim, page, seed=dim + hq)
    q = (torch.randn((sum(news), hq + 2, dim), generator=gen(7), device="cuda") * 1.5).to(dt(x_dt))[:, 1:hq + 1]   # strided rows
    first = check_attention(cache, table, lens, news, q, window)
    assert torch.equal(first, check_attention(cache, table, lens, news, q, window))      # the order of arrival does not matter


PROMPTS = [   # enough query rows for the prompt kernel at every dimension: lens, news, kv heads, q heads, dim, page, window
    ([300], [300], 2, 16, 128, 64, 0),
    ([520, 0, 129, 64], [190, 0, 129, 1], 2, 24, 128, 16, 0),
    ([700, 33], [260, 33], 1, 20, 96, 128, 100),
    ([257, 400], [257, 90], 4, 16, 112, 32, 0),
    ([200], [200], 3, 39, 48, 16, 65),
    ([1030, 5, 64], [500, 5, 64], 1, 16, 64, 64, 0),
    ([600], [129], 1, 37, 192, 32, 0),
    ([700], [290], 2, 16, 256, 128, 300),
    ([1500, 1], [130, 1], 2, 64, 240, 16, 1),
    ([150, 100], [170, 100], 2, 32, 128, 64, 0),      # more new tokens than the sequence is long
]


@pytest.mark.parametrize("case", PROMPTS, ids=[str(i) for i in range(len(PROMPTS))])
@pytest.mark.parametrize("x_dt", ["float16", "bfloat16"])
def test_attention_prompts(cuda, case, x_dt):
    import torch
    lens, news, heads, hq, dim, page, window = case
    assert sum(news) * hq > 4096
    cache, table, _ = make_cache(lens, heads, dim, page, seed=dim + hq)
    q = (torch.randn((sum(news), hq + 2, dim), generator=gen(7), device="cuda") * 1.5).to(dt(x_dt))[:, 1:hq + 1]
    work = vkb.attention_workspace(cache)
    first = check_attention(cache, table, lens, news, q, window, work=work)
    assert torch.equal(first, check_attention(cache, table, lens, news, q, window, work=work))


def test_attention_prompt_scales_and_nan(cuda):
    """test_attention_scales' pages and a NaN row, with enough q heads for the prompt kernel."""
    import torch
    lens, news = [400, 150], [120, 150]
    cache, table, ln = make_cache(lens, 2, 64, 16, seed=3)
    for page_at, k, v in ((3, 1.0, 0.0), (5, 0.0, 1.0), (7, 1.0, 1e4), (8, 1.0, 1e-5), (11, 30.0, 1.0)):
        pg = table[0, page_at].long()
        cache.k_scale[pg] *= k
        cache.v_scale[pg] *= v
        if k == 0.0:
            cache.k[pg] = 128
        if v == 0.0:
            cache.v[pg] = 128
    cache.v_scale[table[1, 0].long()] = 0.0
    cache.v[table[1, 0].long()] = 128
    for mag in (1e-3, 1.0, 30.0):
        q = (torch.randn((270, 32, 64), generator=gen(2), device="cuda") * mag).to(torch.bfloat16)
        check_attention(cache, table, lens, news, q)
        check_attention(cache, table, lens, news, q.half(), scale=0.03)
    q = q.half() * 0.02
    cu = offsets(news)
    want = vkb.attention(cache, table, ln, q, cu=cu)
    q[130, 17, 5] = float("nan")
    out = vkb.attention(cache, table, ln, q, cu=cu)
    keep = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    keep[130, 17] = False
    assert bool(torch.isnan(out[130, 17]).all()) and bool(torch.isfinite(out[keep]).all())
    assert float((out[keep].double() - want[keep].double()).abs().max()) <= 2.0 ** -9 * float(want.abs().max())
    cache.v_scale.zero_()
    cache.v.fill_(128)
    q[130, 17, 5] = 0.0
    assert float(check_attention(cache, table, lens, news, q).abs().max()) == 0.0


@pytest.mark.parametrize("n_new", [1, 3, 64])
def test_attention_scales(cuda, n_new):
    """Pages whose scales are zero, tiny or huge beside one another, sharp and flat scores, q of large and small magnitude."""
    import torch
    lens, news = [400, 150], [n_new, n_new]
    cache, table, _ = make_cache(lens, 2, 64, 16, seed=3)
    cache.v_scale[table[0, 3].long()] = 0.0
    cache.v[table[0, 3].long()] = 128
    cache.k_scale[table[0, 5].long()] = 0.0
    cache.k[table[0, 5].long()] = 128
    cache.v_scale[table[0, 7].long()] *= 1e4
    cache.v_scale[table[0, 8].long()] *= 1e-5
    cache.v_scale[table[1, 0].long()] = 0.0           # the first page of a sequence
    cache.v[table[1, 0].long()] = 128
    cache.k_scale[table[0, 11].long()] *= 30          # one page takes nearly all the weight of rows that like it
    for mag in (1e-3, 1.0, 30.0):
        q = (torch.randn((2 * n_new, 4, 64), generator=gen(n_new), device="cuda") * mag).to(torch.bfloat16)
        check_attention(cache, table, lens, news, q)
        check_attention(cache, table, lens, news, q.half(), scale=0.03)
    cache.v_scale.zero_()
    cache.v.fill_(128)
    out = check_attention(cache, table, lens, news, q)
    assert float(out.abs().max()) == 0.0


def test_attention_nan_stays_in_its_row(cuda):
    import torch
    for n_new in (1, 40):
        cache, table, ln = make_cache([100, 90], 1, 64, 16)
        q = torch.randn((2 * n_new, 4, 64), generator=gen(1), device="cuda").half()
        cu = offsets([n_new, n_new])
        want = vkb.attention(cache, table, ln, q, cu=cu)
        q[1, 2, 5] = float("nan")
        out = vkb.attention(cache, table, ln, q, cu=cu)
        assert bool(torch.isnan(out[1, 2]).all())
        keep = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
        keep[1, 2] = False
        assert bool(torch.isfinite(out[keep]).all())
        # a NaN row makes its tile look for new maxima: other rows of it may round p differently
        assert float((out[keep].double() - want[keep].double()).abs().max()) <= 2.0 ** -9 * float(want.abs().max())


def test_attention_many_sequences_and_long_tables(cuda):
    """More sequences than a block has threads (the division of the work scans them in turns), tables with unused tails."""
    import torch
    r = np.random.default_rng(4)
    lens = [int(x) for x in r.integers(0, 90, 1500)]
    cache, table, _ = make_cache(lens, 1, 64, 32, seed=8)
    wide = torch.full((len(lens), 64), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = torch.randn((len(lens), 2, 64), generator=gen(2), device="cuda").half()
    check_attention(cache, wide, lens, [1] * len(lens), q)


def test_attention_offsets_past_32_bits(cuda):
    """A cache of more than 4 GB per tensor: sequences in its last pages, by every kernel."""
    import torch
    heads, dim, page = 8, 128, 128
    pages = (5 << 30) // (heads * dim * page)
    k = torch.empty((pages, heads, page, dim), dtype=torch.uint8, device="cuda")
    v = torch.empty_like(k)
    g = gen(9)
    for t in (k, v):
        t[-6:] = torch.randint(1, 256, t[-6:].shape, generator=g, device="cuda", dtype=torch.uint8)
    s = torch.rand((2, pages, heads), generator=g, device="cuda") * 0.02 + 0.01
    cache = vkb.KvCache(k, v, s[0].contiguous(), s[1].contiguous())
    table = torch.tensor([[pages - 1, pages - 4], [pages - 2, pages - 6]], dtype=torch.int32, device="cuda")
    lens = [200, 131]
    for news in ([1, 1], [4, 3], [90, 60], [200, 131]):
        T = sum(news)
        q = torch.randn((T, 16, dim), generator=g, device="cuda").half()
        kn = torch.randn((T, heads, dim), generator=g, device="cuda").half()
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        vkb.rope_append(cache, table, ln, None, kn, kn, cu=offsets(news))
        kk, _ = vkb.kv_read(cache, table, torch.zeros(news[0], dtype=torch.int32, device="cuda"),
                            torch.arange(lens[0] - news[0], lens[0], dtype=torch.int32, device="cuda"))
        assert float((kk.double() - kn[:news[0]].double()).abs().max()) <= float(cache.k_scale[table.long()].max())
        check_attention(cache, table, lens, news, q)


def test_attention_streams_graphs_and_growth(cuda):
    """A call on another stream than the current one, and a captured step replayed while its sequences grow (lengths and
    table are read on the device)."""
    import torch
    heads, hq, dim, page = 2, 8, 128, 16
    g = gen(6)
    lens = [5, 30, 0]
    cache, table, ln = make_cache([90, 90, 90], heads, dim, page)
    qkv = torch.randn((3, hq + 2 * heads, dim), generator=g, device="cuda").half()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + heads], qkv[:, hq + heads:]
    turns, _ = vkb.rope_turns(dim)
    work, out, qr = vkb.attention_workspace(cache), torch.empty((3, hq, dim), dtype=torch.float16, device="cuda"), torch.empty((3, hq, dim), dtype=torch.float16, device="cuda")
    ln.copy_(torch.tensor(lens, dtype=torch.int32))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    a = vkb.attention(cache, table, ln, q, work=work, stream=other)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(a, vkb.attention(cache, table, ln, q, work=work))

    def step():
        vkb.rope_append(cache, table, ln, q, k, v, turns=turns, q_out=qr)
        vkb.attention(cache, table, ln, qr, out=out, work=work)
    step()
    torch.cuda.synchronize()
    graph = vkb.Graph()
    with graph:
        step()
    for n in range(1, 40):
        lens = [5 + n, 30 + n, n // 2]
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        if n % 13 == 0:
            o, tol = attention_ref(cache, table, lens, [1, 1, 1], qr)
            assert not bool(((out.double() - o).abs() > tol).any()), n
    assert vkb.device_status() == 0
    del graph


def test_tensors_of_another_stream(cuda):
    """A call on another stream marks its tensors as used there: memory given back at once is not handed out again while
    the call still waits for that stream's earlier work."""
    import torch
    x = torch.randn((4096, 2048), generator=gen(2), device="cuda").half()
    w = torch.ones(2048, device="cuda").half()
    want = vkb.rms_norm(x, w)[0]
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        a = torch.randn((4096, 4096), device="cuda")
        for _ in range(20):
            a = a @ a * 1e-3
    y = vkb.rms_norm(x, w, stream=other)[0]
    ptr = x.data_ptr()
    del x
    z = torch.zeros((4096, 2048), dtype=torch.float16, device="cuda")
    assert z.data_ptr() != ptr
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_attention_refusals(cuda):
    import torch
    cache, table, ln = make_cache([10], 2, 64, 16)
    q = torch.zeros((1, 4, 64), device="cuda").half()
    for kw, what in ((dict(q=q.float()), "fp16 or bf16"), (dict(q=q[:, :3]), "multiple"), (dict(q=torch.zeros((2, 4, 64), device="cuda").half()), "one row per"),
                     (dict(q=q.transpose(1, 2)), "multiple|adjacent"), (dict(ln=ln.long()), "lens"), (dict(table=table.long()), "table"),
                     (dict(cu=torch.zeros(1, dtype=torch.int32, device="cuda")), "cu"), (dict(work=torch.zeros(64, dtype=torch.uint8, device="cuda")), "invalid argument")):
        a = dict(q=q, ln=ln, table=table, cu=None, work=None)
        a.update(kw)
        with pytest.raises(vkb.VkbError, match=what):
            vkb.attention(cache, a["table"], a["ln"], a["q"], cu=a["cu"], work=a["work"])
    odd = torch.zeros(1, 260, device="cuda").half()[:, 2:258].unflatten(1, (4, 64))
    with pytest.raises(vkb.VkbError):       # rows that are not 16-byte aligned
        vkb.attention(cache, table, ln, odd)


# ---- sampling --------------------------------------------------------------------------------------------------------

def sample_ref(z, t, k, p, m):
    """(order-statistics in 64 bits) weights of the kept tokens in index order, or the one greedy token."""
    import torch
    z = z.double()
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    zs, order = z.sort(descending=True, stable=True)
    if float(zs[0]) == -math.inf:
        return None, -1
    if not t > 0 or k == 1 or p <= 0:
        return None, int(order[0])
    w = torch.where(zs == zs[0], torch.ones_like(zs), ((zs - zs[0]) / t).exp())
    if 0 < k < w.numel():
        w[k:] = 0
    keep = (w.cumsum(0) - w) < p * w.sum() if p < 1 else torch.ones_like(w, dtype=torch.bool)
    keep &= w >= min(m, 1.0)
    keep[0] = True
    full = torch.zeros_like(w)
    full[order] = torch.where(keep, w, torch.zeros_like(w))
    return full, None


def check_sample(x, t, k, p, m, u):
    """The token's stretch of the distribution holds u, within 4e-6 of the mass (the weights' fp32 exponents of up to 46 u32,
    sums in fp32 of thousands of terms by warps), which is also the error that may move the top-p boundary by a token."""
    import torch
    B = x.shape[0]
    f = lambda v, d: torch.tensor(v, dtype=d, device="cuda")  # noqa: E731
    args = (f(u, torch.float32), f(t, torch.float32), f(k, torch.int32), f(p, torch.float32), f(m, torch.float32))
    tok, prob = vkb.sample(x, *args)
    again = vkb.sample(x, *args)
    assert torch.equal(tok, again[0]) and torch.equal(prob, again[1])
    for b in range(B):
        full, one = sample_ref(x[b], float(args[1][b]), k[b], float(args[3][b]), float(args[4][b]))   # the fp32 settings it got
        i = int(tok[b])
        if one is not None:
            assert i == one and float(prob[b]) == (0.0 if one < 0 else 1.0), (b, i, one)
            continue
        c = full.cumsum(0)
        total = float(c[-1])
        w, hi = float(full[i]) / total, float(c[i]) / total
        uu = float(args[0][b])
        assert w > 0 and hi - w - 4e-6 <= uu <= hi + 4e-6, (b, i, hi - w, hi, uu)
        assert abs(float(prob[b]) - w) <= 4e-6 + 2e-5 * w, (b, float(prob[b]), w)


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4097, 8200, 32000, 151936])
@pytest.mark.parametrize("x_dt", ["float16", "bfloat16", "float32"])
def test_sample(cuda, V, x_dt):
    import torch
    g, r = gen(V), np.random.default_rng(V)
    B = 12
    x = (torch.randn((B, V), generator=g, device="cuda") * torch.linspace(0.5, 5, B, device="cuda")[:, None]).to(dt(x_dt))
    x[torch.rand((B, V), generator=g, device="cuda") < 0.1] = float("-inf")
    x[3, V // 2] = float("nan")
    x[4] = float("-inf")
    x[5, -1] = float("inf")
    check_sample(x, [float(v) for v in r.choice([0.0, 0.3, 1.0, 2.0], B)], [int(v) for v in r.choice([0, 1, 2, 40, 1000, 3000], B)],
                 [float(v) for v in r.choice([0.0, 0.3, 0.9, 1.0], B)], [float(v) for v in r.choice([0.0, 0.1], B)],
                 [float(v) for v in r.random(B).astype(np.float32)])


@pytest.mark.parametrize("V,k,p", [(5000, 1500, 1.0), (5000, 0, 0.37), (60000, 30001, 0.5), (60000, 0, 0.999), (200000, 2000, 0.9)])
def test_sample_ties_and_crowded_bins(cuda, V, k, p):
    """Equal logits are cut by index; thousands of different logits within one bin of the first histogram are split by their
    bits. One far outlier keeps the bins wide."""
    import torch
    g = gen(V + k)
    flat = torch.zeros((3, V), device="cuda")
    flat[1] = torch.randint(0, 3, (V,), generator=g, device="cuda").float()
    flat[2] = torch.randn(V, generator=g, device="cuda") * 1e-4
    flat[2, 7] = 20.0
    for u in (0.0, 0.5, 0.99999):
        check_sample(flat, [1.0, 1.0, 50.0], [k] * 3, [p] * 3, [0.0] * 3, [u] * 3)


def test_sample_strides_and_defaults(cuda):
    import torch
    g = gen(1)
    x = torch.randn((4, 1003), generator=g, device="cuda").half()
    u = torch.rand(4, generator=g, device="cuda")
    a = vkb.sample(x[:, 1:1001], u)
    b = vkb.sample(x[:, 1:1001].contiguous(), u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    tok = torch.empty(4, dtype=torch.int32, device="cuda")
    assert vkb.sample(x, u, token=tok)[0] is tok
    assert vkb.sample(x[:0], u[:0])[0].shape == (0,)
    assert vkb.lib().vkb_sample(0, x.data_ptr(), 400000, 1, 400000, None, None, None, None, u.data_ptr(), tok.data_ptr(), None, None) == vkb.EUNSUPPORTED
