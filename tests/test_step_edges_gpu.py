"""Edge cases of the decode-step operators on the GPU. Helpers and the derivation of the tolerances: test_step_gpu.py."""
import math

import pytest

import vkb
from test_step_gpu import U, check_attention, dt, gen, make_cache, offsets, turned, values

pytestmark = pytest.mark.gpu


# ---- V scales that grow within a segment ------------------------------------------------------------------------------

def quiet_pages(cache, table, b, first, last, scale):
    """The pages of tokens [first, last) of sequence b get V scale `scale` (0: codes of zero too)."""
    for pg in table[b, first // cache.page:-(-last // cache.page)].long().tolist():
        cache.v_scale[pg] = scale
        if scale == 0.0:
            cache.v[pg] = 128


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 128), (256, 32), (256, 128)])
@pytest.mark.parametrize("quiet", [64, 128, 576])
@pytest.mark.parametrize("scale", [0.01, 0.06, 1.0, 50.0])
def test_first_keys_without_values(cuda, dim, page, quiet, scale):
    """Keys whose V scale is 0 keep their weight, also where they fill the first tiles that a block reads."""
    import torch
    lens, news = [quiet + 700, quiet + 90], [200, 80]
    cache, table, _ = make_cache(lens, 1, dim, page, seed=dim + page)
    cache.v_scale[:] = scale
    for b in range(2):
        quiet_pages(cache, table, b, 0, quiet, 0.0)
    q = (torch.randn((280, 16, dim), generator=gen(quiet), device="cuda") * 1.5).half()
    check_attention(cache, table, lens, news, q)                                      # many rows
    check_attention(cache, table, lens, [1, 1], q[:2])                                # a token each


def come_and_go(dim, low, high):
    """A sequence of 6000 keys with stretches of 512 of V scale `low` and of `high` in turn."""
    cache, table, ln = make_cache([6000], 1, dim, 64, seed=dim)
    cache.v_scale[:] = high
    for at in range(0, 6000, 1024):
        quiet_pages(cache, table, 0, at, min(6000, at + 512), low)
    return cache, table, ln


@pytest.mark.parametrize("low,high,x_dt", [(0.0, 0.1, "float16"), (0.0, 1.0, "bfloat16"), (1e-30, 1.0, "float16"), (1e-9, 1.0, "bfloat16")])
@pytest.mark.parametrize("dim", [128, 256])
def test_values_that_come_and_go(cuda, low, high, x_dt, dim):
    """Blocks that take parts of an item start in stretches of either kind."""
    import torch
    cache, table, _ = come_and_go(dim, low, high)
    q = (torch.randn((300, 16, dim), generator=gen(dim), device="cuda") * 1.5).to(dt(x_dt))
    check_attention(cache, table, [6000], [300], q)
    check_attention(cache, table, [6000], [1], q[:1])


@pytest.mark.parametrize("low", [0.0, 1e-9, 0.2])
@pytest.mark.parametrize("new", [1, 300])
def test_outputs_follow_the_v_scales(cuda, low, new):
    """V scales times a power of two: the outputs times that power, exactly (bf16 holds them all)."""
    import torch
    cache, table, ln = come_and_go(128, low, 30.0)
    q = (torch.randn((new, 16, 128), generator=gen(new), device="cuda") * 1.5).to(torch.bfloat16)
    cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    want = vkb.attention(cache, table, ln, q, cu=cu)
    for k in (-5, 3, 60):
        cache.v_scale *= 2.0 ** k
        assert torch.equal(vkb.attention(cache, table, ln, q, cu=cu), want * 2.0 ** k), k
        cache.v_scale *= 2.0 ** -k


# ---- pages that do not exist ------------------------------------------------------------------------------------------

def masked_ref(cache, table, lens, news, q, gone, window=0):
    """attention_ref() without the keys of the pages `gone` [(sequence, page of it)]: their weight set to zero."""
    import torch
    fixed = table.clone()
    for b, i in gone:
        fixed[b, i] = int(table[b, 0]) if int(table[b, 0]) >= 0 else 0
    o, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at, grp = 0, q.shape[1] // cache.heads
    for b, (n, m) in enumerate(zip(lens, news)):
        k, v = values(cache, fixed, b, n)
        pos, j = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = (j <= pos) & (j > pos - window if window else j >= 0)
        for x, i in gone:
            if x == b:
                seen = seen & ~((j >= i * cache.page) & (j < (i + 1) * cache.page))
        for h in range(q.shape[1]):
            x, kh, vh = q[at:at + m, h].double(), k[:, h // grp], v[:, h // grp]
            s = (x @ kh.T * cache.dim ** -0.5).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            o[at:at + m, h] = p @ vh
            terms = (x.abs() @ kh.abs().T * cache.dim ** -0.5).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            tol[at:at + m, h] = (p @ vh.abs()) * (2.0 ** -11 + 2 * terms * 2 * cache.dim * 2.0 ** -24 + 2.0 ** -21 * 8)
        at += m
    u = U[str(q.dtype).split(".")[1]]
    return o, tol * (1 + u) + o.abs() * u * 1.01 + 1e-6


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (128, 64), (256, 128), (80, 16)])
@pytest.mark.parametrize("new", [1, 4, 150])
@pytest.mark.parametrize("bad", [-1, 1 << 20, None])
def test_keys_of_pages_outside_the_cache_are_left_out(cuda, dim, page, new, bad):
    """They take no weight (a page index that does not exist: bit 16), whatever page 0 holds."""
    import torch
    lens, news = [520, 300], [new, new]
    cache, table, ln = make_cache(lens, 1, dim, page, seed=page)
    unused = sorted(set(range(cache.pages)) - set(table[table >= 0].tolist()))[0]
    table[table == 0] = unused                      # page 0: no sequence's, loud
    cache.k_scale[0], cache.v_scale[0] = 3.0, 1000.0
    gone = [(0, 0), (0, 2), (1, 1)]
    table2 = table.clone()
    for b, i in gone:
        table2[b, i] = cache.pages if bad is None else bad
    q = (torch.randn((2 * new, 16, dim), generator=gen(new), device="cuda")).half()
    out = vkb.attention(cache, table2, ln, q, cu=offsets(news))
    torch.cuda.synchronize()
    assert vkb.device_status() == 16
    o, tol = masked_ref(cache, table, lens, news, q, gone)
    assert not bool(((out.double() - o).abs() > tol).any()), float((out.double() - o).abs().max())
    table2[1] = -1                                   # a sequence without any page: zeros
    out = vkb.attention(cache, table2, ln, q, cu=offsets(news))
    assert float(out[new:].abs().max()) == 0.0 and bool(torch.isfinite(out).all()) and vkb.device_status() == 16


@pytest.mark.parametrize("new", [1, 5, 150])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_pages_behind_the_window_may_be_given_back(cuda, new, page):
    """Pages that no row of the call sees are not looked at: a caller may take them out of the table."""
    import torch
    lens, news, window = [1003, 700], [new, new], 77
    cache, table, ln = make_cache(lens, 2, 128, page)
    q = torch.randn((2 * new, 32, 128), generator=gen(new), device="cuda").half()
    want = vkb.attention(cache, table, ln, q, cu=offsets(news), window=window)
    for b, n in enumerate(lens):
        table[b, :max(0, n - new - window + 1) // page] = -1
    out = vkb.attention(cache, table, ln, q, cu=offsets(news), window=window)
    assert vkb.device_status() == 0 and torch.equal(out, want)


# ---- rows of no sequence ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("with_pos", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_append_leaves_rows_of_no_sequence(cuda, with_pos, layout):
    import torch
    g = gen(1)
    cache, table, _ = make_cache([20, 30, 9], 1, 64, 16)
    ln = torch.tensor([20, 1000, 9], dtype=torch.int32, device="cuda")     # the second is longer than its table
    cu = torch.tensor([1, 4, 6, 9], dtype=torch.int32, device="cuda")      # rows 0 and 9.. are nobody's
    q, k, v = (torch.randn((12, h, 64), generator=g, device="cuda") for h in (2, 1, 1))
    turns, _ = vkb.rope_turns(64)
    pos = torch.arange(100, 112, dtype=torch.int32, device="cuda") if with_pos else None
    out = torch.full_like(q, 7.0)
    vkb.rope_append(cache, table, ln, q, k, v, turns=turns, cu=cu, pos=pos, layout=layout, q_out=out)
    assert vkb.device_status() == 16
    same = q.clone()
    vkb.rope_append(cache, table, ln, same, k, v, turns=turns, cu=cu, pos=pos, layout=layout, q_out=same)
    assert vkb.device_status() == 16
    mine = [1, 2, 3, 6, 7, 8]
    rest = [i for i in range(12) if i not in mine]
    assert bool((out[rest] == 7.0).all()) and torch.equal(same[rest], q[rest]) and torch.equal(same[mine], out[mine])
    at = pos[mine].tolist() if with_pos else [17, 18, 19, 6, 7, 8]
    want = turned(q[mine].double(), at, turns, layout)
    assert float((out[mine].double() - want).abs().max()) <= 2.0 ** -20 * float(q.abs().max())


# ---- windows and counts near 2^31 -------------------------------------------------------------------------------------

@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 20])
@pytest.mark.parametrize("lens,news,hq", [([3], [30], 1), ([100, 30], [170, 90], 32)])
def test_window_wider_than_any_sequence(cuda, window, lens, news, hq):
    """With more new tokens than the sequence is long, the first rows lie before position 0."""
    import torch
    cache, table, _ = make_cache(lens, 1, 64, 16)
    q = torch.randn((sum(news), hq, 64), generator=gen(2), device="cuda").half()
    out = check_attention(cache, table, lens, news, q, window)
    assert torch.equal(out, check_attention(cache, table, lens, news, q, 0))


def test_lengths_near_2_31(cuda):
    """A table of 2^31 tokens, all of them in a few pages: the longest length works, a longer one is left out."""
    import torch
    page, longest = 128, (1 << 31) - 4096
    cache, _, _ = make_cache([3 * page], 1, 64, page, spare=0)
    table = torch.full((1, (1 << 31) // page), 0, dtype=torch.int32, device="cuda")
    at = (longest - 1) // page
    table[0, at - 1], table[0, at] = 1, 2
    g = gen(5)
    q, k, v = (torch.randn((2, h, 64), generator=g, device="cuda").half() for h in (4, 1, 1))
    cu, ln = offsets([2]), torch.tensor([longest], dtype=torch.int32, device="cuda")
    held = cache.k[:2].clone()
    vkb.rope_append(cache, table, ln, None, k, v, cu=cu)
    seq, pos = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([longest - 2, longest - 1], dtype=torch.int32, device="cuda")
    kk, _ = vkb.kv_read(cache, table, seq, pos)
    assert float((kk.double() - k.double()).abs().max()) <= float(cache.k_scale[2, 0])
    out = vkb.attention(cache, table, ln, q, cu=cu, window=200)
    short = torch.tensor([[1, 2]], dtype=torch.int32, device="cuda")       # the same two pages as a short sequence
    want = vkb.attention(cache, short, torch.tensor([2 * page], dtype=torch.int32, device="cuda"), q, cu=cu, window=200)
    assert vkb.device_status() == 0 and torch.equal(out, want) and torch.equal(cache.k[:2], held)
    snap = cache.k.clone()
    for n in (longest + 1, (1 << 31) - 1):
        ln.fill_(n)
        vkb.rope_append(cache, table, ln, None, k, v, cu=cu)
        assert vkb.device_status() == 16 and torch.equal(cache.k, snap)
        vkb.attention(cache, table, ln, q, cu=cu, window=200)
        assert vkb.device_status() == 16


@pytest.mark.parametrize("T,hq,tile", [(16, 32, 8), (16, 256, 32), (64, 512, 256)])     # the last: the prompt kernel
def test_overlapping_spans_of_more_units_than_the_division_holds(cuda, T, hq, tile):
    """Offsets 0, T, 0, T, ..: every second sequence has all rows, and their units in all pass 2^31. The call is left out."""
    import torch
    B, page = 1024, 128
    cache, _, _ = make_cache([page], 8, 64, page, spare=0)
    table = torch.zeros((B, 65536), dtype=torch.int32, device="cuda")
    ln = torch.full((B,), 65536 * page // 2, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, T] * (B // 2) + [0], dtype=torch.int32, device="cuda")
    q, out = torch.zeros((T, hq, 64), device="cuda").half(), torch.full((T, hq, 64), 7.0, device="cuda").half()
    assert B // 2 * 8 * -(-T * hq // 8 // tile) * (int(ln[0]) // 64 + 16) >= (1 << 31) - 1
    vkb.attention(cache, table, ln, q, cu=cu, out=out)
    assert vkb.device_status() == 16 and bool((out == 7.0).all())
    check_attention(cache, table[:2, :1].contiguous(), [100, 128], [1, 1], q[:2])        # the next call is right


def test_offsets_that_decrease(cuda):
    import torch
    cache, table, ln = make_cache([40, 40, 40], 1, 64, 16)
    for hq in (4, 128):
        q = torch.randn((40, hq, 64), generator=gen(3), device="cuda").half()
        out = torch.full_like(q, 7.0)
        vkb.attention(cache, table, ln, q, cu=torch.tensor([0, 30, 10, 40], dtype=torch.int32, device="cuda"), out=out)
        assert vkb.device_status() == 16 and bool((out == 7.0).all())
        check_attention(cache, table, [40, 40, 40], [10, 5, 25], q)


# ---- refusals ---------------------------------------------------------------------------------------------------------

def test_arguments_that_are_no_tensors_are_refused(cuda):
    """None where an argument must be given, plain numbers in the place of arrays, windows that a C int does not hold."""
    import torch
    cache, table, ln = make_cache([20, 20], 1, 64, 16)
    x, w = torch.zeros((2, 64), device="cuda"), torch.ones(64, device="cuda")
    q, u = torch.zeros((2, 1, 64), device="cuda").half(), torch.zeros(2, device="cuda")
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    for name, call in (
            ("weight", lambda: vkb.rms_norm(x, None)), ("residual", lambda: vkb.rms_norm(x, w, 1.0)), ("y", lambda: vkb.rms_norm(x, w, y=0)),
            ("residual_out", lambda: vkb.rms_norm(x, w, x, residual_out=0)),
            ("k", lambda: vkb.rope_append(cache, table, ln, q, None, q)), ("v", lambda: vkb.rope_append(cache, table, ln, q, q, None)),
            ("q", lambda: vkb.rope_append(cache, table, ln, 1, q, q)), ("table", lambda: vkb.rope_append(cache, None, ln, q, q, q)),
            ("lens", lambda: vkb.rope_append(cache, table, None, q, q, q)), ("turns", lambda: vkb.rope_append(cache, table, ln, q, q, q, turns=64)),
            ("turns", lambda: vkb.rope_append(cache, table, ln, q, q, q, turns=torch.tensor(5, device="cuda"))),
            ("pos", lambda: vkb.rope_append(cache, table, ln, q, q, q, pos=3)), ("q_out", lambda: vkb.rope_append(cache, table, ln, q, q, q, q_out=3)),
            ("cache", lambda: vkb.rope_append(None, table, ln, q, q, q)), ("cache", lambda: vkb.kv_read(None, table, i32, i32)),
            ("seq", lambda: vkb.kv_read(cache, table, None, i32)), ("pos", lambda: vkb.kv_read(cache, table, i32, None)),
            ("table", lambda: vkb.kv_read(cache, None, i32, i32)),
            ("q", lambda: vkb.attention(cache, table, ln, None)), ("table", lambda: vkb.attention(cache, None, ln, q)),
            ("lens", lambda: vkb.attention(cache, table, None, q)), ("cu", lambda: vkb.attention(cache, table, ln, q, cu=[0, 1, 2])),
            ("out", lambda: vkb.attention(cache, table, ln, q, out=0)), ("work", lambda: vkb.attention(cache, table, ln, q, work=4096)),
            ("window", lambda: vkb.attention(cache, table, ln, q, window=(1 << 32) + 5)), ("window", lambda: vkb.attention(cache, table, ln, q, window=-1)),
            ("u", lambda: vkb.sample(x, None)), ("top_k", lambda: vkb.sample(x, u, top_k=40)), ("temperature", lambda: vkb.sample(x, u, 0.7)),
            ("prob", lambda: vkb.sample(x, u, prob=1)), ("token", lambda: vkb.sample(x, u, token=1)), ("v", lambda: vkb.KvCache(cache.k, None, x, x)),
            ("scales", lambda: vkb.KvCache(cache.k, cache.v, None, cache.v_scale))):
        with pytest.raises(vkb.VkbError, match=rf"\b{name}\b"):
            call()


# ---- reading the cache back -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("x_dt", ["float16", "bfloat16", "float32"])
def test_kv_read_of_more_tokens_than_the_grid_has_warps(cuda, x_dt):
    """One rounding of code x scale (exact in fp32: 8 bits times 24, rounded once), whatever the number of tokens."""
    import torch
    lens = [70, 33]
    cache, table, _ = make_cache(lens, 2, 48, 16)
    g = gen(4)
    n = 16 * 8 * torch.cuda.get_device_properties(0).multi_processor_count * 2 + 5
    seq = torch.randint(0, 2, (n,), generator=g, device="cuda", dtype=torch.int32)
    pos = (torch.rand(n, generator=g, device="cuda") * torch.tensor(lens, device="cuda")[seq.long()]).to(torch.int32)
    got = vkb.kv_read(cache, table, seq, pos, dtype=dt(x_dt))
    both = [values(cache, table, b, m) for b, m in enumerate(lens)]
    for i in range(2):
        want = torch.stack([torch.nn.functional.pad(both[b][i], (0, 0, 0, 0, 0, 70 - lens[b])) for b in range(2)])[seq.long(), pos.long()]
        assert torch.equal(got[i], want.float().to(dt(x_dt)))
    assert vkb.device_status() == 0


# ---- sizes near 2^31 --------------------------------------------------------------------------------------------------

def test_rms_norm_of_2_31_rows(cuda):
    """The most rows that an int holds, one element each (x / sqrt(x x) is its sign); more are refused, not cut."""
    import torch
    T = (1 << 31) - 1
    x = torch.full((T + 10, 1), 3.0, dtype=torch.float16, device="cuda")
    x[T - 1] = -2.0
    w = torch.full((1,), 0.5, dtype=torch.float16, device="cuda")
    y, *_ = vkb.rms_norm(x[:T], w, eps=0.0)
    assert float(y[-1]) == -0.5 and int((y[:-1] == 0.5).sum()) == T - 1
    with pytest.raises(vkb.VkbError, match="2\\^31"):
        vkb.rms_norm(x, w)


def test_sample_refuses_what_an_int_does_not_hold(cuda):
    import torch
    wide = torch.zeros((1, (1 << 32) + 5), dtype=torch.float16, device="cuda")
    with pytest.raises(vkb.VkbError, match="2\\^31"):
        vkb.sample(wide, torch.zeros(1, device="cuda"))


# ---- variants that larger calls take ----------------------------------------------------------------------------------

MANY = [(2048, 520), (2049, 2560), (2050, 544), (2051, 1032)]     # a row per warp: filled lanes and not, last blocks of 1 to 4 rows


@pytest.mark.parametrize("T,d", MANY)
@pytest.mark.parametrize("x_dt,res_dt", [("float16", "float32"), ("bfloat16", "bfloat16"), ("float32", "float16"), ("float32", None), ("bfloat16", None)])
def test_rms_norm_of_many_rows(cuda, T, d, x_dt, res_dt):
    """A lane's share of the sum is up to 80 squares one after another, 5 additions over the lanes: 85 u32, halved by the root,
    and five roundings: within the bound of (d / 1024 + 60) u32 that the rows per block are held to."""
    from test_step_gpu import test_rms_norm
    test_rms_norm(cuda, T, d, x_dt, res_dt)


@pytest.mark.parametrize("T,d", [(1, 32), (33, 2560), (3, 2080), (4, 16416)] + MANY[1:3])
@pytest.mark.parametrize("x_dt,res_dt", [("float16", "float32"), ("bfloat16", "bfloat16"), ("float32", "float16"), ("float16", None)])
def test_rms_norm_q8_with_residual(cuda, T, d, x_dt, res_dt):
    """Codes and scales of the exact y as in test_rms_norm_q8, for every kernel, and y and the residual as without them."""
    import torch
    g = gen(T + d)
    x = torch.randn((T, d), generator=g, device="cuda").to(dt(x_dt))
    w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt(x_dt))
    res = None if res_dt is None else (4 * torch.randn((T, d), generator=g, device="cuda")).to(dt(res_dt))
    y, r, q, s = vkb.rms_norm(x, w, res, q8=True)
    y2, r2, *_ = vkb.rms_norm(x, w, res)
    assert torch.equal(y, y2) and (res is None or torch.equal(r, r2))
    R = x.double() + (res.double() if res is not None else 0)
    B = (R / torch.sqrt(R.square().mean(1, keepdim=True) + 1e-6) * w.double()).view(T, -1, 32)
    amax = B.abs().amax(-1)
    assert bool(((s.double() - amax / 127).abs() <= amax / 127 * (2.0 ** -11 + 1e-5) + 2.0 ** -24).all())
    val, step = vkb.dequant(vkb.FMT_Q8, q, s, T, d).double().view(T, -1, 32), s.double()[..., None]
    assert bool(((val - B).abs() <= step * (0.5 + 127 * 2.0 ** -11 + 1e-3) + 2.0 ** -11 * B.abs() + 2.0 ** -24).all())


@pytest.mark.parametrize("lens,news,heads,hq,dim,rot,page,layout,x_dt", [
    ([200, 64], [200, 64], 2, 4, 256, 256, 64, "half", "float16"),             # 39 tokens at a time
    ([300], [230], 1, 2, 256, 64, 128, "interleaved", "bfloat16"),
    ([130, 100], [125, 60], 2, 2, 192, 192, 64, "half", "bfloat16"),           # 52
    ([260, 128], [250, 128], 1, 1, 128, 128, 128, "half", "float16"),          # 77
    ([128], [128], 1, 1, 80, 40, 128, "interleaved", "float32"),               # 121
])
def test_rope_append_of_pages_that_take_several_turns(cuda, lens, news, heads, hq, dim, rot, page, layout, x_dt):
    """Pages whose new tokens do not fit a block's shared memory at once."""
    from test_step_gpu import test_rope_append
    assert max(min(n, page) for n in news) > 40960 // (4 * (dim + 4))
    test_rope_append(cuda, lens, news, heads, hq, dim, rot, page, layout, x_dt)
