"""CPU tests of the decode-step operators' boundary: what the library and the binding refuse before any CUDA call, the
frequencies of rope_turns(), and the workspace size without a device."""
import ctypes
import math

import pytest

import vkb

F16, BF16, F32 = 0, 1, 2
A = ctypes.c_void_p(1 << 20)     # an aligned address that is never read: every call below is refused or has no rows


class _Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "ks", "vs")] + [(n, ctypes.c_int) for n in ("pages", "heads", "page", "dim")]


def _cache(**over):
    c = dict(k=1 << 20, v=1 << 20, ks=1 << 20, vs=1 << 20, pages=4, heads=2, page=64, dim=64)
    c.update(over)
    return ctypes.byref(_Cache(**c))


def test_rms_norm_refusals():
    f = vkb.lib().vkb_rms_norm
    ok = dict(dt=F16, x=A, ldx=64, res=None, res_out=None, res_dt=0, w=A, eps=1e-6, y=A, q=None, s=None, T=1, d=64)

    def rc(**over):
        a = dict(ok, **over)
        return f(*a.values(), None)
    assert rc(T=0) == vkb.OK
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(dt=7), dict(d=0), dict(T=-1), dict(ldx=63), dict(eps=-1.0),
                dict(eps=math.nan), dict(q=A), dict(s=A), dict(res_out=A), dict(res=A, res_dt=5), dict(x=ctypes.c_void_p((1 << 20) + 1))):
        assert rc(**bad) == vkb.EINVAL, bad
    assert rc(q=A, s=A, d=48, ldx=48) == vkb.EUNSUPPORTED


def test_rope_append_refusals():
    f = vkb.lib().vkb_rope_append
    ok = dict(cache=_cache(), table=A, ld=4, lens=A, cu=None, B=2, T=2, dt=F16, q=A, ldq=256, qo=A, ldqo=256, hq=4, k=A, ldk=128, v=A,
              ldv=128, pos=None, turns=A, rot=64, layout=0, mscale=1.0)

    def rc(**over):
        return f(*dict(ok, **over).values(), None)
    assert rc(T=0, cu=A) == vkb.OK
    for bad in (dict(cache=None), dict(table=None), dict(ld=0), dict(lens=None), dict(B=0), dict(T=3), dict(T=-1), dict(dt=3),
                dict(k=None), dict(v=None), dict(q=None), dict(qo=None), dict(hq=-1), dict(ldq=255), dict(ldk=127), dict(ldv=127),
                dict(ldqo=255), dict(rot=66), dict(rot=-2), dict(turns=None), dict(layout=2), dict(ldqo=512),
                dict(cache=_cache(k=None)), dict(cache=_cache(k=(1 << 20) + 8)), dict(cache=_cache(pages=0))):
        assert rc(**bad) == vkb.EINVAL, bad
    for bad in (dict(rot=63), dict(cache=_cache(dim=72)), dict(cache=_cache(dim=272)), dict(cache=_cache(page=48)),
                dict(cache=_cache(pages=1 << 25))):
        assert rc(**bad) == vkb.EUNSUPPORTED, bad


def test_kv_read_refusals():
    f = vkb.lib().vkb_kv_read
    ok = dict(cache=_cache(), table=A, ld=4, B=2, seq=A, pos=A, n=3, dt=F16, k=A, v=A)

    def rc(**over):
        return f(*dict(ok, **over).values(), None)
    assert rc(n=0) == vkb.OK
    for bad in (dict(seq=None), dict(pos=None), dict(k=None), dict(v=ctypes.c_void_p((1 << 20) + 8)), dict(dt=9), dict(B=0), dict(n=-1)):
        assert rc(**bad) == vkb.EINVAL, bad


def test_attention_refusals():
    f = vkb.lib().vkb_attention
    ok = dict(cache=_cache(), table=A, ld=4, lens=A, cu=None, B=2, T=2, dt=F16, q=A, ldq=256, out=A, ldo=256, hq=4, scale=0.1, window=0,
              work=A, bytes=1 << 30)

    def rc(**over):
        return f(*dict(ok, **over).values(), None)
    assert rc(T=0, cu=A) == vkb.OK
    for bad in (dict(q=None), dict(out=None), dict(lens=None), dict(hq=3), dict(hq=0), dict(window=-1), dict(scale=-1.0),
                dict(scale=math.nan), dict(work=None), dict(work=ctypes.c_void_p((1 << 20) + 4)), dict(dt=8), dict(T=1), dict(ldq=128),
                dict(ldo=128)):
        assert rc(**bad) == vkb.EINVAL, bad
    for bad in (dict(dt=F32), dict(cache=_cache(dim=40))):
        assert rc(**bad) == vkb.EUNSUPPORTED, bad
    assert vkb.lib().vkb_attention_work_bytes(40) == 0 and vkb.lib().vkb_attention_work_bytes(512) == 0


def test_sample_refusals():
    f = vkb.lib().vkb_sample
    ok = dict(dt=F16, logits=A, ld=100, B=2, V=100, t=None, k=None, p=None, m=None, u=A, token=A, prob=None)

    def rc(**over):
        return f(*dict(ok, **over).values(), None)
    assert rc(B=0) == vkb.OK
    for bad in (dict(logits=None), dict(u=None), dict(token=None), dict(dt=4), dict(V=0), dict(ld=99), dict(B=-1)):
        assert rc(**bad) == vkb.EINVAL, bad


def test_binding_refuses_cpu_tensors_and_wrong_shapes():
    import torch
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.ones(64, dtype=torch.float16)
    with pytest.raises(vkb.VkbError, match="CUDA device"):
        vkb.rms_norm(x, w)
    with pytest.raises(vkb.VkbError, match="adjacent columns"):
        vkb.rms_norm(x.t(), w)
    with pytest.raises(vkb.VkbError, match="CUDA device"):
        vkb.sample(torch.zeros(1, 8), torch.zeros(1))
    with pytest.raises(vkb.VkbError, match="CUDA device"):
        vkb.KvCache(*[torch.zeros(1, 1, 16, 16, dtype=torch.uint8)] * 2, *[torch.zeros(1, 1)] * 2)
    with pytest.raises(AttributeError):
        vkb.no_such_operator


def _freq(turns):
    return [(int(t) % (1 << 64)) / 2.0 ** 64 * 2 * math.pi for t in turns]


def test_rope_turns():
    n = 32
    plain, m = vkb.rope_turns(2 * n, base=10000.0, device="cpu")
    assert m == 1.0 and plain.shape == (n,)
    for i, f in enumerate(_freq(plain)):
        assert abs(f - 10000.0 ** (-i / n)) < 1e-12
    for f, g in zip(_freq(vkb.rope_turns(2 * n, scaling="linear", factor=4.0, device="cpu")[0]), _freq(plain)):
        assert abs(f - g / 4) < 1e-12
    base = _freq(vkb.rope_turns(2 * n, scaling="base", factor=4.0, device="cpu")[0])
    assert abs(base[0] - 1.0) < 1e-12 and abs(base[-1] * 4 / _freq(plain)[-1] - 1) < 1e-9
    parts, m = vkb.rope_turns(2 * n, scaling="parts", factor=4.0, original=4096, device="cpu")
    parts = _freq(parts)
    assert abs(m - (0.1 * math.log(4.0) + 1)) < 1e-12
    assert abs(parts[0] - 1.0) < 1e-12 and abs(parts[-1] * 4 / _freq(plain)[-1] - 1) < 1e-9
    assert all(a >= b for a, b in zip(parts, parts[1:]))
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, scaling="x"), dict(rot=8, scaling="linear", factor=0.5)):
        with pytest.raises(vkb.VkbError):
            vkb.rope_turns(**bad, device="cpu")
