"""The operators between the quantised products of a decode step: rms_norm, rope_append (rotary positions and the write
into a paged 8-bit cache), attention over that cache, and sample. Torch tensors in and out; every call is one kernel
of libvkb.so on the current stream (or `stream`), described in include/vkb.h.

Outputs that are not given are allocated. With `stream` the inputs must be ready on that stream, and the outputs made
here are allocated for it.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import EINVAL, VkbError, _optr, _ptr, _stream, check, lib

DT_F16, DT_BF16, DT_F32 = 0, 1, 2
_DT = {torch.float16: DT_F16, torch.bfloat16: DT_BF16, torch.float32: DT_F32}
_LAYOUT = {"half": 0, "interleaved": 1}
PAGES = (16, 32, 64, 128)


def _bad(where: str, what: str) -> VkbError:
    e = VkbError(EINVAL, where)
    e.args = (f"{where}: {what}",)
    return e


def _need(ok: bool, where: str, what: str) -> None:
    if not ok:
        raise _bad(where, what)


def _on(stream):
    return torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext()


def _like(x, shape, dtype, stream):
    with _on(stream):
        return torch.empty(shape, dtype=dtype, device=x.device)


def _same(where: str, x, **others) -> None:
    """Tensors of the call: on x's device, the current CUDA device."""
    _need(x.is_cuda and x.device.index == torch.cuda.current_device(), where, "tensors must be on the current CUDA device")
    for name, t in others.items():
        _need(t is None or t.device == x.device, where, f"{name} must be on {x.device}")


def _ints(where: str, x, **arrays) -> None:
    _same(where, x, **arrays)
    for name, t in arrays.items():
        _need(t is None or (t.dtype == torch.int32 and t.is_contiguous()), where, f"{name} must be contiguous int32")


def rms_norm(x, weight, residual=None, eps: float = 1e-6, y=None, residual_out=None, q8: bool = False, stream=None):
    """r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight over the last dimension. x [T][d] (fp16, bf16 or fp32;
    rows may be strided), weight [d] of x's type, residual [T][d] of any of the three. Returns (y, r in the residual's
    type or None, codes or None, scales or None): with q8 also y in the Q8 format (int8 [T][d], fp16 [T][d / 32]), which
    dequant() reads. residual_out may be residual."""
    w = "rms_norm"
    _same(w, x, weight=weight, residual=residual, y=y, residual_out=residual_out)
    _need(x.dim() == 2 and x.dtype in _DT and (x.shape[1] == 1 or x.stride(1) == 1), w, "x must be [T][d] fp16, bf16 or fp32 with adjacent columns")
    T, d = x.shape
    _need(d > 0 and weight.dtype == x.dtype and weight.shape == (d,) and weight.is_contiguous(), w, "weight must be [d] of x's type")
    ld = x.stride(0) if T > 1 else d
    res_dt = 0
    if residual is not None:
        _need(residual.dtype in _DT and residual.shape == x.shape and residual.is_contiguous(), w, "residual must be contiguous [T][d]")
        res_dt = _DT[residual.dtype]
        if residual_out is None:
            residual_out = _like(x, (T, d), residual.dtype, stream)
        else:
            _need(residual_out.dtype == residual.dtype and residual_out.shape == x.shape and residual_out.is_contiguous(), w, "residual_out must be like residual")
    else:
        _need(residual_out is None, w, "residual_out without residual")
    if y is None:
        y = _like(x, (T, d), x.dtype, stream)
    else:
        _need(y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous(), w, "y must be contiguous [T][d] of x's type")
    q = s = None
    if q8:
        _need(d % 32 == 0, w, "the Q8 output needs d % 32 == 0")
        q, s = _like(x, (T, d), torch.int8, stream), _like(x, (T, d // 32), torch.float16, stream)
    check(lib().vkb_rms_norm(_DT[x.dtype], x.data_ptr(), ld, _optr(residual), _optr(residual_out), res_dt, weight.data_ptr(), eps,
                             y.data_ptr(), _optr(q), _optr(s), T, d, _stream(stream)), w)
    return y, residual_out, q, s


def rope_turns(rot: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0, original: int = 4096,
               beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda"):
    """Turns per position of the rot / 2 rotated pairs as 64-bit fractions of a turn (int64 tensor), and the factor that
    multiplies cos and sin. Frequencies base^(-2 i / rot), scaled for contexts `factor` times as long:
      "linear"    every frequency divided by factor (positions compressed)
      "base"      base multiplied by factor^(rot / (rot - 2)): the slowest pair is compressed by factor, the fastest kept
      "parts"     pairs that turn more than beta_fast times in `original` positions kept, those that turn less than
                  beta_slow times divided by factor, a linear ramp over the pairs between; cos and sin times
                  0.1 ln(factor) + 1"""
    w = "rope_turns"
    _need(rot >= 2 and rot % 2 == 0, w, "rot must be even and positive")
    _need(scaling in (None, "linear", "base", "parts") and factor >= 1.0, w, "scaling is None, linear, base or parts; factor >= 1")
    n, mscale = rot // 2, 1.0
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    freq = [base ** (-i / n) for i in range(n)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "parts":
        def pair(turns):   # the (fractional) pair that turns this many times in `original` positions
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(0, math.floor(pair(beta_fast))), min(n - 1, math.ceil(pair(beta_slow)))
        for i in range(n):
            r = min(1.0, max(0.0, (i - lo) / max(1e-3, hi - lo)))
            freq[i] *= (1 - r) + r / factor
        mscale = 0.1 * math.log(factor) + 1.0
    whole = [round(f / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for f in freq]
    t = torch.tensor([v - (1 << 64) if v >> 63 else v for v in whole], dtype=torch.int64)
    return t.to(device), mscale


class _CacheStruct(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("pages", ctypes.c_int), ("heads", ctypes.c_int), ("page", ctypes.c_int), ("dim", ctypes.c_int)]


class KvCache:
    """A paged 8-bit key/value cache over the caller's tensors: k, v uint8 [pages][heads][page][dim] (codes + 128),
    k_scale, v_scale fp32 [pages][heads]. KvCache.empty(...) allocates them."""

    def __init__(self, k, v, k_scale, v_scale):
        w = "KvCache"
        _need(k.dim() == 4 and k.dtype == torch.uint8 and k.is_contiguous(), w, "k must be contiguous uint8 [pages][heads][page][dim]")
        _same(w, k, v=v, k_scale=k_scale, v_scale=v_scale)
        _need(v.dtype == torch.uint8 and v.shape == k.shape and v.is_contiguous(), w, "v must be like k")
        for s in (k_scale, v_scale):
            _need(s.dtype == torch.float32 and s.shape == k.shape[:2] and s.is_contiguous(), w, "scales must be contiguous fp32 [pages][heads]")
        pages, self.heads, self.page, self.dim = k.shape
        _need(self.page in PAGES, w, f"page must be one of {PAGES}")
        _need(self.dim % 16 == 0 and 16 <= self.dim <= 256, w, "dim must be a multiple of 16 up to 256")
        self.k, self.v, self.k_scale, self.v_scale, self.pages = k, v, k_scale, v_scale, pages
        self._s = _CacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, self.heads, self.page, self.dim)
        self._ref = ctypes.byref(self._s)

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, page: int = 64, device="cuda"):
        codes = [torch.full((pages, heads, page, dim), 128, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*codes, *[torch.zeros((pages, heads), dtype=torch.float32, device=device) for _ in range(2)])


def _rows(where: str, name: str, x, heads: int, dim: int) -> int:
    """Row stride of x [T][heads][dim] whose heads are adjacent."""
    _need(x.dim() == 3 and x.shape[1] == heads and x.shape[2] == dim, where, f"{name} must be [T][{heads}][{dim}]")
    _need(x.shape[0] == 0 or ((dim == 1 or x.stride(2) == 1) and (heads == 1 or x.stride(1) == dim)), where, f"{name}: the heads of a row must be adjacent")
    return x.stride(0) if x.shape[0] > 1 else heads * dim


def _batch(where: str, cache, table, lens, cu, T: int) -> int:
    _need(table.dim() == 2 and lens.dim() == 1 and table.shape[0] == lens.shape[0] and table.shape[1] > 0, where, "table must be [B][pages], lens [B]")
    _ints(where, cache.k, table=table, lens=lens, cu=cu)
    B = lens.shape[0]
    _need(B > 0 and (cu.shape == (B + 1,) if cu is not None else T == B), where, "cu must be [B + 1]; without it there is one row per sequence")
    return B


def rope_append(cache: KvCache, table, lens, q, k, v, turns=None, cu=None, pos=None, layout: str = "half", mscale: float = 1.0,
                q_out=None, stream=None):
    """Rotate q [T][q_heads][dim] and k, write k and v [T][heads][dim] (fp16, bf16 or fp32; views of a fused row are
    fine) into the cache at the end of their sequences, and return the rotated q (q_out; may be q). table int32
    [B][pages], lens int32 [B] with the new tokens included, cu int32 [B + 1] row offsets (None: one row per sequence),
    pos int32 [T] rotary positions (None: the place in the sequence), turns from rope_turns() (None: no rotation).
    q None: append only."""
    w = "rope_append"
    T = k.shape[0]
    _need(layout in _LAYOUT, w, "layout is half or interleaved")
    _need(k.dtype in _DT and v.dtype == k.dtype, w, "k and v must be fp16, bf16 or fp32, alike")
    ldk, ldv = _rows(w, "k", k, cache.heads, cache.dim), _rows(w, "v", v, cache.heads, cache.dim)
    _need(v.shape[0] == T, w, "k and v must have the same rows")
    _same(w, cache.k, k=k, v=v, q=q, q_out=q_out, turns=turns)
    B = _batch(w, cache, table, lens, cu, T)
    _ints(w, cache.k, pos=pos)
    _need(pos is None or pos.shape == (T,), w, "pos must be [T]")
    rot = 0
    if turns is not None:
        _need(turns.dtype == torch.int64 and turns.dim() == 1 and turns.is_contiguous() and 2 * turns.shape[0] <= cache.dim, w, "turns must be int64 [rot / 2], rot <= dim")
        rot = 2 * turns.shape[0]
    hq = ldq = ldo = 0
    if q is not None:
        hq = q.shape[1]
        _need(q.shape[0] == T and q.dtype == k.dtype, w, "q must have k's rows and type")
        ldq = _rows(w, "q", q, hq, cache.dim)
        if q_out is None:
            q_out = _like(q, (T, hq, cache.dim), q.dtype, stream)
        else:
            _need(q_out.shape == q.shape and q_out.dtype == q.dtype, w, "q_out must be like q")
        ldo = _rows(w, "q_out", q_out, hq, cache.dim)
    else:
        _need(q_out is None, w, "q_out without q")
    check(lib().vkb_rope_append(cache._ref, table.data_ptr(), table.shape[1], lens.data_ptr(), _optr(cu), B, T, _DT[k.dtype],
                                _optr(q), ldq, _optr(q_out), ldo, hq, k.data_ptr(), ldk, v.data_ptr(), ldv, _optr(pos),
                                _optr(turns), rot, _LAYOUT[layout], mscale, _stream(stream)), w)
    return q_out


def kv_read(cache: KvCache, table, seq, pos, dtype=torch.float16, stream=None):
    """Cached tokens as values: (k, v) [n][heads][dim] of tokens pos[i] of sequences seq[i] (int32)."""
    w = "kv_read"
    _need(table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0, w, "table must be [B][pages]")
    _ints(w, cache.k, table=table, seq=seq, pos=pos)
    _need(seq.dim() == 1 and seq.shape == pos.shape and dtype in _DT, w, "seq and pos must be [n], dtype fp16, bf16 or fp32")
    n = seq.shape[0]
    k, v = (_like(seq, (n, cache.heads, cache.dim), dtype, stream) for _ in range(2))
    check(lib().vkb_kv_read(cache._ref, table.data_ptr(), table.shape[1], table.shape[0], seq.data_ptr(), pos.data_ptr(), n,
                            _DT[dtype], k.data_ptr(), v.data_ptr(), _stream(stream)), w)
    return k, v


def attention_workspace(cache: KvCache):
    """The zeroed workspace that attention() over this cache's head dimension needs; keep one per stream."""
    with torch.cuda.device(cache.k.device):
        return torch.zeros(lib().vkb_attention_work_bytes(cache.dim), dtype=torch.uint8, device=cache.k.device)


def attention(cache: KvCache, table, lens, q, cu=None, scale: float | None = None, window: int = 0, out=None, work=None,
              stream=None):
    """Causal attention of q [T][q_heads][dim] (fp16 or bf16; rows may be strided) over the cache: the rows of a
    sequence are its last tokens; lens, cu and table as in rope_append. scale: 1 / sqrt(dim) by default. window > 0:
    only the last `window` keys up to a row's own position. work: attention_workspace() (made here when not given, at
    the cost of an allocation and a memset)."""
    w = "attention"
    T, hq = q.shape[0], q.shape[1]
    _need(q.dtype in _DT, w, "q must be fp16 or bf16")
    ldq = _rows(w, "q", q, hq, cache.dim)
    _same(w, cache.k, q=q, out=out, work=work)
    B = _batch(w, cache, table, lens, cu, T)
    _need(hq > 0 and hq % cache.heads == 0, w, "q heads must be a multiple of the cache's heads")
    if out is None:
        out = _like(q, (T, hq, cache.dim), q.dtype, stream)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype, w, "out must be like q")
    ldo = _rows(w, "out", out, hq, cache.dim)
    if work is None:
        with _on(stream):
            work = attention_workspace(cache)
    check(lib().vkb_attention(cache._ref, table.data_ptr(), table.shape[1], lens.data_ptr(), _optr(cu), B, T, _DT[q.dtype],
                              q.data_ptr(), ldq, out.data_ptr(), ldo, hq, cache.dim ** -0.5 if scale is None else scale,
                              window, work.data_ptr(), work.numel() * work.element_size(), _stream(stream)), w)
    return out


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, token=None, prob=None, stream=None):
    """One token per row of logits [B][V] (fp16, bf16 or fp32; rows may be strided) from uniform numbers u fp32 [B]:
    temperature, top_p, min_p fp32 [B], top_k int32 [B] (None: off). Returns (token int32 [B], its probability among the
    kept tokens fp32 [B]). The rules: include/vkb.h."""
    w = "sample"
    _need(logits.dim() == 2 and logits.dtype in _DT and logits.shape[1] > 0 and (logits.shape[1] == 1 or logits.stride(1) == 1), w, "logits must be [B][V] fp16, bf16 or fp32 with adjacent columns")
    B, V = logits.shape
    _same(w, logits, u=u, temperature=temperature, top_p=top_p, min_p=min_p, prob=prob)
    _ints(w, logits, top_k=top_k, token=token)
    for name, t in (("u", u), ("temperature", temperature), ("top_p", top_p), ("min_p", min_p), ("prob", prob)):
        _need(t is None or (t.dtype == torch.float32 and t.shape == (B,) and t.is_contiguous()), w, f"{name} must be contiguous fp32 [B]")
    for name, t in (("top_k", top_k), ("token", token)):
        _need(t is None or t.shape == (B,), w, f"{name} must be [B]")
    if token is None:
        token = _like(logits, (B,), torch.int32, stream)
    if prob is None:
        prob = _like(logits, (B,), torch.float32, stream)
    check(lib().vkb_sample(_DT[logits.dtype], logits.data_ptr(), logits.stride(0) if B > 1 else V, B, V, _optr(temperature),
                           _optr(top_k), _optr(top_p), _optr(min_p), u.data_ptr(), token.data_ptr(), prob.data_ptr(),
                           _stream(stream)), w)
    return token, prob
