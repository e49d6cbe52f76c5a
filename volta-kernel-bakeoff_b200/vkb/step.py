"""The operators between the quantised products of a decode step: rms_norm, rope_append (rotary positions and the write
into a paged 8-bit cache), attention over that cache, and sample. Torch tensors in and out; every call is one kernel
of libvkb.so on the current stream (or `stream`), described in include/vkb.h.

Outputs that are not given are allocated. With `stream` the inputs must be ready on that stream; outputs made here are
allocated for it, and the allocator is told that the tensors given are in use on it.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import EINVAL, VkbError, check, lib

DT_F16, DT_BF16, DT_F32 = 0, 1, 2
_DT = {torch.float16: DT_F16, torch.bfloat16: DT_BF16, torch.float32: DT_F32}
_LAYOUT = {"half": 0, "interleaved": 1}
PAGES = (16, 32, 64, 128)
_INT = 0x7fffffff     # what the library's sizes hold


class _Refused(VkbError):
    """Arguments refused before the library is called (code EINVAL)."""

    def __init__(self, where: str, what: str):
        super().__init__(EINVAL, where)
        self.args = (f"{where}: {what}",)


# The current stream's handle. torch.cuda.current_stream() makes a Stream object (3 us per call on the host, as long as
# a small launch); the handle alone is a lookup.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _handle(stream, dev: int) -> int:
    return _raw_stream(dev) if stream is None else stream.cuda_stream


def _tensor(where: str, name: str, t) -> None:
    if not isinstance(t, torch.Tensor):
        raise _Refused(where, f"{name} must be a tensor")


def _device(where: str, x) -> int:
    """x's device index, which must be the current CUDA device."""
    dev = x.get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        raise _Refused(where, "tensors must be on the current CUDA device")
    return dev


def _on(stream):
    return torch.cuda.stream(stream) if stream is not None else contextlib.nullcontext()


def _made(like, stream):
    """An output like `like`, rows adjacent, allocated for the stream of the call."""
    if stream is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(like, memory_format=torch.contiguous_format)


def _new(like, shape, dtype, stream):
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _used(stream, *tensors) -> None:
    """Tensors of a call on a stream that need not be their own: their memory is not reused before the call has run."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _p(t):
    return None if t is None else t.data_ptr()


def _array(where: str, name: str, t, n: int, dtype, dev: int, optional: bool = False) -> None:
    """t (or None, where it is optional) is a contiguous [n] array on the device."""
    if t is None and optional:
        return
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or t.get_device() != dev or not t.is_contiguous():
        raise _Refused(where, f"{name} must be contiguous {dtype} [{n}] on the tensors' device")


def rms_norm(x, weight, residual=None, eps: float = 1e-6, y=None, residual_out=None, q8: bool = False, stream=None):
    """r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight over the last dimension. x [T][d] (fp16, bf16 or fp32;
    rows may be strided), weight [d] of x's type, residual [T][d] of any of the three. Returns (y, r in the residual's
    type or None, codes or None, scales or None): with q8 also y in the Q8 format (int8 [T][d], fp16 [T][d / 32]), which
    dequant() reads. residual_out may be residual."""
    w = "rms_norm"
    _tensor(w, "x", x)
    dt = _DT.get(x.dtype)
    if x.dim() != 2 or dt is None or (x.shape[1] > 1 and x.stride(1) != 1):
        raise _Refused(w, "x must be [T][d] fp16, bf16 or fp32 with adjacent columns")
    T, d = x.shape
    dev = _device(w, x)
    if d == 0 or T > _INT or d > _INT:
        raise _Refused(w, "d must be positive, T and d below 2^31")
    _array(w, "weight", weight, d, x.dtype, dev)
    res_dt = 0
    if residual is not None:
        _tensor(w, "residual", residual)
        res_dt = _DT.get(residual.dtype)
        if res_dt is None or residual.shape != x.shape or residual.get_device() != dev or not residual.is_contiguous():
            raise _Refused(w, "residual must be contiguous [T][d] fp16, bf16 or fp32 on x's device")
        if residual_out is None:
            residual_out = _made(residual, stream)
        elif not isinstance(residual_out, torch.Tensor) or residual_out.dtype != residual.dtype or residual_out.shape != x.shape or residual_out.get_device() != dev or not residual_out.is_contiguous():
            raise _Refused(w, "residual_out must be like residual")
    elif residual_out is not None:
        raise _Refused(w, "residual_out without residual")
    if y is None:
        y = _made(x, stream)
    elif not isinstance(y, torch.Tensor) or y.dtype != x.dtype or y.shape != x.shape or y.get_device() != dev or not y.is_contiguous():
        raise _Refused(w, "y must be contiguous [T][d] of x's type")
    q = s = None
    if q8:
        if d % 32:
            raise _Refused(w, "the Q8 output needs d % 32 == 0")
        q, s = _new(x, (T, d), torch.int8, stream), _new(x, (T, d // 32), torch.float16, stream)
    check(lib().vkb_rms_norm(dt, x.data_ptr(), x.stride(0) if T > 1 else d, _p(residual), _p(residual_out), res_dt,
                             weight.data_ptr(), eps, y.data_ptr(), _p(q), _p(s), T, d, _handle(stream, dev)), w)
    _used(stream, x, weight, residual, y, residual_out)
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
    if rot < 2 or rot % 2:
        raise _Refused(w, "rot must be even and positive")
    if scaling not in (None, "linear", "base", "parts") or not factor >= 1.0:
        raise _Refused(w, "scaling is None, linear, base or parts; factor >= 1")
    n, mscale = rot // 2, 1.0
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    freq = [base ** (-i / n) for i in range(n)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "parts":
        def pair(turns):   # the (fractional) pair that turns this many times in `original` positions
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        # the ramp may end past the last pair, which then keeps a share of its frequency
        lo, hi = max(0, math.floor(pair(beta_fast))), min(rot - 1, math.ceil(pair(beta_slow)))
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
        _tensor(w, "k", k)
        _tensor(w, "v", v)
        if k.dim() != 4 or k.dtype != torch.uint8 or not k.is_contiguous() or not k.is_cuda:
            raise _Refused(w, "k must be contiguous uint8 [pages][heads][page][dim] on a CUDA device")
        if v.dtype != torch.uint8 or v.shape != k.shape or v.device != k.device or not v.is_contiguous():
            raise _Refused(w, "v must be like k")
        for s in (k_scale, v_scale):
            if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or s.shape != k.shape[:2] or s.device != k.device or not s.is_contiguous():
                raise _Refused(w, "scales must be contiguous fp32 [pages][heads] on k's device")
        pages, self.heads, self.page, self.dim = k.shape
        if self.page not in PAGES:
            raise _Refused(w, f"page must be one of {PAGES}")
        if self.dim % 16 or not 16 <= self.dim <= 256:
            raise _Refused(w, "dim must be a multiple of 16 up to 256")
        self.device_index = k.get_device()
        self.k, self.v, self.k_scale, self.v_scale, self.pages = k, v, k_scale, v_scale, pages
        self._s = _CacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, self.heads, self.page, self.dim)
        self._ref = ctypes.byref(self._s)
        self.tensors = (k, v, k_scale, v_scale)

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, page: int = 64, device="cuda"):
        codes = [torch.full((pages, heads, page, dim), 128, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*codes, *[torch.zeros((pages, heads), dtype=torch.float32, device=device) for _ in range(2)])


_NO_CACHE = "cache must be a KvCache"


def _rows(where: str, name: str, x, heads: int, dim: int, dev: int) -> int:
    """Row stride of x [T][heads][dim], whose heads are adjacent."""
    n, st = x.shape, x.stride()
    if x.dim() != 3 or n[1] != heads or n[2] != dim or x.get_device() != dev or (n[0] and (st[2] != 1 or (heads > 1 and st[1] != dim))):
        raise _Refused(where, f"{name} must be [T][{heads}][{dim}] with the heads of a row adjacent, on the cache's device")
    return st[0] if n[0] > 1 else heads * dim


def _batch(where: str, table, lens, cu, T: int, dev: int) -> int:
    """The number of sequences."""
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.get_device() != dev or not table.numel():
        raise _Refused(where, "table must be contiguous int32 [B][pages] on the cache's device")
    B = table.shape[0]
    _array(where, "lens", lens, B, torch.int32, dev)
    if cu is not None:
        _array(where, "cu", cu, B + 1, torch.int32, dev)
    elif T != B:
        raise _Refused(where, "without cu there is one row per sequence")
    return B


def rope_append(cache: KvCache, table, lens, q, k, v, turns=None, cu=None, pos=None, layout: str = "half", mscale: float = 1.0,
                q_out=None, stream=None):
    """Rotate q [T][q_heads][dim] and k, write k and v [T][heads][dim] (fp16, bf16 or fp32; views of a fused row are
    fine) into the cache at the end of their sequences, and return the rotated q (q_out; may be q). table int32
    [B][pages], lens int32 [B] with the new tokens included, cu int32 [B + 1] row offsets (None: one row per sequence),
    pos int32 [T] rotary positions (None: the place in the sequence), turns from rope_turns() (None: no rotation).
    q None: append only."""
    w = "rope_append"
    if not isinstance(cache, KvCache):
        raise _Refused(w, _NO_CACHE)
    if not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor) or k.dim() != 3:
        raise _Refused(w, "k and v must be tensors [T][heads][dim]")
    dev = _device(w, k)
    T, heads, dim = k.shape[0], cache.heads, cache.dim
    dt, lay = _DT.get(k.dtype), _LAYOUT.get(layout)
    if dev != cache.device_index:
        raise _Refused(w, "k must be on the cache's device")
    if lay is None:
        raise _Refused(w, "layout is half or interleaved")
    if dt is None or v.dtype != k.dtype or v.shape != k.shape:
        raise _Refused(w, "k and v must be fp16, bf16 or fp32, alike")
    ldk, ldv = _rows(w, "k", k, heads, dim, dev), _rows(w, "v", v, heads, dim, dev)
    B = _batch(w, table, lens, cu, T, dev)
    _array(w, "pos", pos, T, torch.int32, dev, optional=True)
    rot = 0
    if turns is not None:
        rot = 2 * turns.numel() if isinstance(turns, torch.Tensor) else 0
        if rot > dim or rot == 0:
            raise _Refused(w, "turns must be int64 [rot / 2] with 0 < rot <= dim")
        _array(w, "turns", turns, rot // 2, torch.int64, dev)
    hq = ldq = ldo = 0
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.shape[0] != T or q.dtype != k.dtype:
            raise _Refused(w, "q must be [T][q_heads][dim] with k's rows and type")
        hq = q.shape[1]
        ldq = _rows(w, "q", q, hq, dim, dev)
        if q_out is None:
            q_out = _made(q, stream)
            ldo = hq * dim
        else:
            if not isinstance(q_out, torch.Tensor) or q_out.dtype != q.dtype or q_out.shape != q.shape:
                raise _Refused(w, "q_out must be like q")
            ldo = _rows(w, "q_out", q_out, hq, dim, dev)
    elif q_out is not None:
        raise _Refused(w, "q_out without q")
    check(lib().vkb_rope_append(cache._ref, table.data_ptr(), table.shape[1], lens.data_ptr(), _p(cu), B, T, dt,
                                _p(q), ldq, _p(q_out), ldo, hq, k.data_ptr(), ldk, v.data_ptr(), ldv, _p(pos),
                                _p(turns), rot, lay, mscale, _handle(stream, dev)), w)
    _used(stream, table, lens, q, k, v, turns, cu, pos, q_out, *cache.tensors)
    return q_out


def kv_read(cache: KvCache, table, seq, pos, dtype=torch.float16, stream=None):
    """Cached tokens as values: (k, v) [n][heads][dim] of tokens pos[i] of sequences seq[i] (int32)."""
    w = "kv_read"
    if not isinstance(cache, KvCache):
        raise _Refused(w, _NO_CACHE)
    if not isinstance(seq, torch.Tensor):
        raise _Refused(w, "seq must be a tensor")
    dev = _device(w, seq)
    if dev != cache.device_index or seq.dim() != 1 or dtype not in _DT:
        raise _Refused(w, "seq and pos must be [n] on the cache's device, dtype fp16, bf16 or fp32")
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.get_device() != dev or not table.numel():
        raise _Refused(w, "table must be contiguous int32 [B][pages] on the cache's device")
    n = seq.shape[0]
    _array(w, "seq", seq, n, torch.int32, dev)
    _array(w, "pos", pos, n, torch.int32, dev)
    k = _new(seq, (n, cache.heads, cache.dim), dtype, stream)
    v = _made(k, stream)
    check(lib().vkb_kv_read(cache._ref, table.data_ptr(), table.shape[1], table.shape[0], seq.data_ptr(), pos.data_ptr(), n,
                            _DT[dtype], k.data_ptr(), v.data_ptr(), _handle(stream, dev)), w)
    _used(stream, table, seq, pos, *cache.tensors)
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
    if not isinstance(cache, KvCache):
        raise _Refused(w, _NO_CACHE)
    if not isinstance(q, torch.Tensor):
        raise _Refused(w, "q must be a tensor")
    if not 0 <= window <= _INT:
        raise _Refused(w, "window must be 0 (none) or a number of keys below 2^31")
    dev = _device(w, q)
    if dev != cache.device_index or q.dim() != 3:
        raise _Refused(w, "q must be [T][q_heads][dim] on the cache's device")
    T, hq = q.shape[0], q.shape[1]
    if q.dtype != torch.float16 and q.dtype != torch.bfloat16:
        raise _Refused(w, "q must be fp16 or bf16")
    if hq == 0 or hq % cache.heads:
        raise _Refused(w, "q heads must be a multiple of the cache's heads")
    ldq = _rows(w, "q", q, hq, cache.dim, dev)
    B = _batch(w, table, lens, cu, T, dev)
    if out is None:
        out = _made(q, stream)
        ldo = hq * cache.dim
    else:
        if not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype:
            raise _Refused(w, "out must be like q")
        ldo = _rows(w, "out", out, hq, cache.dim, dev)
    if work is None:
        with _on(stream):
            work = attention_workspace(cache)
    elif not isinstance(work, torch.Tensor) or work.get_device() != dev or not work.is_contiguous():
        raise _Refused(w, "work must be attention_workspace()'s tensor on the cache's device")
    check(lib().vkb_attention(cache._ref, table.data_ptr(), table.shape[1], lens.data_ptr(), _p(cu), B, T, _DT[q.dtype],
                              q.data_ptr(), ldq, out.data_ptr(), ldo, hq, cache.dim ** -0.5 if scale is None else scale,
                              window, work.data_ptr(), work.numel() * work.element_size(), _handle(stream, dev)), w)
    _used(stream, table, lens, q, cu, out, work, *cache.tensors)
    return out


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, token=None, prob=None, stream=None):
    """One token per row of logits [B][V] (fp16, bf16 or fp32; rows may be strided) from uniform numbers u fp32 [B]:
    temperature, top_p, min_p fp32 [B], top_k int32 [B] (None: off). Returns (token int32 [B], its probability among the
    kept tokens fp32 [B]). The rules: include/vkb.h."""
    w = "sample"
    _tensor(w, "logits", logits)
    dt = _DT.get(logits.dtype)
    if logits.dim() != 2 or dt is None or logits.shape[1] == 0 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise _Refused(w, "logits must be [B][V] fp16, bf16 or fp32 with adjacent columns")
    B, V = logits.shape
    if B > _INT or V > _INT:
        raise _Refused(w, "B and V must be below 2^31")
    dev, f32 = _device(w, logits), torch.float32
    _array(w, "u", u, B, f32, dev)
    _array(w, "temperature", temperature, B, f32, dev, optional=True)
    _array(w, "top_k", top_k, B, torch.int32, dev, optional=True)
    _array(w, "top_p", top_p, B, f32, dev, optional=True)
    _array(w, "min_p", min_p, B, f32, dev, optional=True)
    if prob is None:
        prob = _made(u, stream)
    else:
        _array(w, "prob", prob, B, f32, dev)
    if token is None:
        token = _new(u, (B,), torch.int32, stream)
    else:
        _array(w, "token", token, B, torch.int32, dev)
    check(lib().vkb_sample(dt, logits.data_ptr(), logits.stride(0) if B > 1 else V, B, V, _p(temperature), _p(top_k), _p(top_p),
                           _p(min_p), u.data_ptr(), token.data_ptr(), prob.data_ptr(), _handle(stream, dev)), w)
    _used(stream, logits, u, temperature, top_k, top_p, min_p, token, prob)
    return token, prob
