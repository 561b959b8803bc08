"""Operators of a decoder layer around the block-scaled products.

  rms_norm, rms_norm_quant   residual addition and RMS norm; the result in the input's type, or as the e4m3
                             codes and 1x128 scales that fp8_gemm / fp4_gemm take
  rope, rope_freqs           rotary positions on part of each head, exact at far positions
  cache_append, cache_attn   a paged e4m3 key/value cache with one scale per page and head, and the attention
                             of each sequence's newest tokens over it

All compute runs in the CUDA library (C ABI: include/bsgemm.h); CPU tensors
are an error.  Calls run on the current stream of the tensors' device, never
synchronise, and can be captured into CUDA graphs.  What only the device
knows (page indices, lengths, positions) is checked there: a page index or
length out of range reads and writes nothing, and ``device_error_check``
reports it.
"""

from __future__ import annotations

import ctypes
import functools
import math
import time as _time
from typing import Optional

import torch

from . import _lib
from .kernel import _X_DT, _tally

__all__ = ["rms_norm", "rms_norm_quant", "rope", "rope_freqs", "cache_append", "cache_attn"]

_I64x3 = ctypes.c_int64 * 3


# Host time counts where a decode step is not captured into a graph: these two are what
# torch.cuda.current_stream(...).cuda_stream and torch.cuda.current_device() end in, without 2 us of wrapping.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _device_of(*ts: Optional[torch.Tensor]) -> int:
    """The index of the CUDA device that all the tensors are on."""
    index = ts[0].get_device()
    if index < 0:
        raise RuntimeError("bsgemm ops run on CUDA tensors only (no CPU fallback)")
    for t in ts:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on {ts[0].device} and {t.device}")
    return index


def _call(index: int, fn, *args) -> None:
    """The library call on the current stream of device ``index``, with that device current."""
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
        if status:
            _lib.check(status)
    else:
        with torch.cuda.device(index):
            _lib.check(fn(*args, _raw_stream(index)))


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _norm_args(x, weight, residual):
    dev = _device_of(x, weight, residual)
    dt = x.dtype
    if dt not in _X_DT:
        raise TypeError(f"rms_norm: x is {dt}, expected bf16, f16 or fp32")
    if weight.dtype != dt or (residual is not None and residual.dtype != dt):
        raise TypeError("rms_norm: x, weight and residual must have one type")
    shape = x.shape
    if not shape or weight.shape != shape[-1:]:
        raise ValueError(f"rms_norm: weight {tuple(weight.shape)} does not match x {tuple(shape)}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"rms_norm: residual {tuple(residual.shape)} does not match x {tuple(shape)}")
    xc = x.contiguous()
    H = shape[-1]
    return (dev, _X_DT[dt], H, xc.numel() // H if H else 0, xc, weight.contiguous(),
            None if residual is None else residual.contiguous(), None if residual is None else torch.empty_like(xc))


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """RMS norm over the last dim: ``y = h * weight / sqrt(mean(h^2) + eps)`` with ``h = x + residual``.

    x and residual [..., H] and weight [H] in one type (bf16, f16 or fp32), H a
    multiple of 8 up to 16384.  h is rounded to the type (it is the residual
    stream that the next layer reads) and the norm is taken of the rounded h;
    statistics and product are fp32, rounded once.  Returns ``y``, or ``(y, h)``
    with a residual.
    """
    t0 = _time.perf_counter()
    dev, dt, H, rows, xc, wc, rc, h = _norm_args(x, weight, residual)
    y = torch.empty_like(xc)
    _call(dev, _lib.load().bs_rms_norm, xc.data_ptr(), _ptr(rc), wc.data_ptr(), dt, rows, H, eps, _ptr(h), y.data_ptr())
    _tally("rms_norm", t0)
    return y if h is None else (y, h)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                   scale_fmt: Optional[str] = None, scale_dtype: torch.dtype = torch.float32):
    """:func:`rms_norm` with its result quantised as :func:`act_quant` does (blocks of 128, the same scale rules
    and ``scale_fmt``), from the fp32 values, without the round trip through memory in 16 bits.

    H a multiple of 128 up to 16384; ``scale_dtype`` torch.float32 or
    torch.float8_e8m0fnu.  Returns ``(codes, scales)``, or ``(codes, scales, h)``
    with a residual; codes and scales go to fp8_gemm / fp4_gemm.
    """
    t0 = _time.perf_counter()
    if scale_dtype not in (torch.float32, torch.float8_e8m0fnu):
        raise NotImplementedError(f"rms_norm_quant: scale_dtype {scale_dtype} not supported")
    dev, dt, H, rows, xc, wc, rc, h = _norm_args(x, weight, residual)
    if H % 128 != 0:
        raise NotImplementedError(f"rms_norm_quant: H={H} is not a multiple of 128")
    y = torch.empty_like(xc, dtype=torch.float8_e4m3fn)
    s = xc.new_empty((*x.shape[:-1], H // 128), dtype=scale_dtype)
    _call(dev, _lib.load().bs_rms_norm_quant, xc.data_ptr(), _ptr(rc), wc.data_ptr(), dt, rows, H, eps,
          0 if scale_fmt is None else 1, _ptr(h), y.data_ptr(), s.data_ptr(),
          _lib.DT_F32 if scale_dtype == torch.float32 else _lib.DT_E8M0)
    _tally("rms_norm_quant", t0)
    return (y, s) if h is None else (y, s, h)


def rope_freqs(rope_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
               original_max_position: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
               device="cuda") -> torch.Tensor:
    """Radians per position of the rope_dim/2 pairs, fp64, for :func:`rope`.

    ``scaling`` stretches them for contexts ``factor`` times as long:
    ``"linear"`` divides every frequency by factor; ``"ntk"`` raises the base
    so that the slowest pair is divided by factor and the fastest is kept;
    ``"yarn"`` keeps pairs that make more than beta_fast turns within
    original_max_position, divides those of fewer than beta_slow by factor,
    and blends linearly between.
    """
    if rope_dim <= 0 or rope_dim % 2:
        raise ValueError(f"rope_freqs: rope_dim={rope_dim}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"rope_freqs: scaling {scaling!r}: expected None, 'linear', 'ntk' or 'yarn'")
    if not factor >= 1.0:
        raise ValueError(f"rope_freqs: factor={factor}")
    if scaling == "ntk" and rope_dim > 2:
        base = base * factor ** (rope_dim / (rope_dim - 2))
    f = base ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64) / rope_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair(turns):   # index of the pair that makes this many turns
            return rope_dim * math.log(original_max_position / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rope_dim - 1)
        ramp = ((torch.arange(rope_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    return f.to(device)


def rope(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, layout: str = "interleaved", offset: int = 0,
         inverse: bool = False, scale: float = 1.0, inplace: bool = False) -> torch.Tensor:
    """Rotary positions: x [..., heads, D] (bf16, f16 or fp32), positions [...] (int32 or int64, any sign), freqs
    fp64 [rope_dim/2] (:func:`rope_freqs`) -> rotated x, contiguous, or x itself with ``inplace``.

    Dims [offset, offset + rope_dim) of each head turn, the others are copied.
    ``layout`` is ``"interleaved"`` (pairs x[2i], x[2i+1]) or ``"half"``
    (x[i], x[i + rope_dim/2]); ``inverse`` turns back (also the gradient of the
    forward turn); ``scale`` multiplies the turned dims.  Angles keep fp64's
    precision at any position.  rope_dim a multiple of 16 up to 512, offset and
    D multiples of 8.
    """
    t0 = _time.perf_counter()
    dev = _device_of(x, positions, freqs)
    dt = _X_DT.get(x.dtype)
    if dt is None:
        raise TypeError(f"rope: x is {x.dtype}, expected bf16, f16 or fp32")
    if positions.dtype != torch.int64 and positions.dtype != torch.int32:
        raise TypeError(f"rope: positions are {positions.dtype}, expected int64 or int32")
    if freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("rope: freqs must be a float64 vector")
    if layout not in ("interleaved", "half"):
        raise ValueError(f"rope: layout {layout!r}: expected 'interleaved' or 'half'")
    shape = x.shape
    if len(shape) < 2 or positions.shape != shape[:-2]:
        raise ValueError(f"rope: positions {tuple(positions.shape)} do not match x {tuple(shape)}")
    H, D = shape[-2:]
    xt, tok, head = x, H * D, D
    if not x.is_contiguous() or x.data_ptr() % 16:
        e = 16 // x.element_size()
        # one token stride: the leading dims collapse into one, heads and dims stay
        tok, head = _token_stride(x), x.stride(-2)
        if tok is None or x.stride(-1) != 1 or head % e or tok % e or x.data_ptr() % 16:
            if inplace:
                raise ValueError("rope: an in-place x needs contiguous 16-byte aligned dims and one stride over its tokens")
            xt, tok, head = x.clone(memory_format=torch.contiguous_format), H * D, D
    out = xt if inplace else torch.empty_like(x, memory_format=torch.contiguous_format)
    pc, fc = positions.contiguous(), freqs.contiguous()
    _call(dev, _lib.load().bs_rope, xt.data_ptr(), dt, pc.numel(), H, D, tok, head, pc.data_ptr(),
          1 if pc.dtype == torch.int64 else 0, fc.data_ptr(), 2 * fc.numel(), offset, 1 if layout == "half" else 0,
          1 if inverse else 0, scale, out.data_ptr(), tok if inplace else H * D, head if inplace else D)
    _tally("rope", t0)
    return out


def _token_stride(x: torch.Tensor) -> Optional[int]:
    """The stride of dims 0..-3 taken as one, or None where they are not one."""
    stride, want = x.size(-1) * x.size(-2), None
    for i in range(x.dim() - 3, -1, -1):
        if x.size(i) == 1:
            continue
        if want is None:
            stride = x.stride(i)
        elif x.stride(i) != want:
            return None
        want = x.stride(i) * x.size(i)
    return stride


def _check_cache(name, cache, scale, D, Hkv):
    if cache.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        raise TypeError(f"{name}: a cache is float8_e4m3fn with fp32 scales")
    if cache.dim() != 4 or cache.size(1) != Hkv or cache.size(3) != D or scale.shape != cache.shape[:2]:
        raise ValueError(f"{name}: cache {tuple(cache.shape)} and scales {tuple(scale.shape)} do not match "
                         f"[n_pages, {Hkv}, page, {D}]")
    if not (cache.is_contiguous() and scale.is_contiguous()):
        raise ValueError(f"{name}: cache and scales must be contiguous")


def _check_index(name, what, t, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{name}: {what} is {t.dtype}, expected int32")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _strided(x: torch.Tensor, unit: int, align: int) -> torch.Tensor:
    """x, or a contiguous copy where its strides do not keep vectors of ``unit`` elements whole."""
    s = x.stride()
    if s[3] == 1 and not (s[0] % unit or s[1] % unit or s[2] % unit or x.data_ptr() % align):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def cache_append(k: torch.Tensor, v: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: Optional[torch.Tensor],
                 k_scale: torch.Tensor, v_scale: Optional[torch.Tensor], block_table: torch.Tensor,
                 start: torch.Tensor, new_lens: Optional[torch.Tensor] = None) -> None:
    """Write new keys and values into a paged e4m3 cache, in place.

    k, v [B, S, Hkv, D] (bf16, f16 or fp32, any strides with the last dim
    contiguous); caches float8_e4m3fn [n_pages, Hkv, page, D] (page 16, 32, 64
    or 128; D a multiple of 16 up to 512) with fp32 scales [n_pages, Hkv];
    block_table int32 [B, max_pages]; start int32 [B], the tokens already
    cached; new_lens int32 [B], how many of the S tokens are real (all, without
    it).  Token i of sequence b becomes position start[b] + i.  ``v``,
    ``v_cache`` and ``v_scale`` None: a cache whose values are its keys.

    A page's scale is the smallest power of two that holds what was written to
    it; when it grows, the page's earlier codes are rounded again.  Writing a
    page's slot 0 starts the page anew; slots behind the new tokens stay as
    they were.  Sequences of one call must not write to the same page.
    """
    t0 = _time.perf_counter()
    dev = _device_of(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, new_lens)
    if k.dim() != 4:
        raise ValueError(f"cache_append: k {tuple(k.shape)}, expected [B, S, Hkv, D]")
    B, S, Hkv, D = k.shape
    if (v is None) != (v_cache is None) or (v is None) != (v_scale is None):
        raise ValueError("cache_append: v, v_cache and v_scale go together")
    if k.dtype not in _X_DT or (v is not None and v.dtype != k.dtype):
        raise TypeError("cache_append: k and v must have one type of bf16, f16 or fp32")
    _check_cache("cache_append", k_cache, k_scale, D, Hkv)
    if v is not None:
        if v.shape != k.shape or v_cache.shape != k_cache.shape:
            raise ValueError("cache_append: v does not match k")
        _check_cache("cache_append", v_cache, v_scale, D, Hkv)
    if block_table.dim() != 2:
        raise ValueError("cache_append: block_table must be [B, max_pages]")
    bt = _check_index("cache_append", "block_table", block_table, (B, block_table.size(1)))
    st = _check_index("cache_append", "start", start, (B,))
    nl = None if new_lens is None else _check_index("cache_append", "new_lens", new_lens, (B,))
    if S == 0 or B == 0:
        return
    e = 16 // k.element_size()
    kc = _strided(k, e, 16)
    vc = None if v is None else _strided(v, e, 16)
    _call(dev, _lib.load().bs_cache_append, kc.data_ptr(), _ptr(vc), _X_DT[k.dtype], B, S, Hkv, D,
          _I64x3(*kc.stride()[:3]), None if vc is None else _I64x3(*vc.stride()[:3]), k_cache.data_ptr(), _ptr(v_cache),
          k_scale.data_ptr(), _ptr(v_scale), k_cache.size(0), k_cache.size(2), bt.data_ptr(), bt.size(1), st.data_ptr(),
          _ptr(nl))
    _tally("cache_append", t0)


@functools.lru_cache(maxsize=4096)
def _attn_workspace(index: int, B: int, S: int, H: int, Hkv: int, D: int, dt: int) -> int:
    with torch.cuda.device(index):
        n = _lib.load().bs_cache_attn_workspace_size(B, S, H, Hkv, D, dt)
    return (max(n, 256) + 3) // 4 * 4


def cache_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: Optional[torch.Tensor], k_scale: torch.Tensor,
               v_scale: Optional[torch.Tensor], block_table: torch.Tensor, seq_lens: torch.Tensor,
               softmax_scale: float, attn_sink: Optional[torch.Tensor] = None,
               new_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of each sequence's newest tokens over a paged e4m3 cache (:func:`cache_append`).

    q [B, S, H, D] bf16 or f16, H a multiple of the cache's Hkv (query heads
    h*H/Hkv ... share kv head h); seq_lens int32 [B] counts all cached tokens,
    the S newest (or new_lens[b] of them) included; query token i sees the
    first seq_lens[b] - S + i + 1.  ``v_cache`` and ``v_scale`` None: the
    values are the keys.  attn_sink fp32 [H]: a logit per head that takes
    softmax weight and adds no value, as in :func:`sparse_attn`.  Returns
    [B, S, H, D] in q's type; rows that see nothing, and padded query tokens,
    are zero.  Infinities and NaN in slots that a row does not see do not reach
    it.
    """
    t0 = _time.perf_counter()
    dev = _device_of(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, attn_sink, new_lens)
    if q.dim() != 4:
        raise ValueError(f"cache_attn: q {tuple(q.shape)}, expected [B, S, H, D]")
    B, S, H, D = q.shape
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"cache_attn: q is {q.dtype}, expected bf16 or f16")
    if (v_cache is None) != (v_scale is None):
        raise ValueError("cache_attn: v_cache and v_scale go together")
    if k_cache.dim() != 4:
        raise ValueError(f"cache_attn: k_cache {tuple(k_cache.shape)}, expected [n_pages, Hkv, page, D]")
    Hkv = k_cache.size(1)
    _check_cache("cache_attn", k_cache, k_scale, D, Hkv)
    if v_cache is not None:
        _check_cache("cache_attn", v_cache, v_scale, D, Hkv)
        if v_cache.shape != k_cache.shape:
            raise ValueError("cache_attn: v_cache does not match k_cache")
    if Hkv == 0 or H % Hkv:
        raise ValueError(f"cache_attn: {H} query heads over {Hkv} kv heads")
    if block_table.dim() != 2:
        raise ValueError("cache_attn: block_table must be [B, max_pages]")
    bt = _check_index("cache_attn", "block_table", block_table, (B, block_table.size(1)))
    sl = _check_index("cache_attn", "seq_lens", seq_lens, (B,))
    nl = None if new_lens is None else _check_index("cache_attn", "new_lens", new_lens, (B,))
    sink = None
    if attn_sink is not None:
        if attn_sink.shape != (H,):
            raise ValueError(f"cache_attn: attn_sink {tuple(attn_sink.shape)}, expected ({H},)")
        sink = attn_sink.float().contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.numel() == 0:
        return out
    qc = _strided(q, 4, 8)
    dt = _X_DT[q.dtype]
    ws = bt.new_empty(_attn_workspace(dev, B, S, H, Hkv, D, dt) // 4)
    _call(dev, _lib.load().bs_cache_attn, qc.data_ptr(), dt, B, S, H, Hkv, D, _I64x3(*qc.stride()[:3]),
          k_cache.data_ptr(), _ptr(v_cache), k_scale.data_ptr(), _ptr(v_scale), k_cache.size(0), k_cache.size(2),
          bt.data_ptr(), bt.size(1), sl.data_ptr(), _ptr(nl), _ptr(sink), softmax_scale, out.data_ptr(), ws.data_ptr(),
          4 * ws.numel())
    _tally("cache_attn", t0)
    return out
