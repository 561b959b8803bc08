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

No operator here records a graph for autograd: results are detached from
inputs that require a gradient.  ``rope(..., inplace=True)`` refuses an x that
does while gradients are recorded; it and ``cache_append`` count as in-place
changes of the tensors that they write.
"""

from __future__ import annotations

import ctypes
import importlib
import math
import threading
import time as _time
from typing import Optional

import torch

from . import _lib
from .kernel import _tally

__all__ = ["rms_norm", "rms_norm_quant", "rope", "rope_freqs", "cache_append", "cache_attn"]

_lock = threading.Lock()
_mod = None
_ENTRY_POINTS = ("bs_rms_norm", "bs_rms_norm_quant", "bs_rope", "bs_cache_append", "bs_cache_attn",
                 "bs_cache_attn_workspace_size")


def _native():
    """The C++ host path (csrc/bind.cpp), calling the library that _lib loaded."""
    global _mod
    if _mod is None:
        with _lock:
            if _mod is None:
                lib = _lib.load()
                try:
                    mod = importlib.import_module("._native", __package__)
                except ImportError as e:
                    raise RuntimeError(f"the serving operators' host path (_native.so) cannot be loaded ({e}): build it "
                                       "with the package's build.py") from e
                mod.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRY_POINTS})
                _mod = mod
    return _mod


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """RMS norm over the last dim: ``y = h * weight / sqrt(mean(h^2) + eps)`` with ``h = x + residual``.

    x and residual [..., H] and weight [H] in one type (bf16, f16 or fp32), H a
    multiple of 8 up to 16384.  h is rounded to the type (it is the residual
    stream that the next layer reads) and the norm is taken of the rounded h;
    statistics and product are fp32, rounded once.  Returns ``y``, or ``(y, h)``
    with a residual.
    """
    t0 = _time.perf_counter()
    got = (_mod or _native()).rms(x, weight, eps, residual, False, False, False)
    if got[0]:
        _lib.check(got[0])
    _tally("rms_norm", t0)
    return got[1] if residual is None else got[1:]


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                   scale_fmt: Optional[str] = None, scale_dtype: torch.dtype = torch.float32):
    """:func:`rms_norm` with its result quantised as :func:`act_quant` does (blocks of 128, the same scale rules
    and ``scale_fmt``), from the fp32 values, without the round trip through memory in 16 bits.

    H a multiple of 128 up to 16384; ``scale_dtype`` torch.float32 or
    torch.float8_e8m0fnu.  Returns ``(codes, scales)``, or ``(codes, scales, h)``
    with a residual; codes and scales go to fp8_gemm / fp4_gemm.
    """
    t0 = _time.perf_counter()
    e8m0 = scale_dtype == torch.float8_e8m0fnu
    if not e8m0 and scale_dtype != torch.float32:
        raise NotImplementedError(f"rms_norm_quant: scale_dtype {scale_dtype} not supported")
    got = (_mod or _native()).rms(x, weight, eps, residual, True, scale_fmt is not None, e8m0)
    if got[0]:
        _lib.check(got[0])
    _tally("rms_norm_quant", t0)
    return got[1:]


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
    if layout not in ("interleaved", "half"):
        raise ValueError(f"rope: layout {layout!r}: expected 'interleaved' or 'half'")
    status, out = (_mod or _native()).rope(x, positions, freqs, layout == "half", offset, inverse, scale, inplace)
    if status:
        _lib.check(status)
    _tally("rope", t0)
    return x if inplace else out


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
    status = (_mod or _native()).append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, start, new_lens)
    if status:
        _lib.check(status)
    _tally("cache_append", t0)


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

    Softmax weights enter the product with the values rounded to about the
    result's type (2^-8 of a weight at most with bf16, 2^-12 with f16).  Among
    the 128 tokens of a tile, those that count less than 2^-20 (f16: 2^-24) of
    the largest one may be lost; what they weigh in the denominator stays.
    """
    t0 = _time.perf_counter()
    status, out = (_mod or _native()).attn(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale,
                                           attn_sink, new_lens)
    if status:
        _lib.check(status)
    _tally("cache_attn", t0)
    return out
