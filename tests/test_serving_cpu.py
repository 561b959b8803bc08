"""Serving operators without a GPU: refusals of the C ABI (before any CUDA call) and of the Python entry points, and the
rotary frequencies."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from conftest import import_pkg


@pytest.fixture(scope="module")
def lib():
    pkg = import_pkg()
    from importlib import import_module
    import_module(pkg.__name__ + ".build").build()
    return pkg._lib.load()


L = import_pkg()._lib
FAKE = ctypes.c_void_p(1 << 20)          # aligned, never read: every call below is refused or empty
S3 = ctypes.c_int64 * 3


def norm(lib, dtype=1, rows=4, H=256, eps=1e-6, x=FAKE, res=None, h=None, y=FAKE):
    return lib.bs_rms_norm(x, res, FAKE, dtype, rows, H, eps, h, y, None)


def norm_quant(lib, H=256, rows=4, s_dtype=0, s=FAKE, x=FAKE):
    return lib.bs_rms_norm_quant(x, None, FAKE, 1, rows, H, 1e-6, 0, None, FAKE, s, s_dtype, None)


def test_norm_refusals(lib):
    assert norm(lib, dtype=3) == L.BS_ERR_INVALID_ARG and b"dtype" in lib.bs_last_error()
    assert norm(lib, rows=-1) == L.BS_ERR_INVALID_ARG
    assert norm(lib, H=0) == L.BS_ERR_INVALID_ARG
    assert norm(lib, H=252) == L.BS_ERR_UNSUPPORTED
    assert norm(lib, H=16392) == L.BS_ERR_UNSUPPORTED
    assert norm(lib, rows=2 ** 31) == L.BS_ERR_UNSUPPORTED
    assert norm(lib, eps=float("nan")) == L.BS_ERR_INVALID_ARG
    assert norm(lib, x=None) == L.BS_ERR_INVALID_ARG
    assert norm(lib, res=FAKE, h=None) == L.BS_ERR_INVALID_ARG
    assert norm(lib, x=ctypes.c_void_p((1 << 20) + 8)) == L.BS_ERR_INVALID_ARG
    assert norm(lib, rows=0, x=None, y=None) == L.BS_OK
    assert norm_quant(lib, H=264) == L.BS_ERR_UNSUPPORTED
    assert norm_quant(lib, s_dtype=1) == L.BS_ERR_UNSUPPORTED
    assert norm_quant(lib, s=None) == L.BS_ERR_INVALID_ARG
    assert norm_quant(lib, rows=0, x=None) == L.BS_OK


def rope(lib, dtype=1, tokens=2, H=2, D=128, n=64, offset=0, stride=256, x=FAKE, pos=FAKE):
    return lib.bs_rope(x, dtype, tokens, H, D, stride, D, pos, 1, FAKE, n, offset, 0, 0, 1.0, FAKE, stride, D, None)


def test_rope_refusals(lib):
    assert rope(lib, dtype=4) == L.BS_ERR_INVALID_ARG
    assert rope(lib, offset=72) == L.BS_ERR_INVALID_ARG            # past the head's end
    assert rope(lib, offset=-8) == L.BS_ERR_INVALID_ARG
    assert rope(lib, n=24) == L.BS_ERR_UNSUPPORTED
    assert rope(lib, n=528, D=1024, stride=2048) == L.BS_ERR_UNSUPPORTED
    assert rope(lib, offset=4) == L.BS_ERR_UNSUPPORTED
    assert rope(lib, D=132, stride=264) == L.BS_ERR_UNSUPPORTED
    assert rope(lib, H=70000) == L.BS_ERR_UNSUPPORTED
    assert rope(lib, stride=260) == L.BS_ERR_INVALID_ARG           # breaks 16-byte vectors
    assert rope(lib, x=None) == L.BS_ERR_INVALID_ARG
    assert rope(lib, pos=ctypes.c_void_p((1 << 20) + 4)) == L.BS_ERR_INVALID_ARG
    assert rope(lib, tokens=0, x=None) == L.BS_OK


def append(lib, dtype=1, B=1, S=1, Hkv=1, D=64, page=16, n_pages=4, max_pages=4, k=FAKE, v=None, v_cache=None, strides=(64, 64, 64)):
    return lib.bs_cache_append(k, v, dtype, B, S, Hkv, D, S3(*strides), S3(*strides), FAKE, v_cache, FAKE, v_cache, n_pages, page,
                               FAKE, max_pages, FAKE, None, None)


def test_append_refusals(lib):
    assert append(lib, dtype=3) == L.BS_ERR_INVALID_ARG
    assert append(lib, S=0) == L.BS_ERR_INVALID_ARG
    assert append(lib, n_pages=0) == L.BS_ERR_INVALID_ARG
    assert append(lib, page=24) == L.BS_ERR_UNSUPPORTED
    assert append(lib, page=256) == L.BS_ERR_UNSUPPORTED
    assert append(lib, D=72) == L.BS_ERR_UNSUPPORTED
    assert append(lib, D=528) == L.BS_ERR_UNSUPPORTED
    assert append(lib, n_pages=2 ** 31) == L.BS_ERR_UNSUPPORTED
    assert append(lib, B=2 ** 30, Hkv=64) == L.BS_ERR_UNSUPPORTED
    assert append(lib, v=FAKE) == L.BS_ERR_INVALID_ARG             # values without a cache
    assert append(lib, strides=(64, 60, 64)) == L.BS_ERR_INVALID_ARG
    assert append(lib, k=None) == L.BS_ERR_INVALID_ARG
    assert append(lib, B=0, k=None) == L.BS_OK


def attn(lib, dtype=1, B=1, S=1, H=8, Hkv=1, D=128, page=64, n_pages=4, max_pages=4, q=FAKE, v=None, v_scale=None,
         strides=(1024, 1024, 128), ws=FAKE, ws_bytes=1 << 40, scale=0.1):
    return lib.bs_cache_attn(q, dtype, B, S, H, Hkv, D, S3(*strides), FAKE, v, FAKE, v_scale, n_pages, page, FAKE, max_pages, FAKE,
                             None, None, scale, FAKE, ws, ws_bytes, None)


def test_attn_refusals(lib):
    assert attn(lib, dtype=0) == L.BS_ERR_UNSUPPORTED
    assert attn(lib, H=7, Hkv=2) == L.BS_ERR_INVALID_ARG
    assert attn(lib, Hkv=0) == L.BS_ERR_INVALID_ARG
    assert attn(lib, S=0) == L.BS_ERR_INVALID_ARG
    assert attn(lib, D=100) == L.BS_ERR_UNSUPPORTED
    assert attn(lib, D=1024) == L.BS_ERR_UNSUPPORTED
    assert attn(lib, page=8) == L.BS_ERR_UNSUPPORTED
    assert attn(lib, n_pages=0) == L.BS_ERR_INVALID_ARG
    assert attn(lib, v=FAKE) == L.BS_ERR_INVALID_ARG               # values without their scales
    assert attn(lib, strides=(1024, 1024, 130)) == L.BS_ERR_INVALID_ARG
    assert attn(lib, ws_bytes=64) == L.BS_ERR_INVALID_ARG and b"needed" in lib.bs_last_error()
    assert attn(lib, ws=None) == L.BS_ERR_INVALID_ARG
    assert attn(lib, q=None) == L.BS_ERR_INVALID_ARG
    assert attn(lib, scale=float("inf")) == L.BS_ERR_INVALID_ARG and attn(lib, scale=float("nan")) == L.BS_ERR_INVALID_ARG
    assert attn(lib, B=2 ** 31) == L.BS_ERR_UNSUPPORTED
    assert attn(lib, B=2 ** 20, H=8 * 2 ** 12, Hkv=2 ** 12, max_pages=2 ** 20) == L.BS_ERR_UNSUPPORTED   # over 2^31 tiles
    assert attn(lib, B=0, q=None) == L.BS_OK
    assert lib.bs_cache_attn_workspace_size(1, 1, 8, 3, 128, 1) == 0
    assert lib.bs_cache_attn_workspace_size(4, 1, 8, 1, 128, 1) > 148 * 8 * 128 * 4


def test_cache_lengths_refused(lib):
    """Positions within a tile's reach of 2^31, where a tile's end would not be a 32-bit number; products past 64 bits."""
    for most in (2 ** 27 - 1, 2 ** 27 - 63, 2 ** 62):              # pages of 16: 2^31 - 16, 2^31 - 1008 tokens
        assert attn(lib, page=16, max_pages=most) == L.BS_ERR_UNSUPPORTED and b"pages per sequence" in lib.bs_last_error()
        assert append(lib, page=16, max_pages=most) == L.BS_ERR_UNSUPPORTED
    assert attn(lib, page=16, max_pages=2 ** 27 - 64, q=None) == L.BS_ERR_INVALID_ARG         # accepted up to the pointers
    assert append(lib, n_pages=2 ** 62, Hkv=4) == L.BS_ERR_UNSUPPORTED


def test_cpu_tensors_rejected(lib):
    pkg = import_pkg()
    x, w = torch.zeros(2, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    c, s = torch.zeros(2, 1, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(2, 1)
    for call in (lambda: pkg.rms_norm(x, w), lambda: pkg.rms_norm_quant(x, w),
                 lambda: pkg.rope(x.view(2, 4, 64), torch.zeros(2, dtype=torch.int64), pkg.rope_freqs(64, device="cpu")),
                 lambda: pkg.cache_append(torch.zeros(1, 1, 1, 64), None, c, None, s, None, i.view(1, 1), i),
                 lambda: pkg.cache_attn(torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), c, None, s, None, i.view(1, 1), i, 1.0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(NotImplementedError):
        pkg.rms_norm_quant(x, w, scale_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="layout"):
        pkg.rope(x.view(2, 4, 64), torch.zeros(2, dtype=torch.int64), pkg.rope_freqs(64, device="cpu"), layout="split")


def test_rope_freqs():
    pkg = import_pkg()
    f = pkg.rope_freqs(64, 10000.0, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert f.dtype == torch.float64 and torch.allclose(f, want, rtol=1e-14, atol=0)
    assert torch.allclose(pkg.rope_freqs(64, scaling="linear", factor=4.0, device="cpu"), f / 4, rtol=1e-14, atol=0)
    n = pkg.rope_freqs(64, scaling="ntk", factor=8.0, device="cpu")
    assert n[0] == f[0] and abs(float(n[-1] / f[-1]) * 8 - 1) < 1e-12
    y = pkg.rope_freqs(64, scaling="yarn", factor=40.0, original_max_position=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns > 40], f[turns > 40])                       # kept: well over beta_fast turns
    assert torch.allclose(y[turns < 0.8], f[turns < 0.8] / 40, rtol=1e-14, atol=0)
    assert ((y <= f) & (y >= f / 40 * (1 - 1e-12))).all() and (y[1:] <= y[:-1]).all()
    for bad in (dict(rope_dim=63), dict(rope_dim=0), dict(rope_dim=64, scaling="cubic"), dict(rope_dim=64, factor=0.5)):
        with pytest.raises(ValueError):
            pkg.rope_freqs(device="cpu", **bad)
