"""Serving operators on the GPU where calls of the usual shapes do not look: segments that follow one another quickly,
weights far below a row's largest, values at the ends of the types' ranges, scales that are no numbers."""

from __future__ import annotations

import ctypes

import pytest
import torch

import serving_ref as ref
from test_serving_gpu import DT, gen, make_cache, make_table, randn, same_codes

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_device_error(pkg):
    yield
    pkg._lib.device_error_check()


def attn_into(pkg, out, ws, q, cache, table, sl, scale):
    """cache_attn through the C ABI, into memory that the caller filled."""
    L, lib = pkg._lib, pkg._lib.load()
    B, S, H, D = q.shape
    k, v, ks, vs = cache
    ptr = lambda t: None if t is None else t.data_ptr()
    L.check(lib.bs_cache_attn(q.data_ptr(), L.DT_BF16 if q.dtype == torch.bfloat16 else L.DT_F16, B, S, H, k.shape[1], D,
                              (ctypes.c_int64 * 3)(*q.stride()[:3]), k.data_ptr(), ptr(v), ks.data_ptr(), ptr(vs),
                              k.shape[0], k.shape[2], table.data_ptr(), table.shape[1], sl.data_ptr(), None, None, scale,
                              out.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("B,S,H,Hkv,D,dt,shared", [
    (256, 1, 64, 8, 128, "bf16", False),          # 8 rows a tile, 7 heads of one tile after another in a CTA
    (256, 1, 128, 8, 128, "f16", False), (200, 16, 32, 8, 128, "bf16", False), (200, 8, 32, 8, 64, "f16", False),
    (320, 1, 64, 1, 512, "bf16", True),           # one buffer of query rows
    (160, 1, 64, 4, 256, "bf16", False), (160, 1, 16, 4, 512, "f16", False)])
def test_cache_attn_quick_segments(pkg, B, S, H, Hkv, D, dt, shared):
    """Many heads of one tile each in every CTA: each row is written, at its own place, with the same bits every time, and
    with the bits of calls whose CTAs have one head at most (a tile is never split, so the arithmetic is the same)."""
    g = gen(B + S + D)
    lens = torch.randint(S, 129, (B,), generator=g, device="cuda").tolist()
    table, n = make_table(g, lens, 64)
    cache = make_cache(g, n, Hkv, 64, D, shared)
    q = randn(g, B, S, H, D, dtype=DT[dt])
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    few = 148 // (2 * Hkv)
    want = torch.cat([pkg.cache_attn(q[b:b + few], *cache, table[b:b + few], sl[b:b + few], D ** -0.5) for b in range(0, B, few)])
    size = pkg._lib.load().bs_cache_attn_workspace_size(B, S, H, Hkv, D, pkg._lib.DT_BF16 if dt == "bf16" else pkg._lib.DT_F16)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    for _ in range(40):
        out.fill_(float("nan"))
        attn_into(pkg, out, ws, q, cache, table, sl, D ** -0.5)
        assert torch.equal(out, want)
