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


# ------------------------------------------------------------------ weights far below a row's largest

def precise_tolerance(q, cache, table, n, scale, lims):
    """Reference and tolerance of one sequence and one kv head, rows [S x G], that do not grow with the longest context.

    A weight enters as two (bf16) or three (f16) e4m3 terms: 2^-8 or 2^-12 of itself, or, where it is too small for that,
    half the last term's smallest step, 2^-10 / 16 or / 256, on a scale where the largest weight x page scale that the row
    sees in the tile of 128 tokens is at least 256 / 4: 2^-20 or 2^-24 of that largest one (in tiles far below the row's
    maximum, of 2^-24 of that and the tile's largest scale), and never more than the weight itself.  Scores: an ulp (2^-23) of the sum of their magnitudes for each of terms x D products; the rest 2^-18; the
    result's own rounding.
    """
    S, H, D = q.shape[1:]
    page = cache[0].shape[2]
    ids = table[0, :(n + page - 1) // page].long()
    k = (cache[0][ids, 0].double() * cache[2][ids, 0].double()[:, None, None]).flatten(0, 1)[:n]
    code = cache[1][ids, 0].double().flatten(0, 1)[:n]
    vs = cache[3][ids, 0].double().repeat_interleave(page)[:n]
    qq = q[0].double()                                                     # [S, H, D]
    a = torch.einsum("shd,td->sht", qq, k) * scale
    see = torch.arange(n, device="cuda")[None, None] < torch.tensor(lims, device="cuda")[:, None, None]
    a = a.masked_fill(~see, -float("inf"))
    w = torch.exp(a - a.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    two = q.dtype == torch.bfloat16
    terms = (torch.einsum("shd,td->sht", qq.abs(), k.abs()) * see).amax(-1, keepdim=True) * scale
    d = (2 if two else 3) * D * 2.0 ** -23 * terms
    wv = w * vs.abs()
    pad = -n % 128
    tiles = torch.nn.functional.pad(wv, (0, pad)).unflatten(-1, (-1, 128))
    scales = torch.nn.functional.pad(vs.abs(), (0, pad)).unflatten(-1, (-1, 128)).amax(-1)[:, None]
    far = w.amax(-1, keepdim=True)[..., None] * scales * 2.0 ** -24
    least = (torch.maximum(tiles.amax(-1, keepdim=True), far) * (2.0 ** -20 if two else 2.0 ** -24)).expand_as(tiles).flatten(-2)[..., :n]
    out, mass = (w * vs) @ code, wv @ code.abs()
    small = torch.minimum(wv, least * see) @ code.abs()
    tol = (mass * ((2.0 ** -8 if two else 2.0 ** -12) + 2 * d + 2.0 ** -18) + small
           + (out.abs() + mass * d) * torch.finfo(q.dtype).eps / 2 + (0.0 if two else 2.0 ** -25) + 1e-30)
    return out, tol


def assert_precise(pkg, q, cache, table, n, scale, B=1):
    """B sequences over the same pages, with the same queries."""
    S = q.shape[1]
    sl = torch.full((B,), n, dtype=torch.int32, device="cuda")
    got = pkg.cache_attn(q.expand(B, -1, -1, -1), *cache, table.expand(B, -1), sl, scale).double()
    want, tol = precise_tolerance(q, cache, table, n, scale, [n - S + i + 1 for i in range(S)])
    err = (got - want).abs()
    print(f"worst error / tolerance {float((err / tol).max()):.3f}, rel. Frobenius {float(err.norm() / want.norm()):.2e}")
    assert (err <= tol).all()
    return err, want


@pytest.mark.parametrize("dt,S", [("bf16", 1), ("f16", 1), ("bf16", 16)])
@pytest.mark.parametrize("nats", [13.0, 15.0, 18.0, 20.0])
@pytest.mark.parametrize("at", [0, 7001])
def test_cache_attn_peak(pkg, dt, S, nats, at):
    """One key far above 20000 others whose value is zero: the result is the others', a few hundredths of the weight or
    less, and keeps its digits.  600 such sequences: a CTA has all of a head's tokens, so its maximum stays the peak's."""
    g = gen(int(nats) + S + at)
    n, page, H, D = 20000, 64, 4, 128
    table, n_pages = make_table(g, [n], page)
    codes = lambda: (torch.randn(n_pages, 1, page, D, generator=g, device="cuda") * 90).clamp(-448, 448)
    k, v = codes(), codes().abs()
    ks, vs = torch.full((n_pages, 1), 2.0 ** -7, device="cuda"), torch.full((n_pages, 1), 2.0 ** -8, device="cuda")
    base = torch.randn(D, generator=g, device="cuda").sign()
    q = (base + 0.1 * randn(g, 1, S, H, D)).to(DT[dt])
    p, slot = table[0, at // page].long(), at % page
    k[p], v[p, 0, slot] = 0, 0                    # a page of the peak's own, so that its scale sets the score
    k[p, 0, slot] = base
    scale = D ** -0.5
    ks[p] = nats / (D * scale)
    cache = (k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn), ks, vs)
    err, want = assert_precise(pkg, q, cache, table, n, scale, 600)
    # Over all outputs: weights off by 2^-8 (2^-12) and a rounding of 2^-9 (2^-12), doubled; and what shares a tile with the
    # peak may be lost whole.  Those 127 of n tokens weigh 1 (score 0 on the peak's page) or as the others do, 127 / n of
    # the result at most.
    assert err.norm() <= want.norm() * 600 ** 0.5 * ((2.0 ** -7 if dt == "bf16" else 2.0 ** -10) + 127 / n)


@pytest.mark.parametrize("dt,H,S,page", [("bf16", 4, 20, 16), ("f16", 4, 20, 16), ("bf16", 1, 7, 16), ("bf16", 2, 24, 32)])
def test_cache_attn_hidden_scale(pkg, dt, H, S, page):
    """A page that a row does not see, or hardly weighs, may have a value scale 2^24 times that of the pages it lives on:
    the row keeps its digits."""
    g = gen(H + S + page)
    n, D = 2 * page + 8, 128
    table, n_pages = make_table(g, [n], page)
    k, v, ks, vs = make_cache(g, n_pages, 1, page, D)
    ids = table[0].long()
    vs.fill_(2.0 ** -22)
    vs[ids[2]] = 4.0
    base = torch.randn(D, generator=g, device="cuda").sign()
    q = (base + 0.5 * randn(g, 1, S, H, D)).to(DT[dt])
    assert_precise(pkg, q, (k, v, ks, vs), table, n, D ** -0.5)
    k[ids[2]] = (-base).to(torch.float8_e4m3fn)                            # the last page 33 nats below
    ks[ids[2]] = 33.0 / (D * D ** -0.5)
    assert_precise(pkg, q, (k, v, ks, vs), table, n, D ** -0.5)
    vs[ids[1]] = 0.0
    assert_precise(pkg, q, (k, v, ks, vs), table, n, D ** -0.5)


@pytest.mark.parametrize("dt,H,S,D,page,n", [("bf16", 8, 1, 128, 16, 9000), ("f16", 16, 1, 64, 32, 5000), ("bf16", 8, 12, 128, 16, 700),
                                             ("bf16", 32, 1, 512, 64, 3000), ("f16", 4, 7, 256, 16, 650), ("bf16", 32, 1, 256, 128, 5000)])
@pytest.mark.parametrize("sharp", [1.0, 5.0])
def test_cache_attn_spread_scales(pkg, dt, H, S, D, page, n, sharp):
    """Value scales from 2^-22 to 2^3 beside each other, flat and sharp rows."""
    g = gen(H + S + n)
    table, n_pages = make_table(g, [n], page)
    k, v, ks, vs = make_cache(g, n_pages, 1, page, D)
    vs.copy_(torch.exp2(torch.randint(-22, 4, vs.shape, generator=g, device="cuda").float()))
    vs[table[0, 1].long()] *= -1.7
    q = (sharp * randn(g, 1, S, H, D)).to(DT[dt])
    assert_precise(pkg, q, (k, v, ks, vs), table, n, D ** -0.5)
    assert_precise(pkg, q, (k, v, ks, vs), table, n, D ** -0.5, 40)


# ------------------------------------------------------------------ norm: values of any size, calls of any number of rows

@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("rows,H", [(3, 512), (5, 7168), (700, 1024), (1500, 1024), (4000, 4096)])
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm_size_of_values(pkg, dt, rows, H, res):
    """Rows of 1e-30 to 1e37, whose squares leave fp32, beside ordinary ones, zeros, infinities and NaN, in every form."""
    g = gen(rows + H)
    big = dt != "f16"
    size = torch.tensor([1.0, 1e20, 1e30, 1e37, 1e-25, 1e-30, 0.0] if big else [1.0, 1e4, 3e-5, 1e-2, 0.0], device="cuda")
    x = (torch.randn(rows, H, generator=g, device="cuda") * size[torch.arange(rows, device="cuda") % len(size)][:, None]).to(DT[dt])
    r = torch.zeros_like(x) if res else None
    w = (1 + 0.1 * randn(g, H)).to(DT[dt])
    for eps in (1e-6, 0.0):
        got = pkg.rms_norm(x, w, eps, residual=r)
        y = got[0] if res else got
        want = ref.rms(x, w, eps)
        tol = want.abs() * (torch.finfo(DT[dt]).eps / 2 + 2.0 ** -18) + (2.0 ** -25 if dt == "f16" else 2.0 ** -126)
        dead = (x == 0).all(-1)                   # 0 / 0 without an eps
        ok = ~dead if eps == 0.0 else torch.ones_like(dead)
        assert ((y.double() - want).abs() <= tol)[ok].all()
        c, s = pkg.rms_norm_quant(x, w, eps, residual=r)[:2]
        deq = c.to(torch.float32).double().unflatten(-1, (-1, 128)) * s.double()[..., None]
        half = torch.maximum(want.abs() * 2.0 ** -4, s.double().repeat_interleave(128, -1) * 2.0 ** -10)
        assert ((deq.flatten(-2) - want).abs() <= half * (1 + 2.0 ** -12) + want.abs() * 2.0 ** -17)[ok].all()
    x[1, 7], x[2, 9] = float("inf"), float("nan")
    y = pkg.rms_norm(x, w, 1e-6)
    assert y[2].isnan().all() and y[1, 7].isnan() and (y[1, :7] == 0).all() and torch.isfinite(y[0]).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("H,res", [(1024, True), (4096, False), (5120, True)])
def test_rms_norm_row_alone(pkg, dt, H, res):
    """A row's result is the same in calls of any number of rows, whatever form of the kernel they take: its sum is the same
    sum of 8-square sums in fp64 up to their order, 2^-50 or so, which a rounding to 16 bits shows in one value of 2^40."""
    g = gen(H)
    rows = 6000
    x = randn(g, rows, H, dtype=DT[dt])
    r = randn(g, rows, H, dtype=DT[dt]) if res else None
    w = (1 + 0.2 * randn(g, H)).to(DT[dt])
    cut = lambda t, n: None if t is None else t[:n]
    y = pkg.rms_norm(x, w, residual=r)
    c = pkg.rms_norm_quant(x, w, residual=r)
    for n in (1, 200, 295, 296, 1000, 1199, 1200, 2500):
        for a, b in zip(pkg.rms_norm(cut(x, n), w, residual=cut(r, n)) if res else [pkg.rms_norm(x[:n], w)], y if res else [y]):
            assert torch.equal(a, b[:n])
        for a, b in zip(pkg.rms_norm_quant(cut(x, n), w, residual=cut(r, n)), c):
            assert torch.equal(a.view(torch.uint8), b[:n].view(torch.uint8))


# ------------------------------------------------------------------ cache append: scales that are no numbers

@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_cache_append_onto_bad_scale(pkg, dt, bad):
    """Tokens behind the first of a page whose scale is NaN or infinite do not turn its codes into numbers; a page begun anew
    forgets it."""
    g = gen(17)
    starts, page, Hkv, D, S = [5, 16, 30], 16, 2, 64, 9
    table, n_pages = make_table(g, [n + S for n in starts], page)
    k_cache, v_cache, ks, vs = make_cache(g, n_pages, Hkv, page, D)
    ks[table[0, 0].long(), 1] = bad
    vs[table[0, 0].long(), 0] = bad
    vs[table[1, 1].long()] = bad                  # written from slot 0 on
    ks[table[2, 1].long(), 0] = bad
    k, v = randn(g, 3, S, Hkv, D, dtype=DT[dt]), randn(g, 3, S, Hkv, D, dtype=DT[dt])
    k[0, 3, 1, 4] = float("inf")
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    wk, wv = ref.append(k, k_cache.float(), ks, table, start), ref.append(v, v_cache.float(), vs, table, start)
    pkg.cache_append(k, v, k_cache, v_cache, ks, vs, table, start)
    for codes, scale, want in ((k_cache, ks, wk), (v_cache, vs, wv)):
        assert same_codes(codes, want[0]) and torch.equal(scale.double().nan_to_num(-1.0, -2.0), want[1].nan_to_num(-1.0, -2.0))
    assert torch.isfinite(vs[table[1, 1].long()]).all()


# ------------------------------------------------------------------ autograd around the in-place operators

def test_in_place_changes_are_seen(pkg):
    """Tensors saved for a backward pass and then written here are noticed, as after torch's own in-place operators; an
    in-place turn of something that needs its gradient is refused; inference tensors and recording turned off are fine."""
    g = gen(5)
    f, pos = pkg.rope_freqs(64), torch.arange(4, device="cuda")
    x, w = randn(g, 4, 2, 64), randn(g, 4, 2, 64).requires_grad_()
    loss = (x * w).sum()
    pkg.rope(x, pos, f, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    y = w * 2
    for t in (w, y):
        was = t.detach().clone()
        with pytest.raises(ValueError, match="gradient"):
            pkg.rope(t, pos, f, inplace=True)
        assert torch.equal(t, was)
    with torch.no_grad():
        assert torch.equal(pkg.rope(y, pos, f, inplace=True), pkg.rope(w * 2, pos, f))
    assert not pkg.rope(w, pos, f).requires_grad
    table, n = make_table(g, [20], 16)
    cache = make_cache(g, n, 2, 16, 64)
    k = randn(g, 1, 3, 2, 64, dtype=torch.bfloat16)
    before = [t._version for t in cache]
    pkg.cache_append(k, k, cache[0], cache[1], cache[2], cache[3], table, torch.tensor([7], dtype=torch.int32, device="cuda"))
    assert all(t._version > b for t, b in zip(cache, before))
    with torch.inference_mode():
        c, s = cache[0].clone(), cache[2].clone()
        z = x.clone()
    pkg.cache_append(k, None, c, None, s, None, table, torch.tensor([0], dtype=torch.int32, device="cuda"))
    pkg.rope(z, pos, f, inplace=True)


@pytest.mark.parametrize("H,D,dt,S", [(4, 128, "bf16", 25), (8, 64, "f16", 9), (2, 512, "bf16", 25), (32, 128, "bf16", 3)])
def test_cache_attn_spread_scales_with_nan(pkg, H, D, dt, S):
    """Very different value scales, one of them zero and one NaN, on pages that some rows see: NaN reaches those rows alone."""
    g = gen(H + D)
    n, page, i = 150, 16, 144
    table, n_pages = make_table(g, [n], page)
    k, v, ks, vs = make_cache(g, n_pages, 1, page, D)
    vs.copy_(torch.exp2(torch.randint(-22, 4, vs.shape, generator=g, device="cuda").float()))
    vs[table[0, 8].long()] = 0.0
    q = randn(g, 1, S, H, D, dtype=DT[dt])
    want, tol = precise_tolerance(q, (k, v, ks, vs), table, n, D ** -0.5, [n - S + j + 1 for j in range(S)])
    vs[table[0, i // page].long()] = float("nan")
    got = pkg.cache_attn(q, k, v, ks, vs, table, torch.tensor([n], dtype=torch.int32, device="cuda"), D ** -0.5)[0].double()
    sees = n - S + 1 + torch.arange(S, device="cuda") > i
    assert got[sees].isnan().all() and ((got - want).abs() <= tol)[~sees].all()


@pytest.mark.parametrize("scale", [1.7 * 2.0 ** -100, 1.3 * 2.0 ** 90])
@pytest.mark.parametrize("n,B", [(300, 1), (9000, 40)])
def test_cache_attn_value_scales_far_from_one(pkg, scale, n, B):
    """Results of any size that bf16 holds."""
    g = gen(n)
    table, n_pages = make_table(g, [n], 64)
    k, v, ks, vs = make_cache(g, n_pages, 1, 64, 128)
    vs.mul_(scale * 2.0 ** 8)
    assert_precise(pkg, 2 * randn(g, 1, 2, 4, 128, dtype=torch.bfloat16), (k, v, ks, vs), table, n, 128 ** -0.5, B)
