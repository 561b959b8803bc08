"""Serving operators (norm, rope, cache append, cache attention) on the GPU against 64-bit definitions.

Tolerances, derived from the kernels' arithmetic:

  norm    fp32 statistics: a thread adds up to 64 squares in a chain and a tree of 10 joins them, so the sum is off by
          at most 74 x 2^-24, its root by half of that; root, quotient and two products add 4 x 2^-24: 2^-18 in all.
          The output's rounding: eps / 2 of its type.  Codes: half a step of e4m3 (2^-4 of the value, 2^-10 of the
          scale below the normal range) on top.
  rope    the angle is rounded once, as a fraction of a turn, to fp32: 2 pi 2^-25; sincospi is within 2 ulp and the
          two products and the sum round once each: 2^-20 (|u| + |v|) covers them.  The output's rounding: eps / 2.
  append  exact.
  attn    serving_ref.attn_tolerance.
"""

from __future__ import annotations

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.fixture(autouse=True)
def no_device_error(pkg):
    yield
    pkg._lib.device_error_check()


# ------------------------------------------------------------------ norm

NORM = [(1, 4096, "bf16", True), (3, 128, "bf16", False), (7, 7168, "bf16", True), (130, 5120, "f16", False),
        (5, 16384, "bf16", True), (33, 640, "f32", True), (2, 16384, "f32", False), (1000, 2304, "f16", True),
        (4, 10368, "bf16", False), (1, 8192, "f16", True), (2500, 4096, "bf16", True), (3001, 640, "f16", False),
        (2400, 8192, "f32", False), (2369, 128, "bf16", True), (4800, 1024, "f32", True)]


def _norm_inputs(rows, H, dt, res, seed=0):
    g = gen(rows * 7 + H + seed)
    x = randn(g, rows, H, dtype=DT[dt])
    r = randn(g, rows, H, dtype=DT[dt], scale=2.0) if res else None
    w = (1 + 0.3 * randn(g, H)).to(DT[dt])
    h = x if r is None else (x.float() + r.float()).to(DT[dt])
    return x, r, w, h


@pytest.mark.parametrize("rows,H,dt,res", NORM)
def test_rms_norm(pkg, rows, H, dt, res):
    x, r, w, h = _norm_inputs(rows, H, dt, res)
    got = pkg.rms_norm(x, w, 1e-6, residual=r)
    y = got if r is None else got[0]
    if r is not None:
        assert torch.equal(got[1], h)
    want = ref.rms(h, w, 1e-6)
    tol = want.abs() * (torch.finfo(DT[dt]).eps / 2 + 2.0 ** -18) + (2.0 ** -25 if dt == "f16" else 0.0)
    assert y.dtype == DT[dt] and ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("rows,H,dt,res", NORM)
@pytest.mark.parametrize("pow2", [False, True])
def test_rms_norm_quant(pkg, rows, H, dt, res, pow2):
    x, r, w, h = _norm_inputs(rows, H, dt, res, 1)
    if rows > 2:
        x[1] = 0
        if r is not None:
            r[1] = 0
        h = x if r is None else (x.float() + r.float()).to(DT[dt])
    sdt = torch.float8_e8m0fnu if pow2 and rows % 2 else torch.float32
    got = pkg.rms_norm_quant(x, w, 1e-6, residual=r, scale_fmt="ue8m0" if pow2 else None, scale_dtype=sdt)
    y, s = got[:2]
    if r is not None:
        assert torch.equal(got[2], h)
    assert y.dtype == torch.float8_e4m3fn and s.dtype == sdt and s.shape == (rows, H // 128)
    want = ref.rms(h, w, 1e-6).view(rows, -1, 128)
    s = s.to(torch.float32).double()
    floor = float(torch.tensor(1e-4, dtype=torch.float32))
    base = want.abs().amax(-1).clamp(min=floor) / 448.0
    if pow2:
        assert (torch.frexp(s.float())[0] == 0.5).all()
        assert (s >= base * (1 - 2.0 ** -17)).all() and (s / 2 < base * (1 + 2.0 ** -17)).all()
    else:
        assert ((s - base).abs() <= base * 2.0 ** -17).all()
    val = y.to(torch.float32).double().view(rows, -1, 128) * s[..., None]
    half = torch.maximum(want.abs() * 2.0 ** -4, s[..., None] * 2.0 ** -10)
    assert ((val - want).abs() <= half * (1 + 2.0 ** -12) + want.abs() * 2.0 ** -17).all()


def test_rms_norm_values(pkg):
    """Zero rows, tiny and huge values, NaN and inf stay in their own row."""
    x = torch.ones(6, 256, dtype=torch.bfloat16, device="cuda")
    x[0] = 0
    x[1] *= 1e-20
    x[2] *= 1e15
    x[3, 5] = float("nan")
    x[4, 200] = float("inf")
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    y = pkg.rms_norm(x, w, 1e-6)
    assert (y[0] == 0).all() and torch.isfinite(y[[0, 1, 2, 5]].float()).all() and y[3].isnan().all()
    assert ((y[2].float() - 1).abs() < 2 ** -7).all()
    c, s = pkg.rms_norm_quant(x, w, 1e-6)
    assert torch.isfinite(c[[0, 1, 2, 5]].float()).all() and torch.isfinite(s[[0, 1, 2, 5]]).all()
    assert s[3].isnan().all()
    assert (c[0].float() == 0).all()


def test_rms_norm_empty_and_strided(pkg):
    w = torch.ones(256, dtype=torch.float16, device="cuda")
    assert pkg.rms_norm(torch.empty(0, 256, dtype=torch.float16, device="cuda"), w).shape == (0, 256)
    x = randn(gen(3), 5, 4, 512, dtype=torch.float16)[:, :, 100:356]
    want = ref.rms(x, w, 1e-6)
    assert ((pkg.rms_norm(x, w).double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25).all()


# ------------------------------------------------------------------ rope

@pytest.mark.parametrize("shape,n,offset,layout,dt", [
    ((1, 1, 1, 64), 64, 0, "interleaved", "bf16"), ((3, 5, 128), 128, 0, "half", "bf16"), ((2, 3, 64, 512), 64, 448, "interleaved", "bf16"),
    ((17, 40, 128), 32, 64, "half", "f16"), ((9, 7, 192), 64, 128, "interleaved", "f32"), ((2, 2, 3, 512), 512, 0, "half", "f32"),
    ((300, 1, 576), 64, 512, "interleaved", "f16"), ((5, 3, 104), 48, 8, "half", "f32"), ((5, 3, 104), 80, 24, "interleaved", "bf16"),
    ((70, 64, 512), 512, 0, "interleaved", "bf16")])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(pkg, shape, n, offset, layout, dt, inverse):
    g = gen(sum(shape) + n)
    x = randn(g, *shape, dtype=DT[dt])
    lead = shape[:-2]
    pos = torch.randint(0, 1 << 20, lead, generator=g, device="cuda")
    if inverse:
        pos = pos.to(torch.int32)
    else:
        pos[..., :1] = -5
    freqs = pkg.rope_freqs(n, 10000.0, "yarn", 16.0)
    sc = 1.25 if inverse else 1.0
    got = pkg.rope(x, pos, freqs, layout=layout, offset=offset, inverse=inverse, scale=sc)
    want = ref.rope(x, pos, freqs, layout, offset, inverse, sc)
    mag = x.double().abs()
    part = mag[..., offset:offset + n]
    if layout == "half":
        both = part[..., :n // 2] + part[..., n // 2:]
        both = torch.cat((both, both), -1)
    else:
        both = (part[..., 0::2] + part[..., 1::2]).repeat_interleave(2, -1)
    tol = want.abs() * torch.finfo(DT[dt]).eps / 2
    tol[..., offset:offset + n] += both * 2.0 ** -20 * sc + (2.0 ** -25 if dt == "f16" else 0.0)
    assert got.dtype == x.dtype and ((got.double() - want).abs() <= tol).all()
    rest = [i for i in range(shape[-1]) if not offset <= i < offset + n]
    assert torch.equal(got[..., rest], x[..., rest])
    y = x.clone()
    assert pkg.rope(y, pos, freqs, layout=layout, offset=offset, inverse=inverse, scale=sc, inplace=True) is y
    assert torch.equal(y, got)


def test_rope_gradient(pkg):
    """The backward turn is the gradient of the forward one: against the formula, and against differences."""
    g = gen(5)
    x, go = randn(g, 6, 3, 128), randn(g, 6, 3, 128)
    pos = torch.randint(0, 5000, (6,), generator=g, device="cuda")
    f = pkg.rope_freqs(64)
    xd = x.double().requires_grad_(True)
    (gr,) = torch.autograd.grad((ref.rope(xd, pos, f, "half", 32) * go.double()).sum(), xd)
    got = pkg.rope(go, pos, f, layout="half", offset=32, inverse=True)
    assert ((got.double() - gr).abs() <= gr.abs() * 2.0 ** -24 + 2.0 ** -20 * 8).all()
    d = randn(g, 6, 3, 128)
    # the turn is linear: a difference of two calls is the call on the difference, to rounding
    step = (pkg.rope(x + d, pos, f, layout="half", offset=32) - pkg.rope(x - d, pos, f, layout="half", offset=32)).double() / 2
    assert abs(float((step * go.double()).sum() - (got.double() * d.double()).sum())) < 2304 * 2.0 ** -18


def test_rope_strided_view(pkg):
    """Query and key heads inside a fused projection's output, in place; the rest of the row is untouched."""
    qkv = randn(gen(6), 9, 3 * 4 * 64, dtype=torch.bfloat16)
    was = qkv.clone()
    pos = torch.arange(9, device="cuda")
    f = pkg.rope_freqs(64)
    view = qkv[:, :8 * 64].view(9, 8, 64)
    pkg.rope(view, pos, f, inplace=True)
    want = pkg.rope(was[:, :8 * 64].view(9, 8, 64).contiguous(), pos, f)
    assert torch.equal(view, want) and torch.equal(qkv[:, 8 * 64:], was[:, 8 * 64:])


# ------------------------------------------------------------------ cache

def make_cache(g, n_pages, Hkv, page, D, shared=False):
    def one():
        codes = (torch.randn(n_pages, Hkv, page, D, generator=g, device="cuda") * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
        return codes, torch.exp2(torch.randint(-10, -5, (n_pages, Hkv), generator=g, device="cuda").float())
    k, ks = one()
    if shared:
        return k, None, ks, None
    v, vs = one()
    return k, v, ks, vs


def make_table(g, lens, page, extra=2):
    used = [max(0, (n + page - 1) // page) for n in lens]
    order = torch.randperm(sum(used) + extra, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(max(used), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(used) + extra


def same_codes(a, b):
    a, b = a.float().double(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("starts,S,Hkv,D,page,dt,shared", [
    ([0], 1, 1, 128, 64, "bf16", False), ([0, 1, 63, 64, 65], 1, 2, 128, 64, "bf16", False), ([5, 0, 130], 200, 3, 64, 16, "f16", False),
    ([127, 128, 3], 7, 1, 512, 128, "bf16", True), ([0, 31, 40], 33, 4, 192, 32, "f32", False), ([17], 1000, 2, 16, 128, "f16", False),
    ([9] * 70, 2, 1, 80, 16, "f32", True)])
def test_cache_append(pkg, starts, S, Hkv, D, page, dt, shared):
    g = gen(S + D + page)
    table, n_pages = make_table(g, [n + S for n in starts], page)
    k_cache, v_cache, ks, vs = make_cache(g, n_pages, Hkv, page, D, shared)
    # values of very different size: some pages' scales grow, some do not
    size = torch.exp2(torch.randint(-6, 7, (len(starts), S, Hkv, 1), generator=g, device="cuda").float())
    k = (randn(g, len(starts), S, Hkv, D) * size).to(DT[dt])
    v = None if shared else (randn(g, len(starts), S, Hkv, D) / size).to(DT[dt])
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    want_k = ref.append(k, k_cache.float(), ks, table, start)
    want_v = None if shared else ref.append(v, v_cache.float(), vs, table, start)
    pkg.cache_append(k, v, k_cache, v_cache, ks, vs, table, start)
    assert same_codes(k_cache, want_k[0]) and torch.equal(ks.double(), want_k[1])
    if not shared:
        assert same_codes(v_cache, want_v[0]) and torch.equal(vs.double(), want_v[1])


def test_cache_append_token_by_token(pkg):
    """Many single-token calls, ragged, strided sources, with non-finite values: the definition applied call by call."""
    g = gen(11)
    starts, page, Hkv, D = [0, 14, 37], 16, 2, 64
    table, n_pages = make_table(g, [n + 40 for n in starts], page)
    k_cache, v_cache, ks, vs = make_cache(g, n_pages, Hkv, page, D)
    wk, wv = (k_cache.float().double(), ks.double()), (v_cache.float().double(), vs.double())
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    for step in range(20):
        kv = randn(g, 3, 2, 2 * Hkv, D, dtype=torch.bfloat16, scale=2.0 ** (step % 7 - 3))
        if step == 6:
            kv[0, 0, 1, 3], kv[1, 0, 2, 5] = float("inf"), float("nan")
        nl = torch.tensor([1, step % 2, 1 + step % 2], dtype=torch.int32, device="cuda")
        k, v = kv[:, :, :Hkv], kv[:, :, Hkv:]
        wk = ref.append(k, *wk, table, start, nl)
        wv = ref.append(v, *wv, table, start, nl)
        pkg.cache_append(k, v, k_cache, v_cache, ks, vs, table, start, nl)
        start = start + nl
        assert same_codes(k_cache, wk[0]) and torch.equal(ks.double(), wk[1])
        assert same_codes(v_cache, wv[0]) and torch.equal(vs.double(), wv[1])


def test_cache_append_bad_index(pkg):
    """Page indices and lengths out of range write nothing and are reported."""
    g = gen(12)
    k_cache, _, ks, _ = make_cache(g, 4, 1, 16, 64, True)
    k = randn(g, 5, 1, 1, 64, dtype=torch.bfloat16)
    was, was_s = k_cache.clone(), ks.clone()
    table = torch.tensor([[4], [-1], [1], [2], [3]], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 3, 16, -1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    pkg.cache_append(k, None, k_cache, None, ks, None, table, start)
    with pytest.raises(pkg._lib.BsError, match="out of range"):
        pkg._lib.device_error_check()
    assert torch.equal(k_cache.view(torch.uint8), was.view(torch.uint8)) and torch.equal(ks, was_s)


def run_attn(pkg, lens, S, H, Hkv, D, page, dt, shared=False, sink=False, new_lens=None, seed=0, q_scale=1.5):
    g = gen(seed + sum(lens) + S * H + D)
    table, n_pages = make_table(g, lens, page)
    cache = make_cache(g, n_pages, Hkv, page, D, shared)
    q = (randn(g, len(lens), S, H, D) * q_scale).to(DT[dt])
    sk = randn(g, H) if sink else None
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    nl = None if new_lens is None else torch.tensor(new_lens, dtype=torch.int32, device="cuda")
    args = (q, *cache, table, sl, D ** -0.5)
    got = pkg.cache_attn(*args, attn_sink=sk, new_lens=nl)
    want, bound = ref.attn(*args, sink=sk, new_lens=nl)
    tol = ref.attn_tolerance(DT[dt], D, want, bound)
    err = (got.double() - want).abs()
    print(f"worst error / tolerance {float((err / tol).max()):.3f}, rel. Frobenius {float(err.norm() / want.norm()):.2e}")
    assert got.dtype == DT[dt] and torch.isfinite(got.float()).all() and (err <= tol).all()
    return args, sk, nl, got


ATTN = [
    # lens, S, H, Hkv, D, page, dtype, shared, sink
    ([1], 1, 8, 1, 128, 64, "bf16", False, False),
    ([128], 1, 8, 1, 128, 128, "bf16", False, False),
    ([100, 1, 257], 1, 32, 8, 128, 64, "bf16", False, True),
    ([1000], 1, 32, 8, 128, 16, "f16", False, False),
    ([700, 129], 1, 16, 2, 64, 32, "bf16", False, False),
    ([513], 1, 5, 5, 16, 16, "f16", False, True),
    ([300, 600], 1, 48, 4, 192, 64, "bf16", False, False),
    ([300, 31], 1, 24, 2, 256, 32, "f16", False, False),
    ([400, 90], 1, 16, 1, 512, 64, "bf16", True, True),
    ([640], 1, 64, 1, 512, 128, "bf16", True, False),
    ([333, 64], 1, 64, 1, 512, 64, "f16", True, True),
    ([200], 2, 20, 1, 384, 64, "bf16", False, False),
    ([200], 1, 20, 1, 320, 64, "f16", True, False),
    ([200], 3, 40, 2, 512, 32, "bf16", False, True),
    ([260, 9], 9, 8, 2, 128, 64, "bf16", False, False),
    ([150, 70], 40, 16, 2, 128, 16, "f16", False, True),
    ([128, 300, 65], 65, 32, 4, 128, 64, "bf16", False, True),
    ([200], 200, 6, 3, 64, 128, "bf16", False, False),
    ([90], 90, 2, 2, 256, 64, "bf16", False, False),
]


# enough tokens that every CTA works through many tiles of several sequences
ATTN_LONG = [
    ([9000, 7777, 1, 128, 4000, 6001], 1, 32, 8, 128, 64, "bf16", False, False),
    ([20000, 17], 1, 64, 8, 128, 128, "f16", False, True),
    ([5000] * 7 + [4999], 1, 64, 4, 128, 32, "bf16", False, False),
    ([9001, 8000], 1, 96, 8, 64, 16, "f16", False, False),
    ([30000, 20000], 1, 64, 2, 128, 64, "bf16", False, True),
    ([30000, 20000], 1, 48, 2, 112, 64, "f16", False, False),
    ([30000, 123], 33, 8, 4, 128, 64, "bf16", False, False),
    ([12000, 12345], 1, 24, 8, 256, 64, "bf16", False, False),
    ([12000, 12345], 1, 64, 4, 256, 128, "f16", False, False),
    ([9999, 10000], 1, 32, 4, 384, 64, "bf16", False, False),
    ([8000, 9000, 300], 1, 64, 2, 512, 64, "bf16", False, False),
    ([8000, 9000, 300], 1, 16, 2, 512, 16, "f16", False, False),
    ([20000, 15000, 1, 40000], 1, 64, 1, 512, 64, "bf16", True, True),
    ([20000, 15000, 40000], 1, 8, 1, 512, 128, "bf16", True, False),
    ([20000, 15000, 40000], 1, 64, 1, 512, 64, "f16", True, False),
]


@pytest.mark.parametrize("case", ATTN + ATTN_LONG, ids=lambda c: "-".join(str(x) for x in c).replace(" ", ""))
def test_cache_attn(pkg, case):
    run_attn(pkg, *case)
