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


def test_rms_norm_unaligned_and_in_place(pkg):
    """Inputs that start off a 16-byte boundary are copied; the C entry point may write h over x or the residual."""
    g = gen(9)
    flat = randn(g, 4 * 256 + 3, dtype=torch.bfloat16)
    x, w = flat[3:].view(4, 256), torch.ones(257, dtype=torch.bfloat16, device="cuda")[1:]
    assert torch.equal(pkg.rms_norm(x, w, residual=x)[0], pkg.rms_norm(x.clone(), w.clone(), residual=x.clone())[0])
    L, st = pkg._lib, torch.cuda.current_stream().cuda_stream
    for rows in (5, 3000):                       # both forms of the kernel
        x, r = randn(g, rows, 1024, dtype=torch.bfloat16), randn(g, rows, 1024, dtype=torch.bfloat16)
        w = torch.ones(1024, dtype=torch.bfloat16, device="cuda")
        y, h = pkg.rms_norm(x, w, residual=r)
        for into in (0, 1):
            a, b = x.clone(), r.clone()
            got = torch.empty_like(y)
            L.check(L.load().bs_rms_norm(a.data_ptr(), b.data_ptr(), w.data_ptr(), L.DT_BF16, rows, 1024, 1e-6,
                                         (b if into else a).data_ptr(), got.data_ptr(), st))
            assert torch.equal(got, y) and torch.equal(b if into else a, h)


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


# ------------------------------------------------------------------ cache attention: what goes wrong at the edges

def check(pkg, q, cache, table, lens, scale=None, sink=None, new_lens=None):
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    nl = None if new_lens is None else torch.tensor(new_lens, dtype=torch.int32, device="cuda")
    got = pkg.cache_attn(q, *cache, table, sl, scale, attn_sink=sink, new_lens=nl)
    want, bound = ref.attn(q, *cache, table, sl, scale, sink=sink, new_lens=nl)
    tol = ref.attn_tolerance(q.dtype, D, want, bound)
    assert ((got.double() - want).abs() <= tol).all()
    return got


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("S", [1, 5])
def test_cache_attn_empty_rows(pkg, dt, S):
    """Sequences without tokens, shorter than their new tokens, padded queries: zero rows, the others right."""
    g = gen(21 + S)
    lens = [0, 300, 2, 129, 0, 1]
    table, n = make_table(g, lens, 32)
    cache = make_cache(g, n, 2, 32, 64)
    q = randn(g, 6, S, 8, 64, dtype=DT[dt])
    got = check(pkg, q, cache, table, lens)
    assert (got[0] == 0).all() and (got[4] == 0).all()
    if S > 2:
        assert (got[2, :S - 2] == 0).all() and (got[2, S - 2:] != 0).any()
    new = [min(S, x) for x in (3, 1, 2, 0, 5, 1)]
    got = check(pkg, q, cache, table, lens, new_lens=new)
    for b, m in enumerate(new):
        assert (got[b, m:] == 0).all()
    sink = randn(g, 8)
    got = check(pkg, q, cache, table, lens, sink=sink)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("page,H,Hkv,D,shared", [(16, 8, 2, 64, False), (64, 64, 1, 512, True), (128, 64, 2, 128, False),
                                                 (32, 12, 1, 256, False), (64, 20, 1, 320, True)])
@pytest.mark.parametrize("S", [1, 9])
def test_cache_attn_nan_in_hidden_slots(pkg, page, H, Hkv, D, shared, S):
    """What lies behind a sequence's tokens (unwritten slots of its last page, here NaN codes) reaches no row; a NaN in
    a new token reaches the rows that see it, in its dims (values) or wholly (keys), and no other."""
    g = gen(page + H + S)
    lens = [page * 3 + 7, 140, page]
    table, n = make_table(g, lens, page)
    cache = make_cache(g, n, Hkv, page, D, shared)
    q = randn(g, 3, S, H, D, dtype=torch.bfloat16)
    clean = check(pkg, q, cache, table, lens)
    dirty = [None if t is None else t.clone() for t in cache]
    for codes in dirty[:2]:
        if codes is not None:
            raw = codes.view(torch.uint8)
            for b, m in enumerate(lens):
                if m % page:
                    raw[table[b, m // page].long(), :, m % page:] = 0x7F
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = pkg.cache_attn(q, *dirty, table, sl, D ** -0.5)
    assert torch.equal(got, clean)
    if S == 1:
        return
    # the fourth new token of sequence 1, kv head 0: dims 3 and D - 1 of its value
    at = lens[1] - S + 3
    i = table[1, at // page].long()
    codes = dirty[0] if shared else dirty[1]
    codes.view(torch.uint8)[i, 0, at % page, 3] = 0xFF
    codes.view(torch.uint8)[i, 0, at % page, D - 1] = 0x7F
    got = pkg.cache_attn(q, *dirty, table, sl, D ** -0.5)
    G = H // Hkv
    bad = torch.zeros_like(got, dtype=torch.bool)
    if shared:
        bad[1, 3:, :G] = True                     # a NaN key is a NaN score
    else:
        bad[1, 3:, :G, 3] = True
        bad[1, 3:, :G, D - 1] = True
    assert torch.equal(got.isnan(), bad)
    assert torch.equal(got[~bad], clean[~bad])


def test_cache_attn_odd_queries(pkg):
    """Rows of zeros, infinities and NaN stay their own; huge and tiny rows; scales of either sign and zero; sinks of
    any size; queries inside a wider projection and at an odd offset."""
    g = gen(31)
    lens = [500, 77]
    table, n = make_table(g, lens, 64)
    cache = make_cache(g, n, 2, 64, 128)
    q = randn(g, 2, 3, 8, 128, dtype=torch.bfloat16)
    q[0, 0, 0] = 0
    q[0, 0, 1] *= 1e-30
    q[0, 1, 2] *= 100
    check(pkg, q, cache, table, lens)
    check(pkg, q, cache, table, lens, scale=-0.05)
    got = check(pkg, q, cache, table, lens, scale=0.0)
    sink = torch.tensor([-float("inf"), -100.0, 0.0, 5.0, 30.0, 80.0, -3e38, 3.0], device="cuda")
    check(pkg, q, cache, table, lens, sink=sink)
    clean = pkg.cache_attn(q, *cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 0.1)
    q2 = q.clone()
    q2[0, 1, 4, 7], q2[1, 2, 0, 127] = float("inf"), float("nan")
    got = pkg.cache_attn(q2, *cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 0.1)
    bad = torch.zeros(2, 3, 8, dtype=torch.bool, device="cuda")
    bad[0, 1, 4] = bad[1, 2, 0] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], clean[~bad])
    wide = torch.zeros(2, 3, 3 * 8 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    for off in (1024, 1028, 1025):               # aligned, 8-byte aligned, neither (copied)
        view = wide[..., off:off + 1024].view(2, 3, 8, 128) if off % 4 == 0 else wide[..., off:off + 1024].unflatten(-1, (8, 128))
        view.copy_(q)
        assert torch.equal(pkg.cache_attn(view, *cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 0.1), clean)


def test_cache_attn_scales(pkg):
    """Page scales of any size, not only powers of two; a page of zeros; a value scale of zero and of very different pages."""
    g = gen(41)
    lens = [700]
    table, n = make_table(g, lens, 16)
    k, v, ks, vs = make_cache(g, n, 4, 16, 64)
    ks.mul_(torch.rand(ks.shape, generator=g, device="cuda") + 0.5)
    vs.copy_(torch.exp2(torch.randint(-30, 10, vs.shape, generator=g, device="cuda").float()) * 1.7)
    vs[table[0, 3].long()] = 0
    k.view(torch.uint8)[table[0, 5].long()] = 0
    check(pkg, randn(g, 1, 1, 16, 64, dtype=torch.float16), (k, v, ks, vs), table, lens)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("H,Hkv,D,dt,which", [(8, 2, 64, "bf16", "v"), (8, 2, 128, "f16", "v"), (64, 2, 128, "bf16", "k"),
                                              (16, 1, 512, "bf16", "shared"), (32, 2, 128, "bf16", "v")])
@pytest.mark.parametrize("n,S,i", [(134, 9, 128), (150, 25, 144), (134, 1, 128)])
def test_cache_attn_nan_scale(pkg, page, H, Hkv, D, dt, which, n, S, i):
    """A page whose scale is NaN (here the one that holds token i, kv head 0) reaches the rows that see a token of it,
    whether or not its tile has other pages, and no row that does not."""
    g = gen(page + H + n)
    table, n_pages = make_table(g, [n], page)
    cache = make_cache(g, n_pages, Hkv, page, D, which == "shared")
    q = randn(g, 1, S, H, D, dtype=DT[dt])
    sl = torch.tensor([n], dtype=torch.int32, device="cuda")
    want, bound = ref.attn(q, *cache, table, sl, D ** -0.5)
    tol = ref.attn_tolerance(DT[dt], D, want, bound)
    (cache[3] if which == "v" else cache[2])[table[0, i // page].long(), 0] = float("nan")
    got = pkg.cache_attn(q, *cache, table, sl, D ** -0.5)
    sees = n - S + 1 + torch.arange(S, device="cuda") > i // page * page
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, sees, :H // Hkv] = True
    assert torch.equal(got.isnan(), bad)
    assert ((got.double() - want).abs() <= tol)[~bad].all()


def test_cache_attn_many_sequences(pkg):
    """More (sequence, row tile) pairs than threads of a CTA, and many empty sequences among them."""
    g = gen(51)
    lens = [int(x) for x in torch.randint(-200, 300, (1500,), generator=g, device="cuda").clamp(min=0).tolist()]
    table, n = make_table(g, lens, 16)
    cache = make_cache(g, n, 1, 16, 32)
    check(pkg, randn(g, 1500, 1, 4, 32, dtype=torch.bfloat16), cache, table, lens)


def test_cache_beyond_32_bits(pkg):
    """Pages whose bytes lie beyond 2^32 in the cache: append and attention."""
    page, D, n = 128, 512, 66000                  # 4.3 GB
    k_cache = torch.zeros(n, 1, page, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ks = torch.ones(n, 1, device="cuda")
    g = gen(61)
    table = torch.tensor([[65999, 3, 65537], [32768, 65536, 1]], dtype=torch.int32, device="cuda")
    k = randn(g, 2, 300, 1, D, dtype=torch.bfloat16)
    start = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    pkg.cache_append(k, None, k_cache, None, ks, None, table, start)
    small = [65999, 3, 65537, 32768, 65536, 1]
    t2 = torch.tensor([[0, 1, 2], [3, 4, 5]], device="cuda")
    want, ws = ref.append(k, torch.zeros(6, 1, page, D, device="cuda"), torch.ones(6, 1, device="cuda"), t2, start)
    assert same_codes(k_cache[small], want) and torch.equal(ks[small].double(), ws)
    q = randn(g, 2, 1, 16, D, dtype=torch.bfloat16)
    lens = torch.tensor([300, 300], dtype=torch.int32, device="cuda")
    got = pkg.cache_attn(q, k_cache, None, ks, None, table, lens, D ** -0.5)
    near = pkg.cache_attn(q, k_cache[small], None, ks[small], None, t2.to(torch.int32), lens, D ** -0.5)
    assert torch.equal(got, near)


def test_cache_attn_bad_index(pkg):
    """Page indices and lengths out of range read as absent and are reported."""
    g = gen(71)
    lens = [200, 150]
    table, n = make_table(g, lens, 64)
    cache = make_cache(g, n, 2, 64, 64)
    q = randn(g, 2, 1, 4, 64, dtype=torch.bfloat16)
    bad = table.clone()
    bad[0, 1] = n
    bad[1, 2] = -7
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = pkg.cache_attn(q, *cache, bad, sl, 0.125)
    with pytest.raises(pkg._lib.BsError, match="out of range"):
        pkg._lib.device_error_check()
    # the same with those pages' tokens taken out
    t2 = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    t2[0] = table[0, [0, 2, 3]]
    t2[1, :2] = table[1, :2]
    check(pkg, q, cache, t2, [136, 128])
    want, bound = ref.attn(q, *cache, t2, torch.tensor([136, 128]), 0.125)
    assert ((got.double() - want).abs() <= ref.attn_tolerance(q.dtype, 64, want, bound)).all()
    got = pkg.cache_attn(q, *cache, table, torch.tensor([-1, 100000], dtype=torch.int32, device="cuda"), 0.125)
    with pytest.raises(pkg._lib.BsError, match="out of range"):
        pkg._lib.device_error_check()
    assert (got == 0).all()


def test_refusals(pkg):
    """Python-level refusals that need CUDA tensors."""
    g = gen(81)
    table, n = make_table(g, [40], 16)
    k, v, ks, vs = make_cache(g, n, 2, 16, 64)
    q = randn(g, 1, 1, 4, 64, dtype=torch.bfloat16)
    sl = torch.tensor([40], dtype=torch.int32, device="cuda")
    x, w = randn(g, 2, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16, device="cuda")
    pos, f = torch.zeros(1, 1, dtype=torch.int64, device="cuda"), pkg.rope_freqs(64)
    for err, call in [
            (TypeError, lambda: pkg.rms_norm(x, w.float())), (TypeError, lambda: pkg.rms_norm(x.double(), w.double())),
            (ValueError, lambda: pkg.rms_norm(x, w[:128])), (ValueError, lambda: pkg.rms_norm(x, w, residual=x[:1])),
            (ValueError, lambda: pkg.rms_norm(x, w.cpu())), (NotImplementedError, lambda: pkg.rms_norm_quant(x[:, :200], w[:200])),
            (TypeError, lambda: pkg.rope(q, pos.float(), f)), (TypeError, lambda: pkg.rope(q, pos, f.float())),
            (ValueError, lambda: pkg.rope(q, pos[0], f)), (ValueError, lambda: pkg.rope(q, pos, f, offset=8)),
            (NotImplementedError, lambda: pkg.rope(q, pos, f[:5])),
            (ValueError, lambda: pkg.rope(q.transpose(2, 3), pos, f, inplace=True)),
            (ValueError, lambda: pkg.rope(q.expand(1, 3, 4, 64), pos.expand(1, 3), f, inplace=True)),
            (ValueError, lambda: pkg.cache_attn(q, k, v, ks, vs, table, sl, float("nan"))),
            (TypeError, lambda: pkg.cache_attn(q.float(), k, v, ks, vs, table, sl, 1.0)),
            (TypeError, lambda: pkg.cache_attn(q, k, v, ks, vs, table.long(), sl, 1.0)),
            (TypeError, lambda: pkg.cache_attn(q, k.view(torch.uint8), v, ks, vs, table, sl, 1.0)),
            (ValueError, lambda: pkg.cache_attn(q, k, v, ks, None, table, sl, 1.0)),
            (ValueError, lambda: pkg.cache_attn(q[:, :, :3], k, v, ks, vs, table, sl, 1.0)),
            (ValueError, lambda: pkg.cache_attn(q, k, v, ks, vs, table, sl, 1.0, attn_sink=ks[0])),
            (ValueError, lambda: pkg.cache_attn(q, k[:, :, :, :32], v, ks, vs, table, sl, 1.0)),
            (ValueError, lambda: pkg.cache_attn(q, k, v, ks, vs, table, torch.cat((sl, sl)), 1.0)),
            (NotImplementedError, lambda: pkg.cache_attn(q, k[:, :, :8].contiguous(), v[:, :, :8].contiguous(), ks, vs, table, sl, 1.0)),
            (TypeError, lambda: pkg.cache_append(q, q.half(), k, v, ks, vs, table, sl)),
            (ValueError, lambda: pkg.cache_append(q, None, k, v, ks, vs, table, sl)),
            (ValueError, lambda: pkg.cache_append(q, q, k, v, ks, vs, table, sl)),
            (ValueError, lambda: pkg.cache_append(q[:, :, :2], q[:, :, :2], k, v, ks, vs[:1], table, sl))]:
        with pytest.raises(err):
            call()


# ------------------------------------------------------------------ streams, graphs, the same bits again

def serving_inputs(g, lens, page=64, Hkv=2, D=128, H=16, S=1):
    table, n = make_table(g, [x + S for x in lens], page)
    cache = make_cache(g, n, Hkv, page, D)
    return (randn(g, len(lens), S, H, D, dtype=torch.bfloat16), randn(g, len(lens), S, Hkv, D, dtype=torch.bfloat16),
            randn(g, len(lens), S, Hkv, D, dtype=torch.bfloat16), cache, table)


def test_same_bits_again(pkg):
    g = gen(91)
    lens = [5000, 1, 700, 12345]
    q, k, v, cache, table = serving_inputs(g, lens)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    first = pkg.cache_attn(q, *cache, table, sl, 0.1)
    for _ in range(20):
        assert torch.equal(pkg.cache_attn(q, *cache, table, sl, 0.1), first)


def test_graphs_and_streams(pkg):
    """One decode step captured twice (two graphs with memory of their own), replayed with new inputs and lengths, at once
    on two streams, against eager calls on a third."""
    P = pkg
    f = P.rope_freqs(128)

    class Step:
        def __init__(self, seed):
            g = gen(seed)
            self.lens = [900, 17, 300]
            self.q, self.k, self.v, (kc, vc, ks, vs), self.table = serving_inputs(g, [x + 30 for x in self.lens])
            self.cache = (kc, vc, ks, vs)
            self.start = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
            self.x, self.w = randn(g, 3, 1024, dtype=torch.bfloat16), torch.ones(1024, dtype=torch.bfloat16, device="cuda")

        def run(self, cache):
            y, s = P.rms_norm_quant(self.x, self.w)
            pos = self.start.view(3, 1)
            q = P.rope(self.q, pos, f)
            P.cache_append(P.rope(self.k, pos, f), self.v, cache[0], cache[1], cache[2], cache[3], self.table, self.start)
            return y, s, P.cache_attn(q, *cache, self.table, self.start + 1, 0.1)

    steps = [Step(1), Step(2)]
    graphs = []
    for st in steps:
        st.eager = [t.clone() for t in st.cache]
        st.run([t.clone() for t in st.cache])
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        keep = [t.clone() for t in st.cache]
        with torch.cuda.graph(gr):
            st.out = st.run(st.cache)
        for a, b in zip(st.cache, keep):
            a.copy_(b)
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    side = torch.cuda.Stream()
    for it in range(6):
        g = gen(100 + it)
        for st in steps:
            for t in (st.q, st.k, st.v, st.x):
                t.copy_(randn(g, *t.shape, dtype=t.dtype))
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        want = []
        with torch.cuda.stream(side):
            for st in steps:
                want.append(st.run(st.eager))
        torch.cuda.synchronize()
        for st, w in zip(steps, want):
            for a, b in zip(st.out, w):
                assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                                   b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
            for a, b in zip(st.cache, st.eager):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            st.start.add_(1)


def test_layer_step(pkg):
    """A decoder layer's attention half as it is used: norm into e4m3, the projection, rotary positions in place on its
    query and key heads, append, attention, for a prompt and then single tokens; against 64-bit operations on the stored
    codes at every step."""
    g = gen(7)
    B, Hd, H, Hkv, D, page = 2, 512, 8, 2, 64, 16
    qkv_rows = (H + 2 * Hkv) * D
    w = (1 + 0.1 * randn(g, Hd)).bfloat16()
    ws = torch.rand(qkv_rows // 128, Hd // 128, generator=g, device="cuda") * 1e-3 + 1e-4
    wq = (randn(g, qkv_rows, Hd) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    freqs = pkg.rope_freqs(32)
    lens = [0, 0]
    table, n = make_table(g, [60, 90], page)
    kc, vc, ks, vs = make_cache(g, n, Hkv, page, D)
    h = None
    for new in ([37, 50], [1, 1], [1, 1], [3, 2]):
        S = max(new)
        x = randn(g, B, S, Hd, dtype=torch.bfloat16)
        res = randn(g, B, S, Hd, dtype=torch.bfloat16) if h is None or h.shape[1] != S else h
        y, s, h = pkg.rms_norm_quant(x, w, residual=res)
        want = ref.rms((x.float() + res.float()).bfloat16(), w, 1e-6)
        deq = y.to(torch.float32).double().unflatten(-1, (-1, 128)) * s.double()[..., None]
        assert ((deq.flatten(-2) - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, s.double().repeat_interleave(128, -1) * 2.0 ** -10) * 1.01).all()
        qkv = pkg.fp8_gemm(y, s, wq, ws)
        exact = deq.flatten(-2) @ (wq.to(torch.float32).double() * ws.double().repeat_interleave(128, 0).repeat_interleave(128, 1)).T
        assert ((qkv.double() - exact).norm() / exact.norm()) < 1e-2
        heads = qkv.view(B, S, H + 2 * Hkv, D)
        start = torch.tensor(lens, dtype=torch.int32, device="cuda")
        pos = start.long()[:, None] + torch.arange(S, device="cuda")
        turned = ref.rope(heads[:, :, :H + Hkv], pos, freqs, "half", 0)
        pkg.rope(heads[:, :, :H + Hkv], pos, freqs, layout="half", inplace=True)
        assert ((heads[:, :, :H + Hkv].double() - turned).abs() <= turned.abs() * 2.0 ** -8 + heads.double().abs().amax() * 2.0 ** -19).all()
        q, k, v = heads[:, :, :H], heads[:, :, H:H + Hkv], heads[:, :, H + Hkv:]
        nl = torch.tensor(new, dtype=torch.int32, device="cuda")
        wk, wv = ref.append(k, kc.float(), ks, table, start, nl), ref.append(v, vc.float(), vs, table, start, nl)
        pkg.cache_append(k, v, kc, vc, ks, vs, table, start, nl)
        assert same_codes(kc, wk[0]) and torch.equal(ks.double(), wk[1]) and same_codes(vc, wv[0]) and torch.equal(vs.double(), wv[1])
        lens = [a + b for a, b in zip(lens, new)]
        check(pkg, q, (kc, vc, ks, vs), table, lens, scale=D ** -0.5 / 4, new_lens=new)
