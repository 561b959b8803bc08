"""Serving operators around the block-scaled products: their inputs, plain forms and 64-bit definitions.

Four operators, in the order in which a decoder layer meets them:

  rms     residual addition and RMS norm; the result in e4m3 with one scale for each 128 values (what
          fp8_gemm and fp4_gemm take), or in the input's type
  rope    rotary positions on part of each head, interleaved or half layout, angles exact at far positions
  append  new keys and values into a paged e4m3 cache with one power-of-two scale for each page and head
  attn    attention of each sequence's newest tokens over that cache (grouped heads, ragged lengths, or one
          latent that is both key and value), with an optional sink logit for each head

``own`` chooses between the plain form (elementary torch operations) and this package's entry points.
"""

import importlib
import math
import random

import torch

own = False

_PKG = "deepseek-v4-experimental-platform-on-dgx-spark_b200"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
_pkg = None


def _package():
    global _pkg
    if _pkg is None:
        _pkg = importlib.import_module(_PKG)
    return _pkg


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of one sequence: latency
        {"name": "rms_decode", "op": "rms", "rows": 1, "hidden": 4096, "dtype": "bf16", "residual": True, "quant": "f32"},
        # a long prompt at the widest hidden size of the quantiser benchmarks
        {"name": "rms_prefill", "op": "rms", "rows": 16384, "hidden": 7168, "dtype": "bf16", "residual": True,
         "quant": "f32"},
        # a ragged batch of f16 activations, power-of-two scales for the tensor cores' own scaling
        {"name": "rms_ragged_f16", "op": "rms", "rows": 1999, "hidden": 5120, "dtype": "f16", "residual": False,
         "quant": "ue8m0"},
        # decode of 64 sequences, 64 heads of 512 with the last 64 dims rotated, positions up to 2^20
        {"name": "rope_decode", "op": "rope", "tokens": 64, "heads": 64, "dim": 512, "rope": 64, "offset": 448,
         "layout": "interleaved", "dtype": "bf16", "far": 1 << 20},
        # prefill of query and key heads of 128 together, whole head, half layout
        {"name": "rope_prefill", "op": "rope", "tokens": 8192, "heads": 40, "dim": 128, "rope": 128, "offset": 0,
         "layout": "half", "dtype": "bf16", "far": 1 << 17},
        # one new token for each of 128 sequences, somewhere inside a page
        {"name": "append_decode", "op": "append", "batch": 128, "new": 1, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "shared": False, "longest": 2048, "lens_seed": 1},
        # prompts of odd lengths written behind what the cache holds
        {"name": "append_prefill", "op": "append", "batch": 4, "new": 4001, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "shared": False, "longest": 2048, "lens_seed": 2},
        # one short conversation: latency
        {"name": "attn_short", "op": "attn", "batch": 1, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "shared": False, "sink": False, "longest": 1000, "lens_seed": 3},
        # a serving batch of very different lengths
        {"name": "attn_ragged", "op": "attn", "batch": 64, "new": 1, "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "shared": False, "sink": False, "longest": 16384, "lens_seed": 4},
        # one long document, f16
        {"name": "attn_long_f16", "op": "attn", "batch": 1, "new": 1, "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 128, "dtype": "f16", "shared": False, "sink": False, "longest": 200000, "lens_seed": 5},
        # decode over a shared latent (key and value in one) with sink logits
        {"name": "attn_latent", "op": "attn", "batch": 48, "new": 1, "heads": 64, "kv_heads": 1, "dim": 512,
         "page": 64, "dtype": "bf16", "shared": True, "sink": True, "longest": 8192, "lens_seed": 6},
        # a chunk of a prompt on top of a cached prefix
        {"name": "attn_chunk", "op": "attn", "batch": 2, "new": 512, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "shared": False, "sink": False, "longest": 8192, "lens_seed": 7},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms", "rope", "append", "attn", "attn"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "rms":
        hidden = 128 * rng.randint(4, 64)
        return {"op": op, "rows": _log(rng, 1, (100 << 20) // hidden), "hidden": hidden,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "residual": rng.random() < 0.6,
                "quant": rng.choice(["f32", "ue8m0", "none"])}
    if op == "rope":
        dim = rng.choice([64, 128, 192, 256, 512])
        rope = rng.choice([r for r in (32, 64, 128, 192, 256) if r <= dim])
        heads = rng.randint(1, 64)
        return {"op": op, "tokens": _log(rng, 1, (40 << 20) // (heads * dim)), "heads": heads, "dim": dim, "rope": rope,
                "offset": rng.choice([0, dim - rope]), "layout": rng.choice(["interleaved", "half"]),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "far": 1 << rng.randint(10, 20)}
    shared = rng.random() < 0.25
    dim = rng.choice([256, 512]) if shared else rng.choice([64, 128, 192, 256])
    kv = 1 if shared else rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    case = {"op": op, "kv_heads": kv, "dim": dim, "page": page, "dtype": dtype, "shared": shared,
            "lens_seed": rng.randrange(1 << 20)}
    if op == "append":
        new = _log(rng, 1, 4000)
        room = (16 << 20) // (new * kv * dim)
        return {**case, "batch": _log(rng, 1, max(1, min(128, room))), "new": new, "longest": rng.randint(1, 2048)}
    group = rng.choice([16, 32, 64]) if shared else rng.choice([1, 2, 4, 5, 8, 16])
    batch = _log(rng, 1, 64)
    room = (256 << 20) // (batch * kv * dim * (1 if shared else 2))
    longest = _log(rng, 1, max(1, min(100000, room)))
    new = 1 if rng.random() < 0.6 else _log(rng, 1, max(1, min(256, longest, (64 << 20) // (batch * kv * group * longest))))
    return {**case, "batch": batch, "new": new, "heads": kv * group, "sink": rng.random() < 0.4, "longest": longest}


def _lens(case):
    """Cached lengths of a batch (for attn with the new tokens, for append before them): the longest first, the rest spread."""
    r = random.Random(case["lens_seed"])
    least = case["new"] if case["op"] == "attn" else 0
    longest = max(case["longest"], least)
    return [longest] + [r.randint(least, longest) for _ in range(case["batch"] - 1)]


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _codes(g, *shape):
    """Codes of normal data whose largest values are near the end of the e4m3 range."""
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        flat[at:at + n] = (torch.randn(n, generator=g, device="cuda") * 80.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return out


def _cache(g, case, lens):
    """A paged cache that holds more pages than the batch uses, in a random order; unused table entries are -1."""
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    used = [(n + page - 1) // page for n in lens]
    total = sum(used) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(max(used), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    st = {"block_table": table, "k_cache": _codes(g, total, kv, page, dim), "v_cache": None, "v_scale": None}
    st["k_scale"] = torch.exp2(torch.randint(-9, -6, (total, kv), generator=g, device="cuda").float())
    if not case["shared"]:
        st["v_cache"] = _codes(g, total, kv, page, dim)
        st["v_scale"] = torch.exp2(torch.randint(-9, -6, (total, kv), generator=g, device="cuda").float())
    return st


def _freqs(n, far):
    """Angle for each position step of n pairs, in 64 bits, stretched smoothly for long contexts (pairs that turn slowly
    are slowed by 8, pairs that turn quickly keep their frequency)."""
    i = torch.arange(n, dtype=torch.float64)
    f = 10000.0 ** (-i / n)
    keep = 1.0 - ((i - 0.3 * n) / (0.3 * n)).clamp(0.0, 1.0)
    return (f * keep + f / 8.0 * (1.0 - keep) if far > 4096 else f).cuda()


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    dt = _DT[case["dtype"]]
    if case["op"] == "rms":
        st["x"] = _normal(g, case["rows"], case["hidden"], dtype=dt)
        st["res"] = _normal(g, case["rows"], case["hidden"], dtype=dt, scale=3.0) if case["residual"] else None
        st["w"] = (1.0 + 0.2 * _normal(g, case["hidden"])).to(dt)
    elif case["op"] == "rope":
        st["x"] = _normal(g, 1, case["tokens"], case["heads"], case["dim"], dtype=dt)
        st["pos"] = torch.randint(0, case["far"], (1, case["tokens"]), generator=g, device="cuda")
        st["freqs"] = _freqs(case["rope"] // 2, case["far"])
    else:
        lens = _lens(case)
        new = case["new"]
        st.update(_cache(g, case, [n + new for n in lens] if case["op"] == "append" else lens))
        st["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
        if case["op"] == "append":
            shape = (case["batch"], new, case["kv_heads"], case["dim"])
            st["k"] = _normal(g, *shape, dtype=dt)
            st["v"] = None if case["shared"] else _normal(g, *shape, dtype=dt)
        else:
            # rows of different sharpness
            st["q"] = (_normal(g, case["batch"], new, case["heads"], case["dim"])
                       * (0.5 + 2.5 * torch.rand(case["batch"], new, case["heads"], 1, generator=g, device="cuda"))).to(dt)
            st["sink"] = _normal(g, case["heads"]) if case["sink"] else None
            st["softmax_scale"] = case["dim"] ** -0.5
    return st


# ------------------------------------------------------------------ plain forms

def _plain_rms(st):
    x, res, w = st["x"], st["res"], st["w"].float()
    out = {}
    h = x
    if res is not None:
        h = (x.float() + res.float()).to(x.dtype)          # the residual stream keeps its type
        out["h"] = h
    h = h.float()
    # the mean in 64 bits: a block's largest value decides its scale, and may lie next to a power of two
    r = torch.rsqrt(h.double().square().mean(-1, keepdim=True) + _EPS)
    y = h.double() * r * w.double()
    if st["quant"] == "none":
        out["y"] = y.to(x.dtype)
        return out
    blk = y.view(y.shape[0], -1, 128)
    s = blk.abs().amax(-1).clamp(min=1e-4) / 448.0
    if st["quant"] == "ue8m0":
        s = torch.exp2(torch.ceil(torch.log2(s)))
    s = s.float()
    out["y"] = (blk.float() / s[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(y.shape)
    out["s"] = s.to(torch.float8_e8m0fnu) if st["quant"] == "ue8m0" else s
    return out


def _plain_rope(st):
    x, o, n = st["x"], st["offset"], st["rope"]
    a = st["pos"].double()[..., None, None] * st["freqs"]      # [1, T, 1, n/2] in 64 bits: far positions
    c, s = torch.cos(a).float(), torch.sin(a).float()
    part = x[..., o:o + n].float()
    if st["layout"] == "interleaved":
        u, v = part[..., 0::2], part[..., 1::2]
        rot = torch.stack((u * c - v * s, u * s + v * c), dim=-1).flatten(-2)
    else:
        u, v = part[..., :n // 2], part[..., n // 2:]
        rot = torch.cat((u * c - v * s, u * s + v * c), dim=-1)
    return torch.cat((x[..., :o], rot.to(x.dtype), x[..., o + n:]), dim=-1)


def _plain_append_one(new, cache, scale, st):
    """new [B, S, Hkv, D] behind each sequence's cached tokens.  A page's scale is a power of two that holds its largest
    value; when it grows, the codes before the new ones are rounded again; a page whose first slot is written starts anew.
    Slots behind the new tokens stay as they were."""
    B, S, H, D = new.shape
    page = st["page"]
    first = st["lens"].long() // page                                            # first page touched
    P = (S + page - 2) // page + 1                                               # pages touched at most
    slots = (first[:, None] + torch.arange(P, device="cuda")) * page             # [B, P] position of each page's slot 0
    pos = slots[..., None] + torch.arange(page, device="cuda")                   # [B, P, page]
    src = pos - st["lens"].long()[:, None, None]
    fresh = (src >= 0) & (src < S)
    live = fresh.any(-1)                                                         # pages that get a token
    b, p = torch.nonzero(live, as_tuple=True)
    ids = st["block_table"].long()[b, first[b] + p]                              # [N]
    src, fresh, slots = src[b, p], fresh[b, p], slots[b, p]
    x = new.float()[b[:, None], src.clamp(0, S - 1)].permute(0, 2, 1, 3)         # [N, H, page, D]
    fr = fresh[:, None, :, None]
    amax = (x.abs() * fr).amax((-1, -2)).clamp(min=1e-4)                         # [N, H]
    want = torch.exp2(torch.ceil(torch.log2(amax.double() / 448.0))).float()
    kept = (slots < st["lens"].long()[b])[:, None]                               # slot 0 was there before
    old = scale[ids]
    s = torch.where(kept, torch.maximum(old, want), want)
    was = cache[ids].float()
    again = (was * (torch.where(kept, old, s) / s)[..., None, None]).to(torch.float8_e4m3fn).float()
    put = (x / s[..., None, None]).clamp(-448.0, 448.0)
    before = (src < 0)[:, None, :, None]
    cache[ids] = torch.where(fr, put, torch.where(before, again, was)).to(torch.float8_e4m3fn)
    scale[ids] = s


def _plain_append(st):
    _plain_append_one(st["k"], st["k_cache"], st["k_scale"], st)
    if not st["shared"]:
        _plain_append_one(st["v"], st["v_cache"], st["v_scale"], st)
    return {k: st[k] for k in ("k_cache", "k_scale", "v_cache", "v_scale") if st[k] is not None}


def _plain_dequant(cache, scale, table):
    x = cache[table].float() * scale[table][..., None, None]                    # [B, P, Hkv, page, D]
    B, P, H, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, P * page, D)


def _plain_attn(st):
    q, lens = st["q"], st["lens"].long()
    B, S, H, D = q.shape
    kv = st["kv_heads"]
    G = H // kv
    table = st["block_table"].long().clamp(min=0)
    k = _plain_dequant(st["k_cache"], st["k_scale"], table)
    v = k if st["shared"] else _plain_dequant(st["v_cache"], st["v_scale"], table)
    N = k.shape[2]
    qr = q.float().view(B, S, kv, G, D).permute(0, 2, 1, 3, 4).reshape(B, kv, S * G, D)
    sc = torch.matmul(qr, k.transpose(-1, -2)).mul_(st["softmax_scale"]).view(B, kv, S, G, N)
    limit = lens[:, None] - S + 1 + torch.arange(S, device="cuda")              # keys that each new token sees
    hide = torch.arange(N, device="cuda") >= limit[..., None]                   # [B, S, N]
    sc.masked_fill_(hide[:, None, :, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    if st["sink"] is not None:
        m = torch.maximum(m, st["sink"].view(1, kv, 1, G, 1))
    sc = sc.sub_(m).exp_()
    z = sc.sum(-1, keepdim=True)
    if st["sink"] is not None:
        z = z + torch.exp(st["sink"].view(1, kv, 1, G, 1) - m)
    o = torch.matmul(sc.view(B, kv, S * G, N), v).view(B, kv, S, G, D) / z
    return o.permute(0, 2, 1, 3, 4).reshape(B, S, H, D).to(q.dtype)


# ------------------------------------------------------------------ one pass

def run(st):
    op = st["op"]
    if own:
        P = _package()
        if op == "rms":
            if st["quant"] == "none":
                got = P.rms_norm(st["x"], st["w"], _EPS, residual=st["res"])
                return {"y": got} if st["res"] is None else {"y": got[0], "h": got[1]}
            pow2 = st["quant"] == "ue8m0"
            got = P.rms_norm_quant(st["x"], st["w"], _EPS, residual=st["res"], scale_fmt="ue8m0" if pow2 else None,
                                   scale_dtype=torch.float8_e8m0fnu if pow2 else torch.float32)
            return dict(zip(("y", "s", "h"), got))
        if op == "rope":
            return P.rope(st["x"], st["pos"], st["freqs"], layout=st["layout"], offset=st["offset"])
        if op == "append":
            P.cache_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"],
                           st["block_table"], st["lens"])
            return {k: st[k] for k in ("k_cache", "k_scale", "v_cache", "v_scale") if st[k] is not None}
        return P.cache_attn(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"], st["block_table"],
                            st["lens"], st["softmax_scale"], attn_sink=st["sink"])
    return {"rms": _plain_rms, "rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}[op](st)


def work(case):
    w = _BYTES[case["dtype"]]
    if case["op"] == "rms":
        n = case["rows"] * case["hidden"]
        each = w + (2 * w if case["residual"] else 0)                           # x; residual in, h out
        each += w if case["quant"] == "none" else 1 + (4 if case["quant"] == "f32" else 1) / 128
        return {"bytes": int(n * each) + case["hidden"] * w, "flops": 6 * n}
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * w + case["tokens"] * 8 + case["rope"] * 4, "flops": 3 * n * case["rope"]}
    lens, kv, dim, page = _lens(case), case["kv_heads"], case["dim"], case["page"]
    both = 1 if case["shared"] else 2
    if case["op"] == "append":
        n = case["batch"] * case["new"] * kv * dim * both
        pages = sum((a + case["new"] - 1) // page - a // page + 1 for a in lens)
        return {"bytes": n * (w + 1) + pages * kv * both * 4 + pages * 4, "flops": 3 * n}
    S = case["new"]
    seen = sum(n * S - S * (S - 1) // 2 for n in lens)                          # (query token, key) pairs
    read = sum(lens) * kv * dim * both
    pages = sum((n + page - 1) // page for n in lens)
    return {"bytes": read + pages * kv * both * 4 + pages * 4 + 2 * case["batch"] * S * case["heads"] * dim * w,
            "flops": 4 * seen * case["heads"] * dim}


# ------------------------------------------------------------------ definitions in 64 bits

def _e4m3(x):
    """Nearest e4m3 value (ties to the even mantissa) of 64-bit numbers of magnitude up to 448."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _pow2_scale(amax):
    return torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-4) / 448.0)))


def _exact_rms(st):
    x = st["x"].double()
    out = {}
    if st["res"] is not None:
        out["h"] = x + st["res"].double()
        x = out["h"].to(st["x"].dtype).double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * st["w"].double()
    if st["quant"] == "none":
        return {**out, "y": y}
    blk = y.unflatten(-1, (-1, 128))
    top = blk.abs().amax(-1)
    s = _pow2_scale(top) if st["quant"] == "ue8m0" else top.clamp(min=1e-4) / 448.0
    return {**out, "y": _e4m3(blk / s[..., None]).flatten(-2), "s": s}


def _exact_rope(st):
    x = st["x"].double()
    o, n = st["offset"], st["rope"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), st["pos"].double()[..., None] * st["freqs"])
    if st["layout"] == "interleaved":
        z = torch.view_as_complex(x[..., o:o + n].unflatten(-1, (-1, 2)).contiguous())
        x[..., o:o + n] = torch.view_as_real(z * turn[..., None, :]).flatten(-2)
    else:
        z = torch.complex(x[..., o:o + n // 2], x[..., o + n // 2:o + n]) * turn[..., None, :]
        x[..., o:o + n // 2], x[..., o + n // 2:o + n] = z.real, z.imag
    return x


def _exact_append(case, st):
    if case["batch"] * case["new"] > 20000:
        return None
    page, S = case["page"], case["new"]
    out = {}
    for name, new in (("k", st["k"]), ("v", st["v"])):
        if new is None:
            continue
        codes, scale = st[name + "_cache"].double(), st[name + "_scale"].double()
        for b, n in enumerate(_lens(case)):
            for j in range(n // page, (n + S - 1) // page + 1):
                a, z = max(n, j * page), min(n + S, (j + 1) * page)              # positions written in this page
                i = int(st["block_table"][b, j])
                x = new[b, a - n:z - n].double().transpose(0, 1)                 # [H, m, D]
                s = _pow2_scale(x.abs().amax((-1, -2)))
                if a > j * page:
                    s = torch.maximum(s, scale[i])
                    m = a - j * page
                    codes[i, :, :m] = _e4m3(codes[i, :, :m] * (scale[i] / s)[:, None, None])
                codes[i, :, a - j * page:z - j * page] = _e4m3(x / s[:, None, None])
                scale[i] = s
        out[name + "_cache"], out[name + "_scale"] = codes, scale
    return out


def _exact_attn(case, st):
    S, G = case["new"], case["heads"] // case["kv_heads"]
    out = []
    for b, n in enumerate(_lens(case)):
        ids = st["block_table"][b, :(n + case["page"] - 1) // case["page"]].long()
        rows = []
        for h in range(case["kv_heads"]):
            k = (st["k_cache"][ids, h].double() * st["k_scale"][ids, h].double()[:, None, None]).flatten(0, 1)[:n]
            v = k
            if not case["shared"]:
                v = (st["v_cache"][ids, h].double() * st["v_scale"][ids, h].double()[:, None, None]).flatten(0, 1)[:n]
            q = st["q"][b, :, h * G:(h + 1) * G].double().reshape(S * G, -1)
            a = q @ k.T * st["softmax_scale"]
            see = torch.arange(n, device="cuda")[None] <= n - S + torch.arange(S, device="cuda")[:, None]
            a = torch.where(see.repeat_interleave(G, 0), a, -math.inf)
            if st["sink"] is not None:
                s = st["sink"][h * G:(h + 1) * G].double().repeat(S)[:, None]
                a = torch.cat((a, s), -1)
                v = torch.cat((v, torch.zeros_like(v[:1])), 0)
            rows.append((torch.softmax(a, -1) @ v).view(S, G, -1))
        out.append(torch.cat(rows, 1))
    return torch.stack(out)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rms":
        return _exact_rms(st)
    if case["op"] == "rope":
        return _exact_rope(st)
    return _exact_append(case, st) if case["op"] == "append" else _exact_attn(case, st)
