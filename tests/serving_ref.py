"""Plain 64-bit definitions of the serving operators, for their tests (torch, any device)."""

from __future__ import annotations

import torch


def e4m3_nearest(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of float64 numbers (ties to the even code); beyond 448 clamped, NaN kept."""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.where(x.isnan(), x, torch.copysign(torch.round(a / step) * step, x))


def pow2_scale(amax: torch.Tensor) -> torch.Tensor:
    """Smallest power of two s with amax / s <= 448, amax at least 1e-4 (in fp32)."""
    a = amax.double().clamp(min=float(torch.tensor(1e-4, dtype=torch.float32)))
    return torch.exp2(torch.ceil(torch.log2(a / 448.0)))


def rms(h: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    h = h.double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))) * w.double()


def rope(x, pos, freqs, layout, offset, inverse=False, scale=1.0):
    x = x.double().clone()
    n = 2 * freqs.numel()
    a = pos.double()[..., None, None] * freqs
    c, s = torch.cos(a) * scale, torch.sin(a) * (-scale if inverse else scale)
    part = x[..., offset:offset + n]
    if layout == "interleaved":
        u, v = part[..., 0::2].clone(), part[..., 1::2].clone()
        part[..., 0::2], part[..., 1::2] = u * c - v * s, u * s + v * c
    else:
        u, v = part[..., :n // 2].clone(), part[..., n // 2:].clone()
        part[..., :n // 2], part[..., n // 2:] = u * c - v * s, u * s + v * c
    return x


def append(new, cache, scale, table, start, new_lens=None):
    """new [B, S, H, D] into cache [n, H, page, D] (float64 code values) / scale [n, H]; returns new ones."""
    cache, scale = cache.double().clone(), scale.double().clone()
    B, S = new.shape[:2]
    page = cache.shape[2]
    for b in range(B):
        n, m = int(start[b]), S if new_lens is None else int(new_lens[b])
        for j in range(n // page, (n + m - 1) // page + 1 if m else 0):
            lo, hi = max(n, j * page), min(n + m, (j + 1) * page)
            i, at = int(table[b, j]), lo - j * page
            x = new[b, lo - n:hi - n].double().transpose(0, 1)                      # [H, rows, D]
            fin = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))
            s = pow2_scale(fin.amax((-1, -2)))
            if at > 0:
                s = torch.maximum(s, scale[i])
                cache[i, :, :at] = e4m3_nearest(cache[i, :, :at] * (scale[i] / s)[:, None, None])
            x = torch.where(x.isfinite(), x, torch.full_like(x, float("nan")))
            cache[i, :, at:at + hi - lo] = e4m3_nearest(x / s[:, None, None])
            scale[i] = s
    return cache, scale


def attn(q, k_cache, v_cache, k_scale, v_scale, table, lens, softmax_scale, sink=None, new_lens=None):
    """Returns (out, bound): out [B, S, H, D] float64, and per output the sum of weights x |v|, the largest sum of
    |q k| terms of a score (times the scale) of its row, 1 / sum of weights relative to the largest, and the largest |v|."""
    B, S, H, D = q.shape
    Hkv = k_cache.shape[1]
    G = H // Hkv
    out = torch.zeros(B, S, H, D, dtype=torch.float64, device=q.device)
    mass, terms, inv, top = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    for b in range(B):
        n, m = int(lens[b]), S if new_lens is None else int(new_lens[b])
        page = k_cache.shape[2]
        ids = table[b, :(n + page - 1) // page].long()
        for h in range(Hkv):
            k = (k_cache[ids, h].double() * k_scale[ids, h].double()[:, None, None]).flatten(0, 1)
            v = k if v_cache is None else (v_cache[ids, h].double() * v_scale[ids, h].double()[:, None, None]).flatten(0, 1)
            for i in range(m):
                lim = max(0, n - m + i + 1)
                if lim == 0:
                    continue
                hs = slice(h * G, (h + 1) * G)
                qq = q[b, i, hs].double()
                a = qq @ k[:lim].T * softmax_scale
                top_a = a.amax(-1, keepdim=True)
                if sink is not None:
                    top_a = torch.maximum(top_a, sink[hs].double()[:, None])
                p = torch.exp(a - top_a)
                z = p.sum(-1, keepdim=True)
                zk = z
                if sink is not None:
                    z = z + torch.exp(sink[hs].double()[:, None] - top_a)
                out[b, i, hs] = p @ v[:lim] / z
                mass[b, i, hs] = p @ v[:lim].abs() / z
                terms[b, i, hs] = (qq.abs() @ k[:lim].abs().T).amax(-1, keepdim=True) * abs(softmax_scale)
                inv[b, i, hs] = lim * p.amax(-1, keepdim=True) / z
                top[b, i, hs] = v[:lim].abs().max()
    return out, (mass, terms, inv, top)


def attn_tolerance(dtype, D, out, bound):
    """How far the kernel may be from the 64-bit result.

    Weights enter the products as two (bf16) or three (f16) e4m3 terms: each
    takes 4 significant bits, so the rest is at most 2^-4 per term of the value,
    2^-8 or 2^-12, of the weighted sum of |v|; weights too small for that keep
    an absolute error of half the smallest e4m3 step of the last term, 2^-10 / 16
    or 2^-10 / 256 of a scale on which the largest weight is 256: 2^-22 or 2^-26
    of it per token.  Scores are sums of (terms x D) products in fp32, an ulp
    (2^-23) of the sum of their magnitudes each at most; an error of d in the
    exponent scales weights by 1 + d, in numerator and denominator.  exp2 and
    the remaining fp32 steps: 2^-18.  The result is rounded once.
    """
    mass, terms, inv, top = bound
    two = dtype == torch.bfloat16
    d = (2 if two else 3) * D * 2.0 ** -23 * terms
    return (mass * ((2.0 ** -8 if two else 2.0 ** -12) + 2 * d + 2.0 ** -18)
            + inv * top * (2.0 ** -22 if two else 2.0 ** -26)
            + (out.abs() + mass * d) * torch.finfo(dtype).eps / 2 + 1e-30
            + (2.0 ** -25 if not two else 0.0))          # f16's own smallest half step
