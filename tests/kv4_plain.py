"""The 4-bit cache's format and the operators over caches in plain torch: f32 where the format says so, 64 bits otherwise.

Written from the format's statement: value d of a row belongs to group (d div W) * (W / 32) + (d mod (W / 4)) div 8,
W = min(D, 128).  Tolerances of the GPU tests are derived here, next to the roundings that they count."""
import math

import torch

U_F16, U_BF16, U_F32 = 2.0 ** -11, 2.0 ** -8, 2.0 ** -24  # half a step, relative to the value


def groups(D):
    W = min(D, 128)
    return torch.tensor([(d // W) * (W // 32) + (d % (W // 4)) // 8 for d in range(D)])


def quantise(x):
    """bf16 [..., D] -> (codes uint8 [..., D/2], scales f16 [..., D/32, 2]), the format's f32 arithmetic."""
    D = x.shape[-1]
    of = groups(D).to(x.device)
    x = x.float()
    scales = torch.zeros(*x.shape[:-1], D // 32, 2, dtype=torch.float16, device=x.device)
    codes = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for g in range(D // 32):
        at = (of == g).nonzero()[:, 0]
        part = x[..., at]
        nan = part.isnan().any(-1)
        part = part.nan_to_num(0.0, math.inf, -math.inf).clamp(-65504, 65504)
        lo = part.amin(-1).half()
        scale = ((part.amax(-1) - lo.float()).clamp(min=0) / 15).half()
        s = scale.float()[..., None]
        c = torch.where(s > 0, torch.round((part - lo.float()[..., None]) / s).clamp(0, 15), 0.0)
        codes[..., at] = torch.where(nan[..., None], 0.0, c).to(torch.uint8)
        scales[..., g, 0] = torch.where(nan, 0.0, scale)
        scales[..., g, 1] = torch.where(nan, math.nan, lo)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), scales


def values(codes, scales, dtype=torch.float64):
    D = 2 * codes.shape[-1]
    of = groups(D).to(codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], D)
    return scales[..., 1].to(dtype)[..., of] + scales[..., 0].to(dtype)[..., of] * c.to(dtype)


def fill(rt, B, Hkv, S, D, seed, device="cuda"):
    """A cache of N(0, 1) values, keys with an offset for every channel, quantised by `quantise`."""
    g = torch.Generator(device=device).manual_seed(seed)
    k = torch.randn(B, Hkv, S, D, device=device, generator=g) + torch.randn(Hkv, 1, D, device=device, generator=g)
    v = torch.randn(B, Hkv, S, D, device=device, generator=g)
    return rt.Kv4Cache(*quantise(k.bfloat16()), *quantise(v.bfloat16()))


def decode(q, cache, lens, scale=None):
    """Per sequence and KV head in 64 bits: out, lse, weights [B,Hkv,S], and what each may be off by."""
    B, Hkv, S, half = cache.k_codes.shape
    D, Hq = 2 * half, q.shape[1]
    G = Hq // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.zeros(B, Hkv, S, dtype=torch.float64, device=q.device)
    out_tol, lse_tol, w_tol = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(w)
    for b in range(B):
        n = min(max(int(lens[b]), 0), S)
        if n == 0:
            continue
        k = values(cache.k_codes[b, :, :n], cache.k_scales[b, :, :n])
        v = values(cache.v_codes[b, :, :n], cache.v_scales[b, :, :n])
        step = 15 * cache.v_scales[b, :, :n, :, 0].double()[..., groups(D).to(q.device)]
        qb = q[b].double().reshape(Hkv, G, D)
        s = torch.einsum("hgd,htd->hgt", qb, k) * scale
        m = torch.logsumexp(s, -1)
        p = torch.exp(s - m[..., None])
        out[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(Hq, D)
        lse[b], w[b, :, :n] = m.reshape(Hq), p.sum(1)
        # A score is a sum of D + D/32 products and sums in f32 (each off by half a step of the partial sums, which are at
        # most sum |q| (|lo| + 15 |scale|)); the exponent, its base's change and the row's sum add a few steps more.
        size = torch.einsum("hgd,htd->hgt", qb.abs(), k.abs() + 15 * cache.k_scales[b, :, :n, :, 0].double()[..., groups(D).to(q.device)]) * scale
        ds = size.amax(-1) * (2 * D + 8) * U_F32 + 16 * U_F32 * (1 + s.abs().amax(-1))
        lse_tol[b] = (ds + 16 * U_F32 * (1 + m.abs())).reshape(Hq)
        # p is rounded to f16, and its product with a token's scale once more; the result to bf16.  p is held times 2^9 and the
        # scale so that the largest is in [1/2, 1): f16's last place, 2^-24, is 2^-33 of p's unit and of twice the largest
        # scale's, and half of it is lost of each.
        near = torch.einsum("hgt,htd->hgd", p, v.abs() + step)
        near = near * (2.1 * U_F16) + near * (2 * ds)[..., None] + n * 2.0 ** -33 * (v.abs().max() + step.max())
        out_tol[b] = (near * (1 + U_BF16)).reshape(Hq, D) + U_BF16 * out[b].abs() + 2.0 ** -40
        w_tol[b, :, :n] = (p * (2 * ds + 64 * U_F32 * (1 + m.abs()))[..., None]).sum(1)
    return out, lse, w, out_tol, lse_tol, w_tol


def weigh(q, k_cache, lse, lens, scale=None):
    """What kv_weigh adds, in 64 bits, and what it may be off by.  q [B,Hq,T,D], lse [B,Hq,T]."""
    B, Hkv, S, D = k_cache.shape
    Hq, T = q.shape[1], q.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    w = torch.zeros(B, Hkv, S, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(w)
    for b in range(B):
        n = min(max(int(lens[b]), 0), S)
        k, qb = k_cache[b, :, :n].double(), q[b].double().reshape(Hkv, -1, D)
        s = torch.einsum("hqd,htd->hqt", qb, k) * scale
        at = n - T + torch.arange(T, device=q.device).repeat(Hq // Hkv)
        ls = lse[b].double().reshape(Hkv, -1, 1)
        seen = (torch.arange(n, device=q.device)[None] <= at[:, None]) & (ls != -math.inf)
        p = torch.where(seen, torch.exp(s - ls), 0.0)
        w[b, :, :n] = p.sum(1)
        size = torch.einsum("hqd,htd->hqt", qb.abs(), k.abs()) * scale
        off = size * (D + 8) * U_F32 + 16 * U_F32 * (1 + s.abs() + torch.where(ls == -math.inf, 0.0, ls).abs())
        tol[b, :, :n] = (p * off).sum(1) + p.sum(1) * (p.shape[1] + 8) * U_F32
    return w, tol


def evict(weights, lens, keep, recent):
    """kept [B][Hkv] -> list of places, by the rule."""
    w = weights.cpu()
    B, Hkv, S = w.shape
    kept = []
    for b in range(B):
        n = min(max(int(lens[b]), 0), S)
        row = []
        for h in range(Hkv):
            at = list(range(n))
            if n > keep:
                x = [math.inf if v != v else v for v in w[b, h, :n - recent].tolist()]
                nan = [v != v for v in w[b, h, :n - recent].tolist()]
                order = sorted(range(n - recent), key=lambda t: (not nan[t], -x[t], t))
                at = sorted(order[:keep - recent]) + at[n - recent:]
            row.append(at)
        kept.append(row)
    return kept
