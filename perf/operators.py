"""A KV cache held in 4 bits and eviction from a cache, as cases that can be timed and compared.

Five kinds, each a pass through one operator of ``rustorch_b200`` as a serving program calls it:

    append  new K and V rows are quantised into a 4-bit cache: a token's rows behind their rotary embedding
            (rope_kv4_append) or a padded batch of prompts straight from the projections' layout (kv4_append).  What is
            returned are the rows' values, as kv4_read gives them.
    read    the context in bf16 that a chunk of a prompt attends to (kv4_read)
    decode  attention of single-token queries over the 4-bit cache (kv4_decode), on request adding every cached token's
            softmax weight to an accumulator
    weigh   the same weights over a bf16 cache, for one query a sequence or the last ones of a prompt (kv_weigh)
    evict   the heaviest and the latest rows of a cache, in order, in a smaller one (kv_evict)

The cache's format.  A row of D values has D / 32 groups of 32: with W = min(D, 128), value d belongs to group
(d div W) * (W / 32) + (d mod (W / 4)) div 8.  A group holds lo = min and scale = (max - lo) / 15 in fp16 and a code of
0 to 15 for each value, round((x - lo) / scale); the code stands for lo + scale * code.  Byte i of a row's codes is
code 2i in the low half and code 2i + 1 in the high one.

Keys carry an offset for every channel, as those of real models do; queries and values are N(0, 1).  Ragged lengths are spread
evenly over [lo, hi] and dealt to the sequences in an order that the seed picks.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

# ------------------------------------------------------------------------------------------------ the cases


def listed():
    return [
        # a step of 16 users: their new rows, rotated and appended, one layer
        dict(name="append_step_16seq", kind="append", rope=True, B=16, Hq=32, Hkv=8, D=128, T=1, max_seq=8192, lo=100, hi=8000),
        # a padded batch of four prompts, as the projections leave it, appended to empty caches
        dict(name="append_prompt", kind="append", rope=False, B=4, Hq=8, Hkv=8, D=128, T=4096, max_seq=8192, lo=1000, hi=4096),
        # the context of a chunk of one long prompt
        dict(name="read_chunk", kind="read", B=1, Hkv=8, D=128, max_seq=8192, lo=6001, hi=6001),
        # a padded batch at head dim 64
        dict(name="read_batch_d64", kind="read", B=16, Hkv=16, D=64, max_seq=2048, lo=256, hi=2048),
        # one user at about a thousand tokens of context
        dict(name="decode_1seq", kind="decode", B=1, Hq=32, Hkv=8, D=128, max_seq=4096, lo=1000, hi=1000, weights=False),
        # a small batch on a model of head dim 256 that weighs its tokens; lengths that are multiples of nothing
        dict(name="decode_7seq_d256_weighed", kind="decode", B=7, Hq=16, Hkv=2, D=256, max_seq=3000, lo=100, hi=3000,
             weights=True),
        # a full server: 64 sequences of 1024 to 8192 tokens
        dict(name="decode_64seq", kind="decode", B=64, Hq=32, Hkv=8, D=128, max_seq=8192, lo=1024, hi=8192, weights=False),
        # one long context, its tokens weighed
        dict(name="decode_long_weighed", kind="decode", B=1, Hq=32, Hkv=8, D=128, max_seq=131072, lo=131072, hi=131072,
             weights=True),
        # the same full server on a bf16 cache: the step's weights
        dict(name="weigh_step_64seq", kind="weigh", B=64, Hq=32, Hkv=8, D=128, Nq=1, max_seq=8192, lo=1024, hi=8192),
        # what the last 64 queries of a prompt looked at
        dict(name="weigh_window", kind="weigh", B=1, Hq=32, Hkv=8, D=128, Nq=64, max_seq=16384, lo=16001, hi=16001),
        # a long prompt cut down to what the decode keeps
        dict(name="evict_prompt", kind="evict", bits=16, B=1, Hkv=8, D=128, max_seq=32768, lo=30001, hi=30001, keep=4096,
             recent=256),
        # a batch on the 4-bit cache, some of its sequences still shorter than what is kept
        dict(name="evict_batch_4bit", kind="evict", bits=4, B=16, Hkv=8, D=64, max_seq=4096, lo=500, hi=4096, keep=1024,
             recent=64),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    """Evenly over the logarithm, every integer possible."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, KV heads): groups of 1 to 8
_HEADS = [(8, 8), (16, 16), (32, 32), (16, 8), (32, 8), (32, 16), (16, 2), (24, 8), (28, 4), (64, 8)]


def _draw_once(rng: random.Random) -> dict:
    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode", "weigh", "weigh", "evict", "evict"])
    Hq, Hkv = rng.choice(_HEADS)
    D, B = rng.choice([64, 128, 128, 256]), _log_int(rng, 1, 64)
    max_seq = _log_int(rng, 256, 131072)
    hi = rng.randint(max(1, max_seq // 2), max_seq)
    lo = hi if B == 1 else rng.randint(max(1, hi // 8), hi)
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, rope=True, B=B, Hq=Hq, Hkv=Hkv, D=D, T=1, max_seq=max_seq, lo=lo - 1, hi=hi - 1)
        T = _log_int(rng, 1, min(max_seq, 8192))
        return dict(kind=kind, rope=False, B=B, Hq=Hkv, Hkv=Hkv, D=D, T=T, max_seq=max_seq,
                    lo=T if B == 1 else rng.randint(max(1, T // 8), T), hi=T)
    if kind == "read":
        return dict(kind=kind, B=B, Hkv=Hkv, D=D, max_seq=max_seq, lo=lo, hi=hi)
    if kind == "decode":
        return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, max_seq=max_seq, lo=lo, hi=hi, weights=rng.random() < 0.4)
    if kind == "weigh":
        return dict(kind=kind, B=B, Hq=Hq, Hkv=Hkv, D=D, Nq=rng.choice([1, 1, _log_int(rng, 2, 128)]), max_seq=max_seq, lo=lo,
                    hi=hi)
    keep = _log_int(rng, max(1, max_seq // 16), max(1, max_seq // 2))
    return dict(kind=kind, bits=rng.choice([16, 4]), B=B, Hkv=Hkv, D=D, max_seq=max_seq, lo=lo, hi=hi, keep=keep,
                recent=rng.randint(0, keep // 2))


# the most that a pass of a kind moves or computes (bytes, flops): about its largest listed case
_MOST = {"append": (120e6, 1e15), "read": (160e6, 1e15), "decode": (420e6, 1e15), "weigh": (650e6, 17e9), "evict": (40e6, 1e15)}


def draw(rng):
    while True:
        case = _draw_once(rng)
        w, most = work(case), _MOST[case["kind"]]
        cache = case["B"] * case["Hkv"] * case["max_seq"] * case["D"]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and cache <= 1 << 30:
            return case


# ------------------------------------------------------------------------------------------------ inputs


def _spread(B: int, lo: int, hi: int):
    return [lo + int(round((hi - lo) * (i + 0.5) / B)) for i in range(B)]


def _lens(case, seed):
    lens = _spread(case["B"], case["lo"], case["hi"])
    random.Random(seed).shuffle(lens)
    return lens


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, dtype=torch.bfloat16, device="cuda", generator=g)

    kind, B, Hkv, D, S = case["kind"], case["B"], case["Hkv"], case["D"], case["max_seq"]
    lens = _lens(case, seed)
    s = {"case": case, "lens": _i32(lens)}
    offset = randn(Hkv, 1, D)

    def cache4():
        """A cache that the format's own quantisation filled (every row, so that rows behind the lengths hold numbers)."""
        planes = []
        for shift in (offset, 0):
            codes = torch.empty((B, Hkv, S, D // 2), dtype=torch.uint8, device="cuda")
            scales = torch.empty((B, Hkv, S, D // 32, 2), dtype=torch.float16, device="cuda")
            step = max(1, (1 << 27) // (Hkv * D))
            for b in range(B):
                for t in range(0, S, step):
                    n = min(step, S - t)
                    codes[b, :, t:t + n], scales[b, :, t:t + n] = _quantise(randn(Hkv, n, D) + shift)
            planes += [codes, scales]
        return planes

    if kind == "append":
        T, Hq = case["T"], case["Hq"]
        if case["rope"]:
            s.update(q=randn(B, Hq, D), k=randn(B, Hkv, D) + offset[:, 0], v=randn(B, Hkv, D), positions=s["lens"],
                     inv_freq=(1.0 / torch.pow(torch.tensor(10000.0), 2.0 * torch.arange(D // 2) / D)).float().cuda())
        else:  # the projections' [B, T, Hkv, D], seen as [B, Hkv, T, D]; every sequence starts where its cache ends
            starts = [random.Random(seed + b).randint(0, S - T) for b in range(B)]
            s.update(k=(randn(B, T, Hkv, D) + offset[:, 0]).permute(0, 2, 1, 3), v=randn(B, T, Hkv, D).permute(0, 2, 1, 3),
                     positions=_i32(starts), ends=_i32([a + n for a, n in zip(starts, lens)]))
        s["planes"] = [torch.zeros((B, Hkv, S) + tail, dtype=t, device="cuda")
                       for _ in "kv" for tail, t in (((D // 2,), torch.uint8), ((D // 32, 2), torch.float16))]
    elif kind == "read":
        s["planes"] = cache4()
    elif kind == "decode":
        s.update(q=randn(B, case["Hq"], D), planes=cache4())
        if case["weights"]:
            s["weights"] = torch.rand((B, Hkv, S), device="cuda", generator=g)
    elif kind == "weigh":
        Hq, Nq = case["Hq"], case["Nq"]
        s.update(q=randn(B, Hq, Nq, D) if Nq > 1 else randn(B, Hq, D), k_cache=randn(B, Hkv, S, D).add_(offset),
                 weights=torch.rand((B, Hkv, S), device="cuda", generator=g))
        s["lse"] = torch.logsumexp(_scores(s["q"], s["k_cache"][:, :, :case["hi"]], s["lens"], Nq), -1).reshape(s["q"].shape[:-1])
    else:
        # weights as a decode accumulates them: a few tokens get most; many, just appended, have none yet
        w = torch.exp(2 * torch.randn((B, Hkv, S), device="cuda", generator=g))
        s["weights"] = w * (torch.rand((B, Hkv, S), device="cuda", generator=g) > 0.2)
        s["planes"] = cache4() if case["bits"] == 4 else [randn(B, Hkv, S, D), randn(B, Hkv, S, D)]
        keep = case["keep"]
        s["out_planes"] = [torch.zeros(p.shape[:2] + (keep,) + p.shape[3:], dtype=p.dtype, device="cuda") for p in s["planes"]]
        s["weights_out"] = torch.zeros((B, Hkv, keep), device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ the plain forms


def _group(x):
    """[..., D] -> [..., D / 32, 32], a group's values together."""
    D = x.shape[-1]
    W = min(D, 128)
    return x.reshape(*x.shape[:-1], D // W, 4, W // 32, 8).transpose(-3, -2).reshape(*x.shape[:-1], D // 32, 32)


def _ungroup(x):
    D = x.shape[-2] * 32
    W = min(D, 128)
    return x.reshape(*x.shape[:-2], D // W, W // 32, 4, 8).transpose(-3, -2).reshape(*x.shape[:-2], D)


def _quantise(x):
    """bf16 [..., D] -> codes uint8 [..., D / 2], (scale, lo) fp16 [..., D / 32, 2]."""
    x = _group(x.float().clamp(-65504, 65504))
    lo = x.amin(-1).half()
    scale = ((x.amax(-1) - lo.float()).clamp(min=0) / 15).half()
    s = scale.float()[..., None]
    c = torch.where(s > 0, ((x - lo.float()[..., None]) / s).round().clamp(0, 15), 0).to(torch.uint8)
    c = _ungroup(c)
    return c[..., 0::2] | c[..., 1::2] << 4, torch.stack([scale, lo], -1)


def _values(codes, scales):
    """The cache's rows in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    return _ungroup(_group(c).float() * scales[..., 0:1].float() + scales[..., 1:2].float())


def _scores(q, k, lens, Nq):
    """q [B, Hkv * G, (Nq,) D], k [B, Hkv, S, D]: scaled scores [B, Hkv, G * Nq, S]; query i of Nq sits at position
    lens - Nq + i, and what it does not see is -inf."""
    B, Hkv, S, D = k.shape
    s = torch.einsum("bhqd,bhtd->bhqt", q.reshape(B, Hkv, -1, D).float(), k.float()) / math.sqrt(D)
    at = torch.arange(s.shape[2], device="cuda") % Nq + (lens[:, None] - Nq)
    return s.masked_fill_(torch.arange(S, device="cuda") > at[:, None, :, None], -math.inf)


def _rope(x, positions, inv_freq):
    """Pairs (i, i + D / 2); the angle is a product in 32 bits, its sine and cosine are taken in 64."""
    a = (positions.float()[:, None] * inv_freq[None, :]).double()[:, None, :]
    c, s = a.cos().float(), a.sin().float()
    x0, x1 = x.float().chunk(2, -1)
    return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], -1).to(torch.bfloat16)


def _append(planes, k, v, starts, lens):
    """Rows 0 to lens - 1 of k, v [B, Hkv, T, D] to positions starts and up."""
    b = torch.arange(len(starts), device="cuda")[:, None]
    i = torch.arange(k.shape[2], device="cuda")
    at, there = starts[:, None] + i, (i < lens[:, None])[:, :, None, None]

    def put(plane, rows):
        there_ = there.reshape(there.shape + (1,) * (plane.dim() - 4))
        plane[b, :, at] = torch.where(there_, rows.transpose(1, 2), plane[b, :, at])

    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    put(planes[0], kc), put(planes[1], ks), put(planes[2], vc), put(planes[3], vs)


def _read(planes, starts, lens, rows):
    """Rows [start, start + rows) in bf16, those from `lens` on zero."""
    b = torch.arange(len(starts), device="cuda")[:, None]
    at = starts[:, None] + torch.arange(rows, device="cuda")
    there = (at < lens[:, None])[:, :, None, None]
    at = at.clamp(max=planes[0].shape[2] - 1)

    def values(codes, scales):
        return torch.where(there, _values(codes[b, :, at], scales[b, :, at]), 0).to(torch.bfloat16).transpose(1, 2).contiguous()

    return [values(planes[0], planes[1]), values(planes[2], planes[3])]


def _run_plain(s):
    case, lens = s["case"], s["lens"]
    kind, B, Hkv, D = case["kind"], case["B"], case["Hkv"], case["D"]
    if kind == "append" and case["rope"]:
        s["q"].copy_(_rope(s["q"], lens, s["inv_freq"]))
        k = _rope(s["k"], lens, s["inv_freq"])
        _append(s["planes"], k[:, :, None], s["v"][:, :, None], lens, torch.ones_like(lens))
        k, v = _read(s["planes"], lens, lens + 1, 1)
        return {"k": k, "v": v, "q": s["q"]}
    if kind == "append":
        _append(s["planes"], s["k"], s["v"], s["positions"], lens)
        k, v = _read(s["planes"], s["positions"], s["ends"], case["T"])
        return {"k": k, "v": v, "q": None}
    if kind == "read":
        return _read(s["planes"], torch.zeros_like(lens), lens, case["hi"])
    if kind == "decode":
        k, v = (_values(*(p[:, :, :case["hi"]] for p in s["planes"][i:i + 2])) for i in (0, 2))
        scores = _scores(s["q"], k, lens, 1)
        lse = torch.logsumexp(scores, -1, keepdim=True)
        w = torch.exp(scores - lse)
        if case["weights"]:
            s["weights"][:, :, :case["hi"]] += w.sum(2)
        out = torch.einsum("bhqt,bhtd->bhqd", w, v).to(torch.bfloat16)
        return {"out": out.reshape(s["q"].shape), "lse": lse.reshape(B, -1), "weights": s.get("weights")}
    if kind == "weigh":
        scores = _scores(s["q"], s["k_cache"][:, :, :case["hi"]], lens, case["Nq"])
        w = torch.exp(scores - s["lse"].reshape(B, Hkv, -1, 1))
        s["weights"][:, :, :case["hi"]] += torch.where(scores == -math.inf, 0, w).sum(2)  # a query of no keys has no weights
        return {"weights": s["weights"]}
    keep, recent, n = case["keep"], case["recent"], lens[:, None, None].long()
    t = torch.arange(case["max_seq"], device="cuda")
    order = torch.where(t < n - recent, s["weights"], -1.0).sort(dim=-1, descending=True, stable=True)[1]
    heavy = torch.zeros_like(s["weights"], dtype=torch.bool).scatter_(2, order[:, :, :keep - recent], True)
    chosen = torch.where(n <= keep, t < n, ((t >= n - recent) & (t < n)) | (heavy & (t < n - recent)))
    at = torch.where(chosen, t, t + case["max_seq"]).sort(dim=-1)[0][:, :, :keep]
    there = torch.arange(keep, device="cuda") < n
    kept = torch.where(there, at, -1).to(torch.int32)
    at = torch.where(there, at, 0)
    s["weights_out"].copy_(torch.where(there, s["weights"].gather(2, at), 0))
    b, h = torch.arange(B, device="cuda")[:, None, None], torch.arange(Hkv, device="cuda")[:, None]

    def move(out, plane):
        out.copy_(torch.where(there.reshape(there.shape + (1,) * (plane.dim() - 3)), plane[b, h, at], out))

    [move(o, p) for o, p in zip(s["out_planes"], s["planes"])]
    lens = lens.clamp(max=keep)
    k, v = _read(s["out_planes"], torch.zeros_like(lens), lens, keep) if case["bits"] == 4 else s["out_planes"]
    return {"k": k, "v": v, "lens": lens, "weights": s["weights_out"], "kept": kept}


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    if not own:
        return _run_plain(s)
    import rustorch_b200 as rt

    case = s["case"]
    kind = case["kind"]
    if kind == "weigh":
        rt.kv_weigh(s["q"], s["k_cache"], s["lse"], s["weights"], kv_lens=s["lens"])
        return {"weights": s["weights"]}
    cache = rt.Kv4Cache(*s["planes"]) if len(s["planes"]) == 4 else tuple(s["planes"])
    if kind == "append" and case["rope"]:
        rt.rope_kv4_append(s["q"], s["k"], s["v"], cache, s["inv_freq"], positions=s["positions"])
        k, v = rt.kv4_read(cache, 1, starts=s["positions"])
        return {"k": k, "v": v, "q": s["q"]}
    if kind == "append":
        rt.kv4_append(cache, s["k"], s["v"], positions=s["positions"], lens=s["lens"])
        k, v = rt.kv4_read(cache, case["T"], starts=s["positions"], kv_lens=s["ends"])
        return {"k": k, "v": v, "q": None}
    if kind == "read":
        return list(rt.kv4_read(cache, case["hi"], kv_lens=s["lens"]))
    if kind == "decode":
        out, lse = rt.kv4_decode(s["q"], cache, kv_lens=s["lens"], weights=s.get("weights"))
        return {"out": out, "lse": lse, "weights": s.get("weights")}
    out = rt.Kv4Cache(*s["out_planes"]) if case["bits"] == 4 else tuple(s["out_planes"])
    lens, weights, kept = rt.kv_evict(cache, out, s["weights"], case["keep"], recent=case["recent"], kv_lens=s["lens"],
                                      weights_out=s["weights_out"])
    k, v = rt.kv4_read(out, case["keep"], kv_lens=lens) if case["bits"] == 4 else out
    return {"k": k, "v": v, "lens": lens, "weights": weights, "kept": kept}


# ------------------------------------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    kind, B, Hkv, D, lens = case["kind"], case["B"], case["Hkv"], case["D"], _lens(case, seed)

    def _members(D):
        """The dims of each group, from the format's rule."""
        W = min(D, 128)
        of = [(d // W) * (W // 32) + d % (W // 4) // 8 for d in range(D)]
        return [[d for d in range(D) if of[d] == g] for g in range(D // 32)]

    def _exact_stored(x):
        """x [..., D] as the cache holds it, in 64 bits."""
        y = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        for dims in _members(x.shape[-1]):
            part = x[..., dims].double()
            lo = part.min(-1, keepdim=True)[0].half().double()
            step = ((part.max(-1, keepdim=True)[0] - lo) / 15).half().double()
            y[..., dims] = lo + step * torch.clamp(torch.round((part - lo) / step.clamp(min=1e-300)), 0, 15) * (step > 0)
        return y

    def _exact_values(codes, scales):
        D = 2 * codes.shape[-1]
        y = torch.empty(codes.shape[:-1] + (D,), dtype=torch.float64, device=codes.device)
        for g, dims in enumerate(_members(D)):
            at = torch.tensor(dims, device=codes.device)
            c = (codes[..., at // 2].int() >> 4 * (at % 2).int()) & 15
            y[..., dims] = scales[..., g, 1:2].double() + scales[..., g, 0:1].double() * c
        return y

    if kind == "append":
        T = case["T"]
        q, k, v = None, s["k"], s["v"]
        if case["rope"]:
            angle = (s["positions"].float()[:, None] * s["inv_freq"]).double()[:, None]
            turn = torch.polar(torch.ones_like(angle), angle)

            def rotated(x):
                z = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * turn
                return torch.cat([z.real, z.imag], -1)

            # a cache's row is quantised from the rotated key in bf16
            q, k, v, counts = rotated(s["q"]), rotated(k).bfloat16()[:, :, None], v[:, :, None], [1] * B
        else:
            counts = lens
        out = [torch.zeros((B, Hkv, T, D), dtype=torch.float64, device="cuda") for _ in "kv"]
        for o, x in zip(out, (k, v)):
            for b, n in enumerate(counts):
                o[b, :, :n] = _exact_stored(x[b, :, :n])
        return {"k": out[0], "v": out[1], "q": q}
    if kind == "read":
        out = [torch.zeros((B, Hkv, case["hi"], D), dtype=torch.float64, device="cuda") for _ in "kv"]
        for b, n in enumerate(lens):
            for i in (0, 1):
                out[i][b, :, :n] = _exact_values(s["planes"][2 * i][b, :, :n], s["planes"][2 * i + 1][b, :, :n])
        return out
    if kind in ("decode", "weigh"):
        Hq, Nq = case["Hq"], case.get("Nq", 1)
        G = Hq // Hkv
        out = torch.zeros((B, Hq, D), dtype=torch.float64, device="cuda")
        lse = torch.zeros((B, Hq), dtype=torch.float64, device="cuda")
        weights = s["weights"].double() if "weights" in s else None
        for b, n in enumerate(lens):
            for h in range(Hkv):
                k = (_exact_values(s["planes"][0][b, h, :n], s["planes"][1][b, h, :n]) if kind == "decode"
                     else s["k_cache"][b, h, :n].double())
                q = s["q"][b, h * G:(h + 1) * G].double().reshape(G, Nq, D)
                z = (q @ k.T) / D ** 0.5  # [G, Nq, n]
                if kind == "weigh":
                    seen = torch.tril(torch.ones((Nq, n), dtype=torch.bool, device="cuda"), diagonal=n - Nq)
                    e = torch.exp(z - s["lse"][b, h * G:(h + 1) * G].double().reshape(G, Nq, 1))
                    weights[b, h, :n] += torch.where(seen, e, 0).sum((0, 1))
                    continue
                e = torch.exp(z[:, 0] - z[:, 0].max(-1, keepdim=True)[0])
                total = e.sum(-1, keepdim=True)
                out[b, h * G:(h + 1) * G] = e @ _exact_values(s["planes"][2][b, h, :n], s["planes"][3][b, h, :n]) / total
                lse[b, h * G:(h + 1) * G] = z[:, 0].max(-1)[0] + total[:, 0].log()
                if weights is not None:
                    weights[b, h, :n] += (e / total).sum(0)
        return {"weights": weights} if kind == "weigh" else {"out": out, "lse": lse, "weights": weights}
    keep, recent = case["keep"], case["recent"]
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    weights = torch.zeros((B, Hkv, keep), dtype=torch.float64)
    # rows behind what is kept are left as they were, zeros here
    k, v = (torch.zeros((B, Hkv, keep, D), dtype=torch.float64, device="cuda") for _ in "kv")
    given = s["weights"].double().cpu().numpy()
    for b, n in enumerate(lens):
        for h in range(Hkv):
            rows = np.arange(n)
            if n > keep:  # of equal weights the first
                heavy = np.lexsort((rows[:n - recent], -given[b, h, :n - recent]))[:keep - recent]
                rows = np.concatenate([np.sort(heavy), rows[n - recent:]])
            m = len(rows)
            kept[b, h, :m] = torch.from_numpy(rows)
            weights[b, h, :m] = torch.from_numpy(given[b, h, rows])
            at = torch.from_numpy(rows).cuda()
            if case["bits"] == 4:
                k[b, h, :m] = _exact_values(s["planes"][0][b, h, at], s["planes"][1][b, h, at])
                v[b, h, :m] = _exact_values(s["planes"][2][b, h, at], s["planes"][3][b, h, at])
            else:
                k[b, h, :m], v[b, h, :m] = s["planes"][0][b, h, at], s["planes"][1][b, h, at]
    return {"k": k, "v": v, "lens": _i32([min(n, keep) for n in lens]), "weights": weights.cuda(), "kept": kept.cuda()}


# ------------------------------------------------------------------------------------------------ what a pass needs


def work(case):
    kind, B, Hkv, D = case["kind"], case["B"], case["Hkv"], case["D"]
    lens = _spread(B, case["lo"], case["hi"])
    tokens = sum(lens)
    row4 = D // 2 + D // 8  # a row's codes and its groups' scales, K or V
    if kind == "append":  # bf16 rows in, the cache's rows and their values out
        rows = B if case["rope"] else tokens
        b = rows * Hkv * (4 * D + 2 * row4) + B * case["T"] * Hkv * 4 * D
        return {"bytes": b + (B * case["Hq"] * 4 * D if case["rope"] else 0), "flops": 0}
    if kind == "read":
        return {"bytes": tokens * Hkv * 2 * row4 + B * case["hi"] * Hkv * 4 * D, "flops": 0}
    if kind == "decode":
        b = tokens * Hkv * (2 * row4 + (8 if case["weights"] else 0))
        b += B * case["Hq"] * (4 * D + 4)
        return {"bytes": b, "flops": 4.0 * tokens * case["Hq"] * D}
    if kind == "weigh":
        Nq = case["Nq"]
        pairs = sum(min(Nq, n) * n - min(Nq, n) * (min(Nq, n) - 1) / 2 for n in lens)
        return {"bytes": tokens * Hkv * (2 * D + 8) + B * case["Hq"] * Nq * (2 * D + 4), "flops": 2.0 * pairs * case["Hq"] * D}
    row = 2 * row4 if case["bits"] == 4 else 4 * D
    kept = sum(min(n, case["keep"]) for n in lens)
    b = tokens * Hkv * 4 + kept * Hkv * 2 * row + B * Hkv * case["keep"] * 8
    if case["bits"] == 4:  # the kept rows' values as well
        b += B * Hkv * case["keep"] * 4 * D
    return {"bytes": b, "flops": 0}
