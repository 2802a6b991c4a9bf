"""Eviction from a KV cache by accumulated attention weight.

A cache that may hold only so many tokens keeps the ones that queries look at.  ``kv_weigh`` (over a bf16 cache) and
``kv4_decode(..., weights=...)`` (over a 4-bit one) add the softmax weight that each cached token got to an accumulator
f32 ``[B, Hkv, max_seq]``, which starts at zero; ``kv_evict`` then moves the heaviest and the latest rows of every sequence and
KV head, in their order, to the front of another cache, and their weights with them.  Two caches used in turn serve a
decode loop: rows that the loop appends behind the kept ones find their weights at zero.

After an eviction a row's place in the cache is no longer its token's position: keys keep the rotation of their own
position, and ``rope_kv4_append`` takes the two apart (``positions`` and ``slots``).
"""
from __future__ import annotations

from typing import Optional

from . import _lib
from .gqa import HeadCountMismatch, _guard
from .kv4 import Kv4Cache, _guard_cache, _guard_ints, _stream


def _guard_bf16_cache(name: str, t, like=None):
    import torch
    _guard(name, t, torch.bfloat16, like=like)
    if t.dim() != 4:
        raise TypeError(f"{name} must be [B, Hkv, max_seq, D], got {tuple(t.shape)}")
    return tuple(t.shape)


def kv_weigh(q, k_cache, lse, weights, kv_lens=None, kv_len: Optional[int] = None, scale: Optional[float] = None) -> None:
    """Adds the softmax weights of q over a bf16 cache to ``weights`` f32 ``[B,Hkv,max_seq]`` (``rt_kv_weigh_bf16``).

    q ``[B,Hq,D]``: single-token queries, lse ``[B,Hq]`` as ``gqa_decode`` returned it for them.  Or q ``[B,Hq,T,D]``, lse
    ``[B,Hq,T]`` from ``prefill_bf16``: the last T tokens of a prompt, each of which sees the tokens up to itself (of a padded batch,
    gathered: they end at ``kv_lens``); a row with lse = -inf adds nothing.  k_cache
    ``[B,Hkv,max_seq,D]`` bf16 (D 64, 128 or 256); ``kv_lens`` int32 CUDA ``[B]`` or a uniform ``kv_len``."""
    if (_lib._binding or _lib.torch_binding()).kv_weigh(q, k_cache, lse, weights, kv_lens, kv_len, scale):
        return
    import torch
    B, Hkv, S, D = _guard_bf16_cache("k_cache", k_cache)
    _guard("q", q, torch.bfloat16, like=k_cache)
    if q.dim() not in (3, 4) or q.shape[0] != B or q.shape[-1] != D:
        raise TypeError(f"q must be [B={B}, Hq, D={D}] or [B, Hq, T, D], got {tuple(q.shape)}")
    Hq, T = q.shape[1], q.shape[2] if q.dim() == 4 else 1
    _guard("lse", lse, torch.float32, like=q, shape=q.shape[:-1])
    _guard("weights", weights, torch.float32, like=q, shape=(B, Hkv, S))
    n = _guard_ints("kv_lens", kv_lens, q, B)
    with torch.cuda.device(q.device):
        rc = _lib.lib().rt_kv_weigh_bf16(q.data_ptr(), k_cache.data_ptr(), lse.data_ptr(), weights.data_ptr(), B, Hq, Hkv, T, D,
                                         S, n, 0 if kv_len is None else int(kv_len), -1.0 if scale is None else float(scale),
                                         _stream(q.device))
    if rc == _lib.RT_ERR_HEAD_COUNT:
        raise HeadCountMismatch(Hq, Hkv)
    _lib.check(rc, "rt_kv_weigh_bf16")


def kv_evict(cache, out, weights, keep: int, recent: int = 0, kv_lens=None, kv_len: Optional[int] = None, weights_out=None):
    """Keeps ``keep`` rows of every (sequence, KV head): the last ``recent`` ones and the heaviest of the others
    (``rt_kv_evict``).

    ``cache`` and ``out``: two ``Kv4Cache``, or two pairs (k_cache, v_cache) of bf16 ``[B,Hkv,max_seq,D]`` tensors; ``out`` holds
    at least ``keep`` rows, shares no memory with ``cache`` nor one of its tensors with another, and has its other rows left as
    they were.  ``weights`` f32 ``[B,Hkv,max_seq]``.  Returns (lens int32 ``[B]``, the lengths in ``out``; weights_out f32 ``[B,Hkv,max_seq of out]``, the
    rows' weights, zero behind them; kept int32 ``[B,Hkv,keep]``, the rows' places in ``cache``, -1 behind them)."""
    if type(cache) is type(out) and type(cache) in (Kv4Cache, tuple):
        r = (_lib._binding or _lib.torch_binding()).kv_evict(cache, out, weights, keep, recent, kv_lens, kv_len, weights_out)
        if r is not None:
            return r
    import torch
    if isinstance(cache, Kv4Cache):
        B, Hkv, S, D = _guard_cache(cache)
        other = _guard_cache(out, "out")
    else:
        for name, pair in (("cache", cache), ("out", out)):
            if not isinstance(pair, (tuple, list)) or isinstance(pair, Kv4Cache) or len(pair) != 2:
                raise TypeError(f"{name} must be a Kv4Cache or a pair (k_cache, v_cache), and out what cache is")
        B, Hkv, S, D = _guard_bf16_cache("cache[0]", cache[0])
        _guard("cache[1]", cache[1], torch.bfloat16, like=cache[0], shape=cache[0].shape)
        other = _guard_bf16_cache("out[0]", out[0], like=cache[0])
        _guard("out[1]", out[1], torch.bfloat16, like=cache[0], shape=out[0].shape)
    like = cache[0]
    if out[0].device != like.device or (other[0], other[1], other[3]) != (B, Hkv, D):
        raise TypeError(f"out must be a cache of B={B}, Hkv={Hkv}, D={D} on {like.device}, got {other} on {out[0].device}")
    keep, recent = int(keep), int(recent)
    if keep < 1 or keep > other[2] or not 0 <= recent <= keep:
        raise _lib.CudaError(_lib.RT_ERR_BAD_LENGTH, "rt_kv_evict")
    _guard("weights", weights, torch.float32, like=like, shape=(B, Hkv, S))
    n = _guard_ints("kv_lens", kv_lens, like, B)
    if weights_out is None:
        weights_out = torch.empty((B, Hkv, other[2]), dtype=torch.float32, device=like.device)
    else:
        _guard("weights_out", weights_out, torch.float32, like=like, shape=(B, Hkv, other[2]))
    kept = torch.empty((B, Hkv, keep), dtype=torch.int32, device=like.device)
    lens = torch.empty((B,), dtype=torch.int32, device=like.device)
    src, dst = _lib.pointers(t.data_ptr() for t in cache), _lib.pointers(t.data_ptr() for t in out)
    sizes = _lib.int32s((D // 2, D // 8, D // 2, D // 8) if len(cache) == 4 else (2 * D, 2 * D))
    with torch.cuda.device(like.device):
        rc = _lib.lib().rt_kv_evict(src, dst, sizes, len(cache), weights.data_ptr(), weights_out.data_ptr(), kept.data_ptr(),
                                    lens.data_ptr(), B, Hkv, S, other[2], n, 0 if kv_len is None else int(kv_len), keep, recent,
                                    _stream(like.device))
    _lib.check(rc, "rt_kv_evict")
    return lens, weights_out, kept
