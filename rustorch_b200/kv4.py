"""A KV cache held in 4 bits: what fills it, what attends to it and what reads it back.

* ``Kv4Cache``          the four planes of a cache of ``[B, Hkv, max_seq, D]`` keys and values, 5 bits a value: codes of 4
                        bits, and a scale and a minimum in fp16 for every 32 values of a row.
* ``kv4_append``        quantises the rows of new tokens (a decode step's, or a padded batch of prompts) into it.
* ``rope_kv4_append``   ``rope_kv_append`` on such a cache: one launch for a step's rotary embedding and append.
* ``kv4_decode``        single-token GQA attention over it (``gqa_decode``'s counterpart), which on request adds every
                        token's softmax weight to an accumulator that ``kv_evict`` chooses by.
* ``kv4_read``          its rows in bf16, which ``prefill_bf16`` of a prompt's chunk attends to (head dims 64 and 128).

The format, value by value, stands in ``include/rustorch_attn.h``.  A third of the bf16 cache's bytes: a decode step reads
1.25 D instead of 4 D bytes a token and KV head.  What it costs: a row of N(0, 1) values is off by 8 % (the bf16 cache's by 0.2 %).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

from . import _lib
from .gqa import _ROPE_STYLES, HeadCountMismatch, _guard


class Kv4Cache(NamedTuple):
    """The planes of a 4-bit cache, contiguous CUDA tensors on one device."""
    k_codes: "torch.Tensor"   # uint8 [B, Hkv, max_seq, D/2], two codes a byte, the even one low
    k_scales: "torch.Tensor"  # float16 [B, Hkv, max_seq, D/32, 2]: (scale, minimum) of each group
    v_codes: "torch.Tensor"
    v_scales: "torch.Tensor"

    @classmethod
    def new(cls, batch: int, n_kv_heads: int, max_seq: int, head_dim: int, device="cuda") -> "Kv4Cache":
        """An empty cache (all zeros).  head_dim is 64, 128 or 256."""
        import torch
        if head_dim not in (64, 128, 256):
            raise _lib.Unsupported(_lib.RT_ERR_UNSUPPORTED, f"Kv4Cache: head_dim {head_dim}")
        shape = (batch, n_kv_heads, max_seq)
        return cls(*(torch.zeros(shape + tail, dtype=dtype, device=device) for _ in "kv"
                     for tail, dtype in (((head_dim // 2,), torch.uint8), ((head_dim // 32, 2), torch.float16))))

    @property
    def dims(self):
        """(B, Hkv, max_seq, D)."""
        B, Hkv, S, half = self.k_codes.shape
        return B, Hkv, S, 2 * half

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self)


def _guard_cache(cache, name: str = "cache"):
    """(B, Hkv, max_seq, D) of a 4-bit cache whose planes are what the kernels take them for."""
    import torch
    if not isinstance(cache, Kv4Cache):
        raise TypeError(f"{name} must be a Kv4Cache, got {type(cache).__name__}")
    _guard(f"{name}.k_codes", cache.k_codes, torch.uint8)
    if cache.k_codes.dim() != 4:
        raise TypeError(f"{name}.k_codes must be [B, Hkv, max_seq, D/2], got {tuple(cache.k_codes.shape)}")
    B, Hkv, S, D = cache.dims
    _guard(f"{name}.v_codes", cache.v_codes, torch.uint8, like=cache.k_codes, shape=cache.k_codes.shape)
    for which in ("k_scales", "v_scales"):
        _guard(f"{name}.{which}", getattr(cache, which), torch.float16, like=cache.k_codes, shape=(B, Hkv, S, D // 32, 2))
    return B, Hkv, S, D


def _guard_ints(name: str, t, like, n: int):
    if t is not None:
        import torch
        _guard(name, t, torch.int32, like=like, shape=(n,))
    return t.data_ptr() if t is not None else None


def _stream(device):
    import torch
    return torch.cuda.current_stream(device).cuda_stream


def _planes(cache):
    return [t.data_ptr() for t in cache]


def kv4_append(cache: Kv4Cache, k, v, pos: Optional[int] = None, positions=None, lens=None) -> None:
    """Quantises new rows into the cache via ``rt_kv4_append``.

    k, v: bf16 CUDA ``[B, Hkv, T, D]`` (or ``[B, Hkv, D]`` for one token each); any strided view whose head dim is contiguous
    and whose strides are multiples of 8, e.g. a projection's ``[B, T, Hkv, D]`` permuted.  Row i goes to position ``pos`` + i
    (default 0) of every sequence, or ``positions[b]`` + i (int32 CUDA ``[B]``; rows outside the cache are dropped then).
    ``lens``: optional int32 CUDA ``[B]``, how many rows of each sequence count.  Enqueues on the current stream."""
    if type(cache) is Kv4Cache and (_lib._binding or _lib.torch_binding()).kv4_append(cache, k, v, pos, positions, lens):
        return
    import torch
    B, Hkv, S, D = _guard_cache(cache)
    ptrs, strides = [], []
    rows = None
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device != cache.k_codes.device or t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be a bfloat16 CUDA tensor on the cache's device")
        if t.dim() == 3:
            t = t.unsqueeze(2)
        if t.dim() != 4 or (t.shape[0], t.shape[1], t.shape[3]) != (B, Hkv, D) or rows not in (None, t.shape[2]):
            raise TypeError(f"{name} must be [B={B}, Hkv={Hkv}, T, D={D}] like the other, got {tuple(t.shape)}")
        rows = t.shape[2]
        if t.numel() and t.stride(3) != 1:
            raise TypeError(f"{name}: the head dim must be contiguous")
        ptrs.append(t.data_ptr())
        # the stride of a dim of one element means nothing
        strides.append(_lib.int64s(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])))
    at, n = _guard_ints("positions", positions, cache.k_codes, B), _guard_ints("lens", lens, cache.k_codes, B)
    with torch.cuda.device(cache.k_codes.device):
        rc = _lib.lib().rt_kv4_append(*_planes(cache), *ptrs, *strides, B, Hkv, rows, D, S, 0 if pos is None else int(pos), at,
                                      n, _stream(cache.k_codes.device))
    _lib.check(rc, "rt_kv4_append")


def rope_kv4_append(q, k_in, v_in, cache: Kv4Cache, inv_freq, pos: Optional[int] = None, positions=None,
                    slot: Optional[int] = None, slots=None, style: str = "half_split") -> None:
    """Rotary embedding of q (in place) and of the new K row, and append of K and V to a 4-bit cache, one launch
    (``rt_rope_kv4_append``).  q ``[B,Hq,D]``, k_in, v_in ``[B,Hkv,D]`` as for ``rope_kv_append``.  The rows go to the rotary
    position, or to ``slot`` / ``slots`` (int32 CUDA ``[B]``) where a cache's rows and positions have come apart."""
    if type(cache) is Kv4Cache and (_lib._binding or _lib.torch_binding()).rope_kv4_append(
            q, k_in, v_in, cache, inv_freq, pos, positions, slot, slots, _ROPE_STYLES[style]):
        return
    import torch
    B, Hkv, S, D = _guard_cache(cache)
    _guard("q", q, torch.bfloat16, like=cache.k_codes)
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != D:
        raise TypeError(f"q must be [B={B}, Hq, D={D}], got {tuple(q.shape)}")
    _guard("k_in", k_in, torch.bfloat16, like=q, shape=(B, Hkv, D))
    _guard("v_in", v_in, torch.bfloat16, like=q, shape=(B, Hkv, D))
    _guard("inv_freq", inv_freq, torch.float32, like=q, shape=(D // 2,))
    at, to = _guard_ints("positions", positions, q, B), _guard_ints("slots", slots, q, B)
    if slot is not None and int(slot) < 0:
        raise _lib.CudaError(_lib.RT_ERR_BAD_LENGTH, "rt_rope_kv4_append")
    with torch.cuda.device(q.device):
        rc = _lib.lib().rt_rope_kv4_append(q.data_ptr(), k_in.data_ptr(), v_in.data_ptr(), *_planes(cache), inv_freq.data_ptr(),
                                           B, q.shape[1], Hkv, D, S, 0 if pos is None else int(pos), at,
                                           -1 if slot is None else int(slot), to, _ROPE_STYLES[style], _stream(q.device))
    _lib.check(rc, "rt_rope_kv4_append")


def kv4_read(cache: Kv4Cache, rows: int, start: int = 0, starts=None, kv_lens=None, out=None):
    """Rows of the cache in bf16 via ``rt_kv4_read``: (k, v) ``[B, Hkv, rows, D]``, row i being the cache's row ``start`` + i
    or ``starts[b]`` + i (int32 CUDA ``[B]``), and zero from ``kv_lens[b]`` (int32 CUDA ``[B]``; default: the cache's end) on.
    ``out``: optional pair of tensors to write."""
    if type(cache) is Kv4Cache:
        r = (_lib._binding or _lib.torch_binding()).kv4_read(cache, rows, start, starts, kv_lens, out)
        if r is not None:
            return r
    import torch
    B, Hkv, S, D = _guard_cache(cache)
    rows = int(rows)
    if rows < 0:
        raise _lib.CudaError(_lib.RT_ERR_BAD_LENGTH, "rt_kv4_read")
    at, n = _guard_ints("starts", starts, cache.k_codes, B), _guard_ints("kv_lens", kv_lens, cache.k_codes, B)
    if out is None:
        out = tuple(torch.empty((B, Hkv, rows, D), dtype=torch.bfloat16, device=cache.k_codes.device) for _ in "kv")
    k, v = out
    for name, t in (("out[0]", k), ("out[1]", v)):
        _guard(name, t, torch.bfloat16, like=cache.k_codes, shape=(B, Hkv, rows, D))
    with torch.cuda.device(cache.k_codes.device):
        rc = _lib.lib().rt_kv4_read(*_planes(cache), k.data_ptr(), v.data_ptr(), B, Hkv, D, S, rows, int(start), at, n,
                                    _stream(cache.k_codes.device))
    _lib.check(rc, "rt_kv4_read")
    return k, v


def kv4_workspace_bytes(batch: int, n_heads: int, n_kv_heads: int, head_dim: int, max_seq: int, weighed: bool = False) -> int:
    return int(_lib.lib().rt_kv4_decode_workspace_bytes(batch, n_heads, n_kv_heads, head_dim, max_seq, int(weighed)))


def kv4_decode(q, cache: Kv4Cache, kv_lens=None, kv_len: Optional[int] = None, scale: Optional[float] = None,
               return_lse: bool = True, weights=None, workspace=None, out=None, lse=None):
    """Batched single-token GQA decode over a 4-bit cache via ``rt_kv4_decode``.

    q ``[B,Hq,D]`` bf16, Hq up to 8 times the cache's KV heads; ``kv_lens`` int32 CUDA ``[B]`` or a uniform ``kv_len``.  Returns
    (out bf16 ``[B,Hq,D]``, lse f32 ``[B,Hq]`` or None); both may be passed in.  ``weights``: optional f32 ``[B,Hkv,max_seq]``
    to which every token's softmax weight, summed over the query heads of its KV head, is added.  ``workspace``: optional
    uint8 CUDA tensor of ``kv4_workspace_bytes(...)`` bytes (with ``weights``, ``max_seq`` floats a query head: the scores of a
    long sequence); two calls that overlap on the GPU need one each."""
    if type(cache) is Kv4Cache:
        r = (_lib._binding or _lib.torch_binding()).kv4_decode(q, cache, kv_lens, kv_len, scale, return_lse, weights, workspace, out,
                                                               lse)
        if r is not None:
            return r
    import torch
    B, Hkv, S, D = _guard_cache(cache)
    _guard("q", q, torch.bfloat16, like=cache.k_codes)
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != D:
        raise TypeError(f"q must be [B={B}, Hq, D={D}], got {tuple(q.shape)}")
    Hq = q.shape[1]
    n = _guard_ints("kv_lens", kv_lens, q, B)
    if out is None:
        out = torch.empty_like(q)
    _guard("out", out, torch.bfloat16, like=q, shape=(B, Hq, D))
    if lse is None and return_lse:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device)
    if lse is not None:
        _guard("lse", lse, torch.float32, like=q, shape=(B, Hq))
    if weights is not None:
        _guard("weights", weights, torch.float32, like=q, shape=(B, Hkv, S))
    need = kv4_workspace_bytes(B, Hq, Hkv, D, S, weights is not None)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    else:
        _guard("workspace", workspace, torch.uint8, like=q)
    with torch.cuda.device(q.device):
        rc = _lib.lib().rt_kv4_decode(q.data_ptr(), *_planes(cache), out.data_ptr(), lse.data_ptr() if lse is not None else None,
                                      weights.data_ptr() if weights is not None else None, B, Hq, Hkv, D, S, n,
                                      0 if kv_len is None else int(kv_len), -1.0 if scale is None else float(scale),
                                      workspace.data_ptr() if workspace is not None else None,
                                      workspace.numel() if workspace is not None else 0, _stream(q.device))
    if rc == _lib.RT_ERR_HEAD_COUNT:
        raise HeadCountMismatch(Hq, Hkv)
    _lib.check(rc, "rt_kv4_decode")
    return out, lse
