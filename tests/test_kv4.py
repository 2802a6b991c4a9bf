"""The 4-bit cache and eviction without a GPU: the format's own rules, and every refusal before anything is launched."""
import ctypes

import pytest
import torch

import rustorch_b200 as rt
from tests import kv4_plain as plain


@pytest.mark.parametrize("D", [64, 128, 256])
def test_format_groups_hold_one_octet_of_every_quarter(D):
    of = plain.groups(D)
    W = min(D, 128)
    for g in range(D // 32):
        dims = (of == g).nonzero()[:, 0]
        assert len(dims) == 32
        span = dims[0] // W
        assert {int(d % W) // (W // 4) for d in dims} == {0, 1, 2, 3} and (dims // W == span).all()
    if D <= 128:  # a rotary pair's two values share a group
        assert (of[:D // 2] == of[D // 2:]).all()


@pytest.mark.parametrize("D", [64, 256])
def test_format_is_off_by_half_a_step_at_most(D):
    x = (torch.randn(50, D, generator=torch.Generator().manual_seed(1)) * 3 + 1).bfloat16()
    codes, scales = plain.quantise(x)
    of = plain.groups(D)
    lo, step = scales[..., 1].double()[:, of], scales[..., 0].double()[:, of]
    # half a step, the rounding of the minimum, and of the scale times 15 codes
    slack = 0.5 * step + plain.U_F16 * lo.abs() + 15 * plain.U_F16 * step + 1e-6
    assert ((plain.values(codes, scales) - x.double()).abs() <= slack).all()


def _lib():
    from rustorch_b200 import _lib as L, build
    build.build()
    return L, L.lib()


def test_entries_validate_before_any_device_work():
    L, lib = _lib()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15
    planes = (p, p, p, p)
    a = lambda rows=1, d=128, S=64, pos=0, strides=None, x=p, B=1, H=2: lib.rt_kv4_append(
        *planes, x, p, strides, None, B, H, rows, d, S, pos, None, None, None)
    assert a(d=0) == L.RT_ERR_ZERO_DIM and a(d=96) == L.RT_ERR_UNSUPPORTED and a(rows=-1) == L.RT_ERR_BAD_LENGTH
    assert a(pos=64) == L.RT_ERR_BAD_LENGTH and a(rows=65) == L.RT_ERR_BAD_LENGTH and a(pos=-1) == L.RT_ERR_BAD_LENGTH
    assert a(x=None) == L.RT_ERR_NULL_POINTER and a(x=p + 2) == L.RT_ERR_ALIGNMENT and a(B=65536) == L.RT_ERR_UNSUPPORTED
    assert a(strides=L.int64s([256, 128, 132])) == L.RT_ERR_ALIGNMENT
    assert a(rows=0) == L.RT_OK and a(B=0) == L.RT_OK
    assert lib.rt_kv4_append(p, p, None, p, p, p, None, None, 1, 2, 1, 128, 64, 0, None, None, None) == L.RT_ERR_NULL_POINTER
    assert lib.rt_kv4_append(p, p + 8, p, p, p, p, None, None, 1, 2, 1, 128, 64, 0, None, None, None) == L.RT_ERR_ALIGNMENT

    r = lambda d=128, pos=0, slot=-1, style=0, freq=p, Hq=4: lib.rt_rope_kv4_append(
        p, p, p, *planes, freq, 1, Hq, 2, d, 64, pos, None, slot, None, style, None)
    assert r(d=127) == L.RT_ERR_UNSUPPORTED and r(style=2) == L.RT_ERR_UNSUPPORTED and r(pos=64) == L.RT_ERR_BAD_LENGTH
    assert r(slot=64) == L.RT_ERR_BAD_LENGTH and r(pos=-1, slot=3) == L.RT_ERR_BAD_LENGTH and r(freq=None) == L.RT_ERR_NULL_POINTER

    rd = lambda rows=4, d=128, out=p, start=0: lib.rt_kv4_read(*planes, out, p, 1, 2, d, 64, rows, start, None, None, None)
    assert rd(d=0) == L.RT_ERR_ZERO_DIM and rd(rows=-1) == L.RT_ERR_BAD_LENGTH and rd(out=None) == L.RT_ERR_NULL_POINTER
    assert rd(out=p + 8) == L.RT_ERR_ALIGNMENT and rd(rows=0) == L.RT_OK and rd(start=1 << 40) == L.RT_ERR_UNSUPPORTED

    def d(Hq=4, Hkv=2, D=128, S=64, n=3, out=p, w=None, ws=None, nbytes=0, B=1):
        return lib.rt_kv4_decode(p, *planes, out, None, w, B, Hq, Hkv, D, S, None, n, -1.0, ws, nbytes, None)
    assert d(Hq=5) == L.RT_ERR_HEAD_COUNT and d(Hq=18, Hkv=2) == L.RT_ERR_UNSUPPORTED and d(D=96) == L.RT_ERR_UNSUPPORTED
    assert d(n=65) == L.RT_ERR_BAD_LENGTH and d(n=-1) == L.RT_ERR_BAD_LENGTH and d(out=None) == L.RT_ERR_NULL_POINTER
    assert d(S=1 << 20) == L.RT_ERR_WORKSPACE and d(w=p, S=1 << 20) == L.RT_ERR_WORKSPACE and d(B=0) == L.RT_OK

    def wg(Hq=4, Hkv=2, T=1, D=128, n=3, q=p, lse=p):
        return lib.rt_kv_weigh_bf16(q, p, lse, p, 1, Hq, Hkv, T, D, 64, None, n, -1.0, None)
    assert wg(Hq=5) == L.RT_ERR_HEAD_COUNT and wg(Hq=18) == L.RT_ERR_UNSUPPORTED and wg(D=80) == L.RT_ERR_UNSUPPORTED
    assert wg(T=-1) == L.RT_ERR_BAD_LENGTH and wg(n=65) == L.RT_ERR_BAD_LENGTH and wg(lse=None) == L.RT_ERR_NULL_POINTER
    assert wg(q=p + 4) == L.RT_ERR_ALIGNMENT and wg(T=0) == L.RT_OK

    far = 1 << 40

    def e(src=(far,), dst=(2 * far,), sizes=(256,), keep=4, recent=1, S=64, out=8, n=9, w=p, wo=3 * far, lens=None, lo=p):
        return lib.rt_kv_evict(L.pointers(src), L.pointers(dst), L.int32s(sizes), len(src), w, wo, p, lo, 1, 2, S, out, lens, n,
                               keep, recent, None)
    assert e(keep=0) == L.RT_ERR_BAD_LENGTH and e(keep=9) == L.RT_ERR_BAD_LENGTH and e(recent=5) == L.RT_ERR_BAD_LENGTH
    assert e(recent=-1) == L.RT_ERR_BAD_LENGTH and e(n=65) == L.RT_ERR_BAD_LENGTH and e(w=None) == L.RT_ERR_NULL_POINTER
    assert e(sizes=(12,)) == L.RT_ERR_UNSUPPORTED and e(src=(far + 4,)) == L.RT_ERR_ALIGNMENT
    assert e(src=(far,) * 5, dst=(2 * far,) * 5, sizes=(8,) * 5) == L.RT_ERR_UNSUPPORTED
    assert e(dst=(far + 64 * 2 * 256 - 16,)) == L.RT_ERR_UNSUPPORTED  # the destination begins inside the source
    assert e(w=3 * far) == L.RT_ERR_UNSUPPORTED and e(lens=p) == L.RT_ERR_UNSUPPORTED


def test_cpu_tensors_are_refused():
    c = rt.Kv4Cache.new(1, 2, 16, 64, device="cpu")
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    w = torch.zeros(1, 2, 16)
    for call in (lambda: rt.kv4_append(c, x, x, pos=0), lambda: rt.rope_kv4_append(x, x, x, c, torch.zeros(32), pos=0),
                 lambda: rt.kv4_read(c, 3), lambda: rt.kv4_decode(x, c, kv_len=3), lambda: rt.kv_evict(c, c, w, 4, kv_len=3),
                 lambda: rt.kv_weigh(x, torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16), w[..., 0], w, kv_len=3)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    with pytest.raises(rt.kv4._lib.Unsupported):
        rt.Kv4Cache.new(1, 2, 16, 96, device="cpu")
    assert c.dims == (1, 2, 16, 64) and c.nbytes == 2 * 2 * 16 * (32 + 8)
    with pytest.raises(TypeError, match="Kv4Cache"):
        rt.kv4_decode(x, tuple(c), kv_len=3)
