"""Calls of the 4-bit cache and of eviction next to the edges of what their documentation allows, against forms in 64 bits."""
import math

import pytest

from tests import kv4_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture
def rt():
    import rustorch_b200 as rt
    return rt


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(*shape, seed=0, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale).bfloat16()


def _cut(cache, n):
    return type(cache)(*(t[:, :, :n].contiguous() for t in cache))


# ------------------------------------------------------------------------------------------------ decode


# max_seq 8192 is the longest that one launch of clusters takes; 20,000 is cut into runs for the workers
@pytest.mark.parametrize("S,n", [(8192, 8192), (20000, 20000)])
@pytest.mark.parametrize("D,G", [(64, 4), (128, 1), (128, 4), (128, 8), (256, 2)])
@pytest.mark.parametrize("spread", [1e-4, 3e-4, 1e-3, 1e-2])
def test_decode_of_nearly_equal_scores(rt, S, n, D, G, spread):
    """Attention that is next to a mean: the result is a small rest of values that cancel.

    Rounding p_t to 11 bits moves a term p_t v_t by at most U_F16 of it, one way or the other as the score's last bits have
    it.  n such moves add up to U_F16 sqrt(sum (p_t v_t)^2) (their root mean square), which is U_F16 of the result where the
    values are N(0, 1) and the p_t alike; twice that here.  The result's rounding to bf16 is U_BF16 at most."""
    cache, q = plain.fill(rt, 1, 2, S, D, 11), _randn(1, 2 * G, D, seed=12)
    k = plain.values(cache.k_codes[0, :, :n], cache.k_scales[0, :, :n])
    v = plain.values(cache.v_codes[0, :, :n], cache.v_scales[0, :, :n])
    s = torch.einsum("hgd,htd->hgt", q[0].double().view(2, G, D), k)
    scale = spread * math.log(2) / s.std(-1).mean().item()
    want = torch.einsum("hgt,htd->hgd", torch.softmax(s * scale, -1), v).reshape(2 * G, D)
    out, lse = rt.kv4_decode(q, cache, kv_len=n, scale=scale)
    off = (out[0].double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert off.max() <= plain.U_BF16 + 2 * plain.U_F16, off.max().item()
    assert (lse[0].double() - torch.logsumexp(s * scale, -1).reshape(-1)).abs().max() <= 32 * plain.U_F32 * (1 + math.log(n))


@pytest.mark.parametrize("S", [700, 20000])
@pytest.mark.parametrize("D,G", [(64, 4), (128, 2), (128, 8), (256, 4), (256, 5)])
def test_decode_of_value_groups_far_apart(rt, S, D, G):
    """Values of one group 2^18 times those of the next: each group keeps f16's 11 bits of its probabilities and is then
    rounded to bf16, as `test_decode_of_nearly_equal_scores` has it."""
    g = torch.Generator(device="cuda").manual_seed(21)
    k, v = (torch.randn(1, 2, S, D, device="cuda", generator=g) for _ in "kv")
    of = plain.groups(D).cuda()
    v = v * torch.where(of % 2 == 0, 2.0 ** 11, 2.0 ** -7)
    cache, q = rt.Kv4Cache(*plain.quantise(k.bfloat16()), *plain.quantise(v.bfloat16())), _randn(1, 2 * G, D, seed=22)
    out, _ = rt.kv4_decode(q, cache, kv_len=S)
    want = plain.decode(q, cache, (S,))[0]
    for i in range(D // 32):
        off = (out.double() - want)[..., of == i].norm(dim=-1) / want[..., of == i].norm(dim=-1)
        assert off.max() <= plain.U_BF16 + 2 * plain.U_F16, (i, off.max().item())


@pytest.mark.parametrize("S", [700, 20000])
@pytest.mark.parametrize("D,G,at", [(64, 4, 3), (128, 1, 0), (128, 8, 77), (256, 4, 200)])
@pytest.mark.parametrize("far", [20, 26, 28, 31])
def test_decode_of_queries_with_one_large_value(rt, S, D, G, at, far):
    """One value 2^far times the others, at a place where all keys are zero: the others make the scores.

    Odd places are held in f16 16 times smaller than even ones, the largest value in [2^14, 2^15): f16's last place, 2^-24, is
    2^-34 of the largest there, and half of it is lost of a value, which meets codes of up to 15 scales; a group's sum of
    32 values, in units of 64, loses 2^-33 of the largest, less than the 32 values' 2^-35 each, and meets the minimum."""
    of = plain.groups(D).cuda()
    g = torch.Generator(device="cuda").manual_seed(31)
    k, v = (torch.randn(1, 2, S, D, device="cuda", generator=g) for _ in "kv")
    k[..., of == of[at]] = 0
    cache, q = rt.Kv4Cache(*plain.quantise(k.bfloat16()), *plain.quantise(v.bfloat16())), _randn(1, 2 * G, D, seed=32)
    q[:, :, at] = 2.0 ** far
    out, lse = rt.kv4_decode(q, cache, kv_len=S)
    want, want_lse, _, out_tol, lse_tol, _ = plain.decode(q, cache, (S,))
    scales = cache.k_scales[0].double().abs()
    lost = (2.0 ** (far - 35) * 32 / math.sqrt(D) * (15 * scales[..., 0] + scales[..., 1]).sum(-1)).amax(-1).repeat_interleave(G)
    values = (plain.values(cache.v_codes[0], cache.v_scales[0]).abs() + 15 * cache.v_scales[0, ..., 0].double()[..., of]).amax(1).repeat_interleave(G, 0)
    assert ((lse[0].double() - want_lse[0]).abs() <= lse_tol[0] + lost).all()
    assert ((out[0].double() - want[0]).abs() <= out_tol[0] + 2 * lost[:, None] * values).all()


# ------------------------------------------------------------------------------------------------ weights


@pytest.mark.parametrize("T,D", [(1, 64), (1, 128), (1, 256), (5, 64), (5, 128), (7, 256), (40, 64), (40, 128), (64, 256), (150, 128)])
@pytest.mark.parametrize("junk", [math.nan, math.inf])
def test_weigh_of_rows_that_saw_nothing(rt, T, D, junk):
    """A row whose lse is -inf adds nothing, whatever its query holds: the rows of a batch's padding."""
    B, Hq, Hkv, S = 2, 8, 2, 400
    lens = (400, 211)
    q, k = _randn(B, Hq, T, D, seed=1), _randn(B, Hkv, S, D, seed=2)
    s = torch.einsum("bhqd,bhtd->bhqt", q.double(), k.double().repeat_interleave(Hq // Hkv, 1)) / math.sqrt(D)
    lse = torch.logsumexp(s, -1).float()
    gone = torch.rand(B, Hq, T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.4
    gone[:, 0], gone[:, 1] = True, False  # in every group some and not all
    lse[gone] = -math.inf
    w = torch.zeros(B, Hkv, S, device="cuda")
    want, tol = plain.weigh(q, k, lse, lens)
    bad = torch.where(gone[..., None], torch.full_like(q, junk), q)
    if T == 1:
        rt.kv_weigh(bad[:, :, 0].contiguous(), k, lse[:, :, 0].contiguous(), w, kv_lens=_i32(*lens))
    else:
        rt.kv_weigh(bad, k, lse, w, kv_lens=_i32(*lens))
    assert ((w.double() - want).abs() <= tol + 2 * plain.U_F32 * (1 + want)).all()
