"""Weights over a bf16 cache and eviction, against plain forms."""
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


def _weigh(rt, B, Hq, Hkv, T, D, S, lens, seed=1, scale=None):
    q, k = _randn(B, Hq, T, D, seed=seed), _randn(B, Hkv, S, D, seed=seed + 1)
    lse = torch.empty(B, Hq, T, device="cuda")
    for b in range(B):
        n = min(max(lens[b], 0), S)
        s = torch.einsum("hqd,htd->hqt", q[b].double(), k[b, :, :n].double().repeat_interleave(Hq // Hkv, 0))
        s *= 1 / math.sqrt(D) if scale is None else scale
        at = n - T + torch.arange(T, device="cuda")
        s.masked_fill_(torch.arange(n, device="cuda") > at[:, None], -math.inf)
        lse[b] = torch.logsumexp(s, -1).float() if n else -math.inf
    before = torch.rand(B, Hkv, S, device="cuda")
    w = before.clone()
    if T == 1:
        rt.kv_weigh(q[:, :, 0].contiguous(), k, lse[:, :, 0].contiguous(), w, kv_lens=_i32(*lens), scale=scale)
    else:
        rt.kv_weigh(q, k, lse, w, kv_lens=_i32(*lens), scale=scale)
    want, tol = plain.weigh(q, k, lse, lens, scale)
    off = (w.double() - before.double() - want).abs()
    bad = off > tol + 2 * plain.U_F32 * (1 + want)
    assert not bad.any(), (off[bad].max().item(), tol[bad].min().item(), int(bad.sum()))
    for b, n in enumerate(lens):
        n = min(max(n, 0), S)
        assert torch.equal(w[b, :, n:], before[b, :, n:])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
def test_weigh_groups_and_head_dims(rt, D, G):
    _weigh(rt, 2, 2 * G, 2, 1, D, 150, (150, 77), seed=G)
    _weigh(rt, 2, 2 * G, 2, 9, D, 150, (150, 77), seed=G)


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("T", [1, 3, 16, 33])
def test_weigh_lengths(rt, n, T):
    """Among them fewer tokens than queries: the first queries see nothing."""
    _weigh(rt, 1, 8, 2, T, 128, 1000, (n,), seed=n)


@pytest.mark.parametrize("B,Hq,Hkv,T,D,S,lens", [
    (5, 8, 1, 1, 128, 1, (1, 0, 1, 7, -3)),
    (3, 14, 2, 5, 64, 513, (513, 2, 300)),
    (33, 8, 8, 1, 128, 130, tuple(4 * i for i in range(33))),
    (1, 4, 1, 130, 256, 300, (299,)),
    (2, 8, 2, 64, 128, 2000, (2000, 1111)),
    (1, 2, 2, 257, 64, 257, (257,)),
])
def test_weigh_batches(rt, B, Hq, Hkv, T, D, S, lens):
    _weigh(rt, B, Hq, Hkv, T, D, S, lens, scale=0.11)


def test_weigh_of_what_decode_and_prefill_return(rt):
    """The weights of a decode's queries sum to one each, those of a prompt's last queries too."""
    B, Hq, Hkv, D, S = 2, 8, 2, 128, 500
    k, v, q = _randn(B, Hkv, S, D, seed=1), _randn(B, Hkv, S, D, seed=2), _randn(B, Hq, D, seed=3)
    lens = _i32(500, 123)
    _, lse = rt.gqa_decode(q, k, v, kv_lens=lens)
    w = torch.zeros(B, Hkv, S, device="cuda")
    rt.kv_weigh(q, k, lse, w, kv_lens=lens)
    # a sum over 500 weights, each off by about the steps of its score (|s| < 16) and of lse
    assert (w.sum(-1) - Hq // Hkv).abs().max() < 500 * 2.0 ** -24 + 64 * 16 * 2.0 ** -24
    T = 40
    q = _randn(B, Hq, T, D, seed=4)
    _, lse = rt.prefill_bf16(q, k, v, causal=True, kv_lens=lens, q_offsets=lens - T)
    w.zero_()
    rt.kv_weigh(q, k, lse, w, kv_lens=lens)
    assert (w.sum(-1) / (T * Hq // Hkv) - 1).abs().max() < 1e-4  # the prefill's own lse: approximate exponentials


def test_weigh_rows_behind_the_length_are_not_read(rt):
    q, k = _randn(1, 4, 64, seed=1), _randn(1, 2, 100, 64, seed=2)
    lse, w = torch.full((1, 4), 3.0, device="cuda"), torch.zeros(1, 2, 100, device="cuda")
    rt.kv_weigh(q, k, lse, w, kv_len=37)
    k[:, :, 37:] = math.nan
    w2 = torch.zeros_like(w)
    rt.kv_weigh(q, k, lse, w2, kv_len=37)
    assert torch.equal(w, w2) and not w[:, :, 37:].any()


# ------------------------------------------------------------------------------------------------ eviction


def _evict(rt, bits, B, Hkv, D, S, S_out, lens, keep, recent, weights=None, uniform=False, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if weights is None:  # heavy tails, and many equal ones
        weights = torch.exp(2 * torch.randn(B, Hkv, S, device="cuda", generator=g))
        weights *= torch.rand(B, Hkv, S, device="cuda", generator=g) > 0.3
        weights = torch.where(torch.rand(B, Hkv, S, device="cuda", generator=g) > 0.2, weights, 0.25)
    if bits == 4:
        cache = plain.fill(rt, B, Hkv, S, D, seed)
        out = rt.Kv4Cache(*(t.random_(0, 200) if t.dtype == torch.uint8 else t.fill_(7) for t in rt.Kv4Cache.new(B, Hkv, S_out, D)))
    else:
        cache = (_randn(B, Hkv, S, D, seed=seed), _randn(B, Hkv, S, D, seed=seed + 1))
        out = tuple(torch.full((B, Hkv, S_out, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    before, source = [t.clone() for t in out], [t.clone() for t in cache]
    kw = dict(kv_len=lens[0]) if uniform else dict(kv_lens=_i32(*lens))
    new_lens, w_out, kept = rt.kv_evict(cache, out, weights, keep, recent=recent, **kw)
    want = plain.evict(weights, lens, keep, recent)
    assert new_lens.dtype == torch.int32 and new_lens.tolist() == [min(max(n, 0), S, keep) for n in lens]
    for b in range(B):
        for h in range(Hkv):
            at = want[b][h]
            m = len(at)
            assert kept[b, h].tolist() == at + [-1] * (keep - m), (b, h)
            idx = torch.tensor(at, dtype=torch.long, device="cuda")
            assert torch.equal(w_out[b, h, :m].nan_to_num(9e9), weights[b, h, idx].nan_to_num(9e9)) and not w_out[b, h, m:].any()
            for o, c, was in zip(out, cache, before):
                assert torch.equal(o[b, h, :m], c[b, h, idx]) and torch.equal(o[b, h, m:], was[b, h, m:])
    for a, b in zip(cache, source):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits,D", [(16, 64), (16, 128), (16, 256), (4, 64), (4, 128), (4, 256)])
def test_evict_caches(rt, bits, D):
    _evict(rt, bits, 3, 2, D, 300, 120, (300, 40, 151), 100, 7)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (2, 1), (17, 17), (64, 0), (500, 3), (2000, 1000), (2999, 5)])
def test_evict_sizes(rt, keep, recent):
    _evict(rt, 4, 1, 3, 64, 3000, keep + 3, (3000,), keep, recent, uniform=True)
    _evict(rt, 16, 2, 1, 64, 3000, keep, (keep + 1 if keep < 3000 else keep, keep), keep, recent)


@pytest.mark.parametrize("n", [0, 1, 99, 100, 101, 1023, 1024, 1025, 4097, 9000])
def test_evict_lengths(rt, n):
    _evict(rt, 4, 2, 2, 64, 9000, 128, (n, 5), 100, 10, seed=n)


@pytest.mark.parametrize("what", ["zeros", "equal", "negative", "special", "denormal", "sorted", "close"])
def test_evict_order_of_weights(rt, what):
    """Ties go to the first; -0 is 0; NaN is the largest, infinities and negatives in their places."""
    S = 2500
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.rand(1, 2, S, device="cuda", generator=g)
    if what == "zeros":
        w = torch.where(torch.rand(1, 2, S, device="cuda", generator=g) > 0.5, 0.0, -0.0)
    elif what == "equal":
        w = torch.full((1, 2, S), 0.7, device="cuda")
    elif what == "negative":
        w = torch.randn(1, 2, S, device="cuda", generator=g)
    elif what == "special":
        w[:, :, ::50], w[:, :, 1::70], w[:, :, 2::90] = math.nan, math.inf, -math.inf
    elif what == "denormal":
        w = (w * 50).floor() * 1e-45
    elif what == "sorted":
        w = torch.arange(S, device="cuda").float().expand(1, 2, S).contiguous()
    else:
        w = 1 + (w * 100).floor() * 2.0 ** -23
    _evict(rt, 16, 1, 2, 64, S, 700, (S,), 700, 50, weights=w)


def test_evict_large(rt):
    _evict(rt, 16, 1, 2, 128, 40000, 9000, (39001,), 9000, 1000)
    _evict(rt, 4, 70, 8, 64, 150, 40, tuple(2 * i + 3 for i in range(70)), 40, 4)


def test_evict_refusals(rt):
    from rustorch_b200 import _lib
    a, b = rt.Kv4Cache.new(1, 2, 32, 64), rt.Kv4Cache.new(1, 2, 16, 64)
    w = torch.zeros(1, 2, 32, device="cuda")
    for keep, recent in ((0, 0), (17, 0), (8, 9), (8, -1)):
        with pytest.raises(_lib.CudaError):
            rt.kv_evict(a, b, w, keep, recent=recent, kv_len=20)
    with pytest.raises(_lib.CudaError):
        rt.kv_evict(a, b, w, 8, kv_len=33)
    with pytest.raises(_lib.Unsupported):  # the move has no order: not in place
        rt.kv_evict(a, a, w, 8, kv_len=20)
    with pytest.raises(TypeError):
        rt.kv_evict(a, (a[0], a[2]), w, 8, kv_len=20)
    with pytest.raises(TypeError, match="out must be"):
        rt.kv_evict(a, rt.Kv4Cache.new(1, 2, 16, 128), w, 8, kv_len=20)
    with pytest.raises(TypeError, match="weights"):
        rt.kv_evict(a, b, w.double(), 8, kv_len=20)


def test_evicted_decode_loop(rt):
    """Decode steps that weigh, an eviction, and steps behind it: rows apart from positions, weights that start at zero."""
    B, Hq, Hkv, D, S = 2, 8, 2, 64, 300
    cache, small = plain.fill(rt, B, Hkv, S, D, 1), rt.Kv4Cache.new(B, Hkv, 80, D)
    freq, lens = rt.rope_inv_freq(D), _i32(250, 40)
    weights = torch.zeros(B, Hkv, S, device="cuda")
    positions = lens.clone()
    for step in range(2):
        q, k, v = (_randn(B, h, D, seed=10 * step + i) for i, h in enumerate((Hq, Hkv, Hkv)))
        rt.rope_kv4_append(q, k, v, cache, freq, positions=positions)
        positions = positions + 1
        rt.kv4_decode(q, cache, kv_lens=positions, weights=weights)
    total = weights.sum(-1)
    assert (total - 2 * Hq // Hkv).abs().max() < 1e-4
    lens, weights, kept = rt.kv_evict(cache, small, weights, 64, recent=8, kv_lens=positions)
    assert lens.tolist() == [64, 42] and kept[0, 0, -8:].tolist() == list(range(244, 252))
    assert (weights.sum(-1) <= total + 1e-4).all() and (weights[1].sum(-1) - total[1]).abs().max() < 1e-5
    for step in range(3):
        q, k, v = (_randn(B, h, D, seed=50 + 10 * step + i) for i, h in enumerate((Hq, Hkv, Hkv)))
        rt.rope_kv4_append(q, k, v, small, freq, positions=positions, slots=lens)
        positions, lens = positions + 1, lens + 1
        before = weights.clone()
        out, lse = rt.kv4_decode(q, small, kv_lens=lens, weights=weights)
        o, l, w, ot, lt, wt = plain.decode(q, small, lens.tolist())
        assert ((out.double() - o).abs() <= ot).all() and ((lse.double() - l).abs() <= lt).all()
        assert ((weights - before).double() - w).abs().max() <= wt.max() + 4 * plain.U_F32 * (1 + float(before.max()))
        assert not before[0, :, 64 + step:].any()  # what was appended behind the kept rows starts at zero
