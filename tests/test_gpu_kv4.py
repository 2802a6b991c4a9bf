"""The 4-bit KV cache on the GPU against plain forms in f32 (the format) and 64 bits (the attention)."""
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


def _same(got, want):
    return torch.equal(torch.nan_to_num(got.float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0))


# ------------------------------------------------------------------------------------------------ append and read


@pytest.mark.parametrize("B,H,T,D,S,starts,lens", [
    (1, 1, 1, 64, 1, (0,), (1,)),
    (2, 3, 5, 128, 33, (0, 28), (5, 3)),
    (3, 2, 70, 256, 77, (7, 0, 1), (0, 70, 69)),
    (2, 8, 130, 128, 131, (1, 0), (130, 1)),
    (1, 5, 257, 64, 300, (43,), (257,)),
])
def test_append_quantises_as_the_format_says(rt, B, H, T, D, S, starts, lens):
    k, v = _randn(B, H, T, D, seed=1, scale=3), _randn(B, H, T, D, seed=2)
    cache = rt.Kv4Cache(*(t.random_(0, 200) if t.dtype == torch.uint8 else t.fill_(7) for t in rt.Kv4Cache.new(B, H, S, D)))
    want = [t.clone() for t in cache]
    rt.kv4_append(cache, k, v, positions=_i32(*starts), lens=_i32(*lens))
    for b in range(B):
        at = slice(starts[b], starts[b] + lens[b])
        for i, x in ((0, k), (2, v)):
            want[i][b, :, at], want[i + 1][b, :, at] = plain.quantise(x[b, :, :lens[b]])
    for got, w in zip(cache, want):  # the rows around them as they were
        assert torch.equal(got, w)
    ends = _i32(*(s + n for s, n in zip(starts, lens)))
    for got, i in zip(rt.kv4_read(cache, T, starts=_i32(*starts), kv_lens=ends), (0, 2)):
        for b in range(B):
            rows = plain.values(want[i][b], want[i + 1][b], torch.float32)[:, starts[b]:starts[b] + lens[b]]
            assert torch.equal(got[b, :, :lens[b]], rows.bfloat16()) and not got[b, :, lens[b]:].any()


@pytest.mark.parametrize("layout", ["projection", "sliced", "one row", "broadcast"])
def test_append_takes_strided_rows(rt, layout):
    B, H, T, D = 2, 3, 9, 128
    if layout == "projection":
        k, v = (_randn(B, T, H, D, seed=i).permute(0, 2, 1, 3) for i in (1, 2))
    elif layout == "sliced":
        k, v = (_randn(B, H, T + 4, 2 * D, seed=i)[:, :, 2:-2, D:] for i in (1, 2))
    elif layout == "broadcast":
        k, v = (_randn(1, 1, T, D, seed=i).expand(B, H, T, D) for i in (1, 2))
    else:
        T = 1
        k, v = (_randn(B, H, 1, D, seed=i) for i in (1, 2))
        k, v = k[:, :, 0], v.as_strided((B, H, 1, D), (H * D, D, 3, 1))  # a stride that nothing steps by
    cache, dense = rt.Kv4Cache.new(B, H, 12, D), rt.Kv4Cache.new(B, H, 12, D)
    rt.kv4_append(cache, k, v, pos=3)
    rt.kv4_append(dense, k.contiguous().view(B, H, T, D), v.contiguous().view(B, H, T, D), pos=3)
    for a, b in zip(cache, dense):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_of_extreme_values(rt, D):
    """Constant rows, zeros, tiny and huge ranges, infinities, values past fp16, NaN in one group; ties to the even code."""
    x = torch.zeros(1, 1, 10, D)
    x[0, 0, 1] = 3.0
    x[0, 0, 2] = torch.linspace(-1, 1, D) * 1e-7
    x[0, 0, 3] = torch.linspace(-3e38, 3e38, D)
    x[0, 0, 4, 5], x[0, 0, 4, 6] = math.inf, -math.inf
    x[0, 0, 5] = torch.linspace(0, 1, D)
    x[0, 0, 5, 9] = math.nan
    x[0, 0, 6] = torch.arange(D) % 16 + 0.5 * (torch.arange(D) % 3 == 1)
    x[0, 0, 7] = -70000.0
    x[0, 0, 8, ::2] = 1e-30
    x[0, 0, 9] = torch.arange(D) - 128.0
    x = x.bfloat16().cuda()
    cache = rt.Kv4Cache.new(1, 1, 10, D)
    rt.kv4_append(cache, x, -x)
    for i, y in ((0, x), (2, -x)):
        codes, scales = plain.quantise(y)
        assert torch.equal(cache[i], codes) and _same(cache[i + 1], scales)
    k, _ = rt.kv4_read(cache, 10)
    assert _same(k, plain.values(cache[0], cache[1], torch.float32).bfloat16())
    assert int(k[0, 0, 5].isnan().sum()) == 32 and k[0, 0, 4].isfinite().all()


def test_append_drops_rows_outside_the_cache(rt):
    cache = rt.Kv4Cache.new(3, 1, 8, 64)
    x = _randn(3, 1, 4, 64, seed=3)
    rt.kv4_append(cache, x, x, positions=_i32(6, -2, 100))
    codes, scales = plain.quantise(x)
    assert torch.equal(cache[0][0, 0, 6:], codes[0, 0, :2]) and torch.equal(cache[0][1, 0, :2], codes[1, 0, 2:])
    assert not cache[0][0, 0, :6].any() and not cache[0][1, 0, 2:].any() and not cache[0][2].any() and not cache[1][2].any()


def test_read_outside_the_sequence_is_zero(rt):
    cache = plain.fill(rt, 2, 2, 20, 128, 4)
    k, v = rt.kv4_read(cache, 9, starts=_i32(-3, 15), kv_lens=_i32(4, 99))
    for got, i in ((k, 0), (v, 2)):
        want = plain.values(cache[i], cache[i + 1], torch.float32).bfloat16()
        assert not got[0, :, :3].any() and torch.equal(got[0, :, 3:7], want[0, :, :4]) and not got[0, :, 7:].any()
        assert torch.equal(got[1, :, :5], want[1, :, 15:]) and not got[1, :, 5:].any()
    assert rt.kv4_read(cache, 0)[0].shape == (2, 2, 0, 128)


@pytest.mark.parametrize("style", ["half_split", "adjacent"])
@pytest.mark.parametrize("B,Hq,Hkv,D", [(1, 1, 1, 64), (3, 7, 1, 128), (2, 8, 4, 256), (5, 32, 8, 128)])
def test_rope_append_is_rope_kv_append_quantised(rt, B, Hq, Hkv, D, style):
    S = 5000
    q, k, v = _randn(B, Hq, D, seed=1), _randn(B, Hkv, D, seed=2), _randn(B, Hkv, D, seed=3)
    freq, at = rt.rope_inv_freq(D), _i32(*(4999 - 1000 * b for b in range(B)))
    kc, vc = torch.zeros(B, Hkv, S, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, Hkv, S, D, device="cuda", dtype=torch.bfloat16)
    q_ref = q.clone()
    rt.rope_kv_append(q_ref, k, v, kc, vc, freq, positions=at, style=style)
    rows = torch.arange(B, device="cuda"), at.long()
    for slots in (None, _i32(*(17 + b for b in range(B)))):
        cache, q4 = rt.Kv4Cache.new(B, Hkv, S, D), q.clone()
        rt.rope_kv4_append(q4, k, v, cache, freq, positions=at, slots=slots, style=style)
        assert torch.equal(q4, q_ref)
        to = at.long() if slots is None else slots.long()
        for i, ref in ((0, kc), (2, vc)):
            codes, scales = plain.quantise(ref[rows[0], :, rows[1]])
            assert torch.equal(cache[i][rows[0], :, to], codes) and torch.equal(cache[i + 1][rows[0], :, to], scales)
            assert int(cache[i + 1].abs().sum(-1).sum(-1).count_nonzero()) == B * Hkv  # no other row


def test_rope_append_leaves_invalid_sequences_alone(rt):
    q, k = _randn(3, 4, 64, seed=1), _randn(3, 2, 64, seed=2)
    cache, before = rt.Kv4Cache.new(3, 2, 8, 64), q.clone()
    rt.rope_kv4_append(q, k, k, cache, rt.rope_inv_freq(64), positions=_i32(-1, 8, 3), style="half_split")
    assert torch.equal(q[:2], before[:2]) and not torch.equal(q[2], before[2]) and not cache[1][:2].any()
    q = before.clone()  # a position past the cache, at a row inside it
    rt.rope_kv4_append(q, k, k, cache, rt.rope_inv_freq(64), pos=100, slot=1)
    assert not torch.equal(q[0], before[0]) and cache[1][:, :, 1].any(-1).any(-1).all()


# ------------------------------------------------------------------------------------------------ decode


def _check(got, want, tol, what):
    off = (got.double() - want).abs()
    finite = want.isfinite()
    assert torch.equal(got[~finite].double(), want[~finite]), what
    bad = finite & ~(off <= tol)
    assert not bad.any(), f"{what}: off by {off[bad].max().item():.3g}, allowed {tol[bad][off[bad].argmax()].item():.3g}, {int(bad.sum())} values"


def _decode_case(rt, B, Hq, Hkv, D, S, lens, seed=0, scale=None, uniform=False, q=None, cache=None):
    cache = plain.fill(rt, B, Hkv, S, D, seed) if cache is None else cache
    q = _randn(B, Hq, D, seed=seed + 50) if q is None else q
    before = torch.rand(B, Hkv, S, device="cuda")
    weights = before.clone()
    kw = dict(kv_len=lens[0]) if uniform else dict(kv_lens=_i32(*lens))
    out, lse = rt.kv4_decode(q, cache, scale=scale, weights=weights, **kw)
    o, l, w, ot, lt, wt = plain.decode(q, cache, lens, scale)
    _check(out, o, ot, "out")
    _check(lse, l, lt, "lse")
    _check(weights, before.double() + w, wt + 2 * plain.U_F32 * (1 + w), "weights")
    out2, none = rt.kv4_decode(q, cache, scale=scale, return_lse=False, **kw)
    assert none is None and torch.equal(out2, out)
    for b, n in enumerate(lens):
        n = min(max(n, 0), S)
        assert torch.equal(weights[b, :, n:], before[b, :, n:])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8])
def test_decode_groups_and_head_dims(rt, D, G):
    _decode_case(rt, 2, 2 * G, 2, D, 200, (200, 137), seed=G)


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2047, 4096])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_lengths(rt, D, n):
    _decode_case(rt, 1, 8, 2, D, 4096, (n,), seed=n, uniform=True)


@pytest.mark.parametrize("B,Hq,Hkv,D,S,lens", [
    (5, 8, 1, 128, 1, (1, 0, 1, 7, -3)),                  # a cache of one row; lengths outside it
    (4, 4, 4, 64, 513, (513, 0, 1, 300)),
    (3, 14, 2, 256, 3001, (3001, 64, 1500)),
    (1, 32, 8, 128, 20000, (19999,)),
    (37, 8, 8, 128, 150, tuple(range(3, 151, 4))),
    (2, 16, 2, 64, 40001, (40001, 12345)),
    (64, 32, 8, 128, 600, tuple(5 + 9 * i for i in range(64))),
    (130, 8, 4, 64, 260, tuple((i * 37) % 261 for i in range(130))),
])
def test_decode_batches(rt, B, Hq, Hkv, D, S, lens):
    _decode_case(rt, B, Hq, Hkv, D, S, lens, seed=7)


def test_decode_rows_behind_the_length_are_not_read(rt):
    """Scales of NaN and infinity in the rows behind a sequence change nothing."""
    cache = plain.fill(rt, 2, 2, 300, 128, 5)
    q = _randn(2, 8, 128, seed=6)
    want = rt.kv4_decode(q, cache, kv_lens=_i32(100, 7))
    for i in (1, 3):
        cache[i][0, :, 100:] = math.nan
        cache[i][1, :, 7:] = math.inf
    got = rt.kv4_decode(q, cache, kv_lens=_i32(100, 7))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("what", ["far scores", "one token", "large q", "small q", "tiny v", "huge v", "mixed v", "scale"])
def test_decode_of_wide_ranges(rt, what):
    B, Hq, Hkv, D, S = 1, 8, 2, 128, 700
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = (torch.randn(B, Hkv, S, D, device="cuda", generator=g) for _ in "kv")
    q, scale = _randn(B, Hq, D, seed=9), None
    if what == "far scores":
        k = k * 30
    elif what == "one token":
        k[:, :, 333] += 8 * q.view(B, Hkv, -1, D)[:, :, 0].float()
    elif what == "large q":
        q, scale = (q.float() * 2.0 ** 60).bfloat16(), 2.0 ** -62
    elif what == "small q":
        q, scale = (q.float() * 2.0 ** -90).bfloat16(), 2.0 ** 88
    elif what == "tiny v":
        v = v * 2e-4
    elif what == "huge v":
        v = v * 9000
    elif what == "mixed v":
        v[:, :, ::3] *= 4000
    else:
        scale = 0.7
    cache = rt.Kv4Cache(*plain.quantise(k.bfloat16()), *plain.quantise(v.bfloat16()))
    _decode_case(rt, B, Hq, Hkv, D, S, (S,), scale=scale, q=q, cache=cache)


def test_decode_of_a_zero_cache_and_of_nan(rt):
    cache = rt.Kv4Cache.new(1, 2, 100, 64)
    q = _randn(1, 4, 64, seed=1)
    out, lse = rt.kv4_decode(q, cache, kv_len=100)
    assert not out.any() and (lse - math.log(100)).abs().max() < 1e-5
    q[0, 1, 3] = math.nan
    out, lse = rt.kv4_decode(q, cache, kv_len=100)
    assert out[0, 1].isnan().all() and lse[0, 1].isnan() and not out[0, [0, 2, 3]].any()
    x = _randn(1, 2, 1, 64, seed=2)
    x[0, 1, 0, 0] = math.nan  # one key of head 1
    rt.kv4_append(cache, x, x.nan_to_num(0.0), pos=50)
    out, lse = rt.kv4_decode(_randn(1, 4, 64, seed=1), cache, kv_len=100)
    assert out[0, 2:].isnan().all() and lse[0, 2:].isnan().all() and out[0, :2].isfinite().all()
    x = _randn(1, 2, 1, 64, seed=2)
    v = x.clone()
    v[0, 1, 0, 0] = math.nan  # and one value: its group of 32
    rt.kv4_append(cache, x, v, pos=50)
    out, lse = rt.kv4_decode(_randn(1, 4, 64, seed=1), cache, kv_len=100)
    of = plain.groups(64).cuda()
    assert torch.equal(out[0, 2:].isnan(), (of == 0).expand(2, 64)) and lse.isfinite().all()


def test_decode_streams_graphs_and_workspaces(rt):
    """Two streams at once, and two graphs replayed with lengths that changed between the replays."""
    B, Hq, Hkv, D, S = 2, 8, 2, 128, 3000
    caches = [plain.fill(rt, B, Hkv, S, D, s) for s in (1, 2)]
    qs = [_randn(B, Hq, D, seed=s) for s in (3, 4)]
    lens = [_i32(3000, 100), _i32(5, 2999)]
    want = [rt.kv4_decode(q, c, kv_lens=n) for q, c, n in zip(qs, caches, lens)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in "ab"]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = rt.kv4_decode(qs[i], caches[i], kv_lens=lens[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    weights = torch.zeros(B, Hkv, S, device="cuda")
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(rt.kv4_decode(qs[i], caches[i], kv_lens=lens[i], weights=weights))
        graphs.append(graph)
    for swap in (False, True):
        if swap:
            a = lens[0].clone()
            lens[0].copy_(lens[1])
            lens[1].copy_(a)
        for i in (0, 1):
            weights.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            fresh = torch.zeros_like(weights)
            w = rt.kv4_decode(qs[i], caches[i], kv_lens=lens[i], weights=fresh)
            assert torch.equal(outs[i][0], w[0]) and torch.equal(outs[i][1], w[1]) and torch.equal(weights, fresh)


def test_decode_caller_owned_outputs_and_workspace(rt):
    B, Hq, Hkv, D, S = 3, 8, 2, 64, 900
    cache, q = plain.fill(rt, B, Hkv, S, D, 3), _randn(B, Hq, D, seed=4)
    want = rt.kv4_decode(q, cache, kv_len=900)
    out, lse = torch.full_like(q, math.nan), torch.full((B, Hq), math.nan, device="cuda")
    ws = torch.full((max(1, rt.kv4_workspace_bytes(B, Hq, Hkv, D, S, True)),), 255, dtype=torch.uint8, device="cuda")
    got = rt.kv4_decode(q, cache, kv_len=900, out=out, lse=lse, workspace=ws)
    assert got[0] is out and got[1] is lse and torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_decode_refusals(rt):
    from rustorch_b200 import _lib
    cache, q = rt.Kv4Cache.new(2, 2, 16, 64), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError, match="q must be"):
        rt.kv4_decode(q[:1].contiguous(), cache, kv_len=3)
    with pytest.raises(TypeError, match="bfloat16"):
        rt.kv4_decode(q.float(), cache, kv_len=3)
    with pytest.raises(TypeError, match="kv_lens"):
        rt.kv4_decode(q, cache, kv_lens=torch.tensor([3, 4], device="cuda"))
    with pytest.raises(TypeError, match="contiguous"):
        rt.kv4_decode(q, rt.Kv4Cache(*(t.transpose(1, 2) for t in cache)), kv_len=3)
    with pytest.raises(TypeError, match="k_scales"):
        rt.kv4_decode(q, cache._replace(k_scales=cache.k_scales[:, :, :8].contiguous()), kv_len=3)
    with pytest.raises(TypeError, match="weights"):
        rt.kv4_decode(q, cache, kv_len=3, weights=torch.zeros(2, 2, 15, device="cuda"))
    with pytest.raises(rt.HeadCountMismatch):
        rt.kv4_decode(torch.zeros(2, 5, 64, dtype=torch.bfloat16, device="cuda"), cache, kv_len=3)
    with pytest.raises(_lib.Unsupported):
        rt.kv4_decode(torch.zeros(2, 18, 64, dtype=torch.bfloat16, device="cuda"), cache, kv_len=3)
    with pytest.raises(_lib.CudaError):
        rt.kv4_decode(q, cache, kv_len=17)
    x = torch.zeros(2, 2, 17, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.CudaError):
        rt.kv4_append(cache, x, x)
    with pytest.raises(TypeError, match="head dim"):
        rt.kv4_append(cache, x.transpose(2, 3).contiguous().transpose(2, 3), x)
    with pytest.raises(_lib.CudaError):
        rt.kv4_append(cache, torch.zeros(2, 2, 4, 65, dtype=torch.bfloat16, device="cuda")[..., :64],
                      torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16, device="cuda"))


def test_offsets_past_32_bits(rt):
    """The second head's rows start behind 2^32 bytes of codes."""
    S, D = 34_000_000, 256
    cache = rt.Kv4Cache(*(torch.empty((1, 2, S) + tail, dtype=t, device="cuda") for _ in "kv"
                          for tail, t in (((D // 2,), torch.uint8), ((D // 32, 2), torch.float16))))
    k, v = _randn(1, 2, 70, D, seed=1), _randn(1, 2, 70, D, seed=2)
    rt.kv4_append(cache, k, v, pos=0)
    rt.kv4_append(cache, k, v, pos=S - 70)
    small = rt.Kv4Cache.new(1, 2, 70, D)
    rt.kv4_append(small, k, v)
    for at in (0, S - 70):
        for a, b in zip(rt.kv4_read(cache, 70, start=at), rt.kv4_read(small, 70)):
            assert torch.equal(a, b)
    q = _randn(1, 4, D, seed=3)
    o, l, _, ot, lt, _ = plain.decode(q, small, (70,))
    out, lse = rt.kv4_decode(q, cache, kv_len=70)
    _check(out, o, ot, "out")
    _check(lse, l, lt, "lse")


def test_steps_of_a_token_loop(rt):
    """Prompt append, the chunk's read-back and prefill, then steps of rope, append and decode: each against 64 bits on the
    cache's own values."""
    B, Hq, Hkv, D, S, T = 2, 8, 2, 128, 400, 150
    cache = rt.Kv4Cache.new(B, Hkv, S, D)
    k, v = (_randn(B, T, Hkv, D, seed=i).permute(0, 2, 1, 3) for i in (1, 2))
    lens = _i32(150, 97)
    rt.kv4_append(cache, k, v, lens=lens)
    kb, vb = rt.kv4_read(cache, T, kv_lens=lens)
    q = _randn(B, Hq, T, D, seed=3)
    out, lse = rt.prefill_bf16(q, kb, vb, causal=True, kv_lens=lens)
    for b in range(B):
        kk, vv = (plain.values(cache[i][b], cache[i + 1][b])[:, :T].repeat_interleave(Hq // Hkv, 0) for i in (0, 2))
        s = torch.einsum("hqd,htd->hqt", q[b].double(), kk) / math.sqrt(D)
        s.masked_fill_(torch.ones(T, T, device="cuda").triu(1).bool(), -math.inf)
        s[:, :, int(lens[b]):] = -math.inf
        want = torch.softmax(s, -1) @ vv
        n = int(lens[b])
        assert (out[b, :, :n].double() - want[:, :n]).abs().max() <= 0.03  # values of 4: K, V and the result in bf16
    freq, one = rt.rope_inv_freq(D), torch.ones_like(lens)
    for step in range(3):
        qs, ks, vs = _randn(B, Hq, D, seed=10 + step), _randn(B, Hkv, D, seed=20 + step), _randn(B, Hkv, D, seed=30 + step)
        rt.rope_kv4_append(qs, ks, vs, cache, freq, positions=lens)
        lens = lens + one
        o, l, _, ot, lt, _ = plain.decode(qs, cache, lens.tolist())
        got, got_lse = rt.kv4_decode(qs, cache, kv_lens=lens)
        _check(got, o, ot, "out")
        _check(got_lse, l, lt, "lse")


# ------------------------------------------------------------------------------------------------ the two paths to the entries


class _Nothing:
    """Stands in for the extension and covers nothing."""
    def __getattr__(self, name):
        return lambda *args: None


def _every_call(rt):
    B, Hq, Hkv, D, S = 2, 8, 2, 64, 100
    lens, at = _i32(90, 13), _i32(95, 14)
    q, k, v = _randn(B, Hq, D, seed=1), _randn(B, Hkv, D, seed=2), _randn(B, Hkv, D, seed=3)
    cache = plain.fill(rt, B, Hkv, S, D, 4)
    rt.kv4_append(cache, k, v, pos=2)
    rt.kv4_append(cache, *(_randn(B, 5, Hkv, D, seed=i).transpose(1, 2) for i in (5, 6)), positions=_i32(20, 99), lens=_i32(5, 1))
    rt.rope_kv4_append(q, k, v, cache, rt.rope_inv_freq(D), positions=at, slot=40, style="adjacent")
    rt.rope_kv4_append(q, k, v, cache, rt.rope_inv_freq(D), pos=7, slots=at)
    weights, ws = torch.zeros(B, Hkv, S, device="cuda"), torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    out, lse = rt.kv4_decode(q, cache, kv_lens=lens, weights=weights, scale=0.2, workspace=ws)
    out2, none = rt.kv4_decode(q, cache, kv_len=77, return_lse=False, out=torch.empty_like(q))
    assert none is None
    kb, vb = rt.kv4_read(cache, S)
    k2, v2 = rt.kv4_read(cache, 9, starts=at, kv_lens=lens, out=(torch.empty(B, Hkv, 9, D, dtype=torch.bfloat16, device="cuda"),) * 2)
    _, l16 = rt.gqa_decode(q, kb, vb, kv_lens=lens)
    rt.kv_weigh(q, kb, l16, weights, kv_lens=lens)
    rt.kv_weigh(q[:, :, None].expand(B, Hq, 3, D).contiguous(), kb, l16[:, :, None].expand(B, Hq, 3).contiguous(), weights, kv_len=50)
    small, pair = rt.Kv4Cache.new(B, Hkv, 30, D), (torch.zeros(B, Hkv, 30, D, dtype=torch.bfloat16, device="cuda"),
                                                  torch.zeros(B, Hkv, 30, D, dtype=torch.bfloat16, device="cuda"))
    evicted = rt.kv_evict(cache, small, weights, 20, recent=3, kv_lens=lens)
    evicted += rt.kv_evict((kb, vb), pair, weights, 25, kv_len=100, weights_out=torch.ones(B, Hkv, 30, device="cuda"))
    return [q, *cache, weights, out, lse, out2, kb, vb, k2, *small, *pair, *evicted]


def test_extension_and_ctypes_paths_agree(rt, monkeypatch):
    from rustorch_b200 import _lib
    got = _every_call(rt)
    monkeypatch.setattr(_lib, "_binding", _Nothing())
    want = _every_call(rt)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
