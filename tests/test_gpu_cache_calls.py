"""Calls of the 4-bit cache and of eviction next to the edges of what their documentation allows, against forms in 64 bits."""
import math

import pytest

from tests import kv4_plain as plain
from tests.test_gpu_kv4 import _check, _decode_case

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


# ------------------------------------------------------------------------------------------------ decode


# 8192 tokens are taken in one launch of clusters; 20,000 are cut into runs for the workers
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


# Below, what runs in one launch of clusters at the sizes of tests/test_gpu_kv4.py is run where the workers take it: more than
# 16,384 rows of cache, or more (sequence, KV head) pairs than SMs, and several steps a worker.
@pytest.mark.parametrize("B,S", [(80, 3000), (1, 60000)])
@pytest.mark.parametrize("what", ["far scores", "growing scores", "falling scores", "one token", "large q", "small q", "tiny v", "huge v",
                                  "mixed v", "growing v", "scale"])
def test_decode_of_wide_ranges_in_runs(rt, what, B, S):
    Hq, Hkv, D = 8, 2, 128
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = (torch.randn(B, Hkv, S, D, device="cuda", generator=g) for _ in "kv")
    along = torch.arange(S, device="cuda")[:, None] / S
    q, scale = _randn(B, Hq, D, seed=9), None
    if what == "far scores":
        k = k * 30
    elif what == "growing scores":
        k = k * (40 * along)
    elif what == "falling scores":
        k = k * (40 - 40 * along)
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
    elif what == "growing v":
        v = v * torch.exp2(18 * along - 6)
    else:
        scale = 0.7
    cache = rt.Kv4Cache(*plain.quantise(k.bfloat16()), *plain.quantise(v.bfloat16()))
    _decode_case(rt, B, Hq, Hkv, D, S, tuple(S - 31 * b for b in range(B)), scale=scale, q=q, cache=cache)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [8191, 8192, 8193, 16383, 16384, 16385])
@pytest.mark.parametrize("B", [1, 9])
def test_decode_on_both_sides_of_the_longest_cluster(rt, B, n, D):
    """Weighed and not, as many rows of cache as tokens, then fewer tokens than the cache has room for.  Weights can change how
    a sequence is cut, so that each call is held against 64 bits and not against the other."""
    for Hq, lens in ((8, (n,) * B), (16, tuple(n - 900 * b - 1 for b in range(B)))):
        cache, q = plain.fill(rt, B, 2, n, D, n), _randn(B, Hq, D, seed=n + 50)
        o, l, w, ot, lt, wt = plain.decode(q, cache, lens)
        for weights in (None, torch.zeros(B, 2, n, device="cuda")):
            kw = dict(kv_len=n) if lens[-1] == n else dict(kv_lens=_i32(*lens))
            out, lse = rt.kv4_decode(q, cache, weights=weights, **kw)
            _check(out, o, ot, "out")
            _check(lse, l, lt, "lse")
        _check(weights, w, wt + 2 * plain.U_F32 * (1 + w), "weights")


@pytest.mark.parametrize("B,Hq,Hkv,D,S", [(18, 32, 8, 128, 1000), (18, 16, 8, 64, 2000), (148, 8, 1, 128, 4096), (74, 4, 2, 64, 4097)])
def test_decode_of_as_many_clusters_as_fit(rt, B, Hq, Hkv, D, S):
    """Clusters of two CTAs, two CTAs an SM."""
    lens = tuple(S - (53 * b) % S for b in range(B))
    cache, q = plain.fill(rt, B, Hkv, S, D, 13), _randn(B, Hq, D, seed=14)
    o, l, w, ot, lt, wt = plain.decode(q, cache, lens)
    for weights in (None, torch.zeros(B, Hkv, S, device="cuda")):
        out, lse = rt.kv4_decode(q, cache, kv_lens=_i32(*lens), weights=weights)
        _check(out, o, ot, "out")
        _check(lse, l, lt, "lse")
    _check(weights, w, wt + 2 * plain.U_F32 * (1 + w), "weights")


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 8), (128, 32, 8), (256, 8, 1)])
def test_decode_of_a_cache_much_larger_than_its_sequences(rt, D, Hq, Hkv):
    _decode_case(rt, 3, Hq, Hkv, D, 131072, (1000, 33, 257), seed=3)


@pytest.mark.parametrize("S", [6000, 6001])
def test_decode_weights_of_more_tokens_than_a_wave_of_ctas(rt, S):
    """Weights of 640 (sequence, KV head) pairs: threads that walk over several pieces; rows of weights on 16 bytes and not."""
    B, Hq, Hkv, D = 160, 8, 4, 64
    lens = tuple((S - 43 * b) % (S + 1) for b in range(B))
    cache, q, weights = plain.fill(rt, B, Hkv, S, D, 3), _randn(B, Hq, D, seed=4), torch.zeros(B, Hkv, S, device="cuda")
    out, lse = rt.kv4_decode(q, cache, kv_lens=_i32(*lens), weights=weights)
    o, l, w, ot, lt, wt = plain.decode(q, cache, lens)
    _check(out, o, ot, "out")
    _check(lse, l, lt, "lse")
    _check(weights, w, wt + 2 * plain.U_F32 * (1 + w), "weights")


def test_decode_in_runs_does_not_read_rows_behind_the_length(rt):
    lens = tuple(100 + 23 * b for b in range(80))
    cache, q = plain.fill(rt, 80, 2, 2000, 128, 5), _randn(80, 8, 128, seed=6)
    want = rt.kv4_decode(q, cache, kv_lens=_i32(*lens))
    for b, n in enumerate(lens):
        cache[1][b, :, n:], cache[3][b, :, n:] = math.nan, math.inf
    got = rt.kv4_decode(q, cache, kv_lens=_i32(*lens))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("B,S", [(80, 3000), (2, 20001)])
def test_decode_in_runs_keeps_to_its_workspace(rt, B, S):
    """Scratch of exactly the size that is asked for, full of ones: the bytes around it stay."""
    Hq, Hkv, D = 8, 2, 64
    lens = tuple(S - 61 * b for b in range(B))
    cache, q = plain.fill(rt, B, Hkv, S, D, 3), _randn(B, Hq, D, seed=4)
    for weighed in (False, True):
        weights = torch.zeros(B, Hkv, S, device="cuda") if weighed else None
        need = rt.kv4_workspace_bytes(B, Hq, Hkv, D, S, weighed)
        assert need > 0
        room = torch.full((need + 4096,), 255, dtype=torch.uint8, device="cuda")
        out, lse = torch.full_like(q, math.nan), torch.full((B, Hq), math.nan, device="cuda")
        rt.kv4_decode(q, cache, kv_lens=_i32(*lens), weights=weights, workspace=room[2048:2048 + need], out=out, lse=lse)
        assert (room[:2048] == 255).all() and (room[2048 + need:] == 255).all()
        o, l, w, ot, lt, wt = plain.decode(q, cache, lens)
        _check(out, o, ot, "out")
        _check(lse, l, lt, "lse")
        if weighed:
            _check(weights, w, wt + 2 * plain.U_F32 * (1 + w), "weights")


@pytest.mark.parametrize("B,S", [(80, 3000), (2, 20001)])
def test_decode_in_runs_on_streams_and_in_graphs(rt, B, S):
    """Two streams at once, and two graphs that share a pool, replayed with lengths that change: decode, merge and weights."""
    Hq, Hkv, D = 8, 2, 128
    caches = [plain.fill(rt, B, Hkv, S, D, s) for s in (1, 2)]
    qs = [_randn(B, Hq, D, seed=s) for s in (3, 4)]
    lens = [_i32(*(S - 7 * b for b in range(B))), _i32(*(5 + 13 * b for b in range(B)))]

    def call(i, **kw):
        w = torch.zeros(B, Hkv, S, device="cuda")
        return *rt.kv4_decode(qs[i], caches[i], kv_lens=lens[i], weights=w, **kw), w
    want = [call(i) for i in (0, 1)]
    for i in (0, 1):
        o, l, w, ot, lt, wt = plain.decode(qs[i], caches[i], lens[i].tolist())
        for got, ref, tol, what in zip(want[i], (o, l, w), (ot, lt, wt + 2 * plain.U_F32 * (1 + w)), ("out", "lse", "weights")):
            _check(got, ref, tol, what)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in "ab"], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = call(i)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(call(i))
        graphs.append(graph)
    for swap in (False, True):
        if swap:
            a = lens[0].clone()
            lens[0].copy_(lens[1])
            lens[1].copy_(a)
        for i in (0, 1):
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], call(i)))


def test_read_into_tensors_of_the_caller(rt):
    cache = plain.fill(rt, 2, 3, 50, 128, 9)
    want = rt.kv4_read(cache, 20, start=7, kv_lens=_i32(50, 12))
    out = tuple(torch.full((2, 3, 20, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    got = rt.kv4_read(cache, 20, start=7, kv_lens=_i32(50, 12), out=out)
    assert got[0] is out[0] and got[1] is out[1]
    for g, w, i in zip(got, want, (0, 2)):
        rows = plain.values(cache[i], cache[i + 1], torch.float32).bfloat16()[:, :, 7:27]
        assert torch.equal(g, w) and torch.equal(g[0], rows[0]) and torch.equal(g[1, :, :5], rows[1, :, :5]) and not g[1, :, 5:].any()


# ------------------------------------------------------------------------------------------------ weights


@pytest.mark.parametrize("T,D", [(1, 64), (1, 128), (1, 256), (5, 64), (3, 128), (5, 256), (5, 128), (7, 256), (40, 64), (40, 128), (64, 256), (150, 128)])
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


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("B,Hkv,D,S", [(64, 8, 128, 3000), (70, 8, 64, 4000), (64, 8, 256, 1000), (1, 8, 128, 131072)])
def test_weigh_of_more_tokens_than_a_wave_of_ctas(rt, B, Hkv, D, S, T):
    """CTAs that walk over several pieces of a sequence, and ones that find none."""
    G, lens = 2, tuple((S - 37 * b) % S + 1 for b in range(B))
    q, k = _randn(B, G * Hkv, T, D, seed=1), _randn(B, Hkv, S, D, seed=2)
    lse = 6 + torch.rand(B, G * Hkv, T, device="cuda")
    w = torch.zeros(B, Hkv, S, device="cuda")
    if T == 1:
        rt.kv_weigh(q[:, :, 0], k, lse[:, :, 0], w, kv_lens=_i32(*lens))
    else:
        rt.kv_weigh(q, k, lse, w, kv_lens=_i32(*lens))
    for b in range(B):
        want, tol = plain.weigh(q[b:b + 1], k[b:b + 1], lse[b:b + 1], lens[b:b + 1])
        assert ((w[b].double() - want[0]).abs() <= tol[0] + 2 * plain.U_F32 * (1 + want[0])).all(), b


# 296 CTAs at most (148 at D = 256) share the tiles of 128 tokens: here the longest sequences have 4 to 10 for each.  1, 4, 5 and
# 17 blocks of 64 query rows; sequences shorter than their queries, and tiles in which the last queries hide tokens.
@pytest.mark.parametrize("B,Hq,Hkv,T,D,S,lens", [
    (8, 64, 8, 8, 128, 3000, (3000, 1, 127, 128, 129, 2000, 385, 2999)),
    (8, 32, 8, 64, 64, 3000, (3000, 1500, 63, 2900, 129, 2000, 2561, 2999)),
    (8, 32, 8, 80, 128, 3000, (79, 2560, 3000, 2900, 2561, 2000, 2816, 2999)),
    (4, 16, 8, 160, 256, 5000, (5000, 159, 4001, 2048)),
    (2, 8, 1, 136, 256, 40000, (40000, 33333)),
    (1, 16, 2, 136, 64, 100000, (99999,)),
])
def test_weigh_of_many_tiles_a_cta(rt, B, Hq, Hkv, T, D, S, lens):
    q, k = _randn(B, Hq, T, D, seed=1), _randn(B, Hkv, S, D, seed=2)
    lse = torch.full((B, Hq, T), 7.5, device="cuda") + torch.rand(B, Hq, T, device="cuda")
    before = torch.rand(B, Hkv, S, device="cuda")
    w = before.clone()
    rt.kv_weigh(q, k, lse, w, kv_lens=_i32(*lens))
    for b in range(B):  # a sequence at a time: the scores of all in 64 bits would not fit
        want, tol = plain.weigh(q[b:b + 1], k[b:b + 1], lse[b:b + 1], lens[b:b + 1])
        off = (w[b].double() - before[b].double() - want[0]).abs()
        assert (off <= tol[0] + 2 * plain.U_F32 * (1 + want[0])).all(), (b, off.max().item())
        assert torch.equal(w[b, :, lens[b]:], before[b, :, lens[b]:])
    from rustorch_b200 import _lib
    assert _lib.device_status() == 0


# ------------------------------------------------------------------------------------------------ eviction


@pytest.mark.parametrize("B,Hkv,S,keep,recent", [
    (1, 1, 300_000, 20_000, 100),   # runs of 37,500 in clusters of 8: more than a CTA's shared memory holds
    (10, 8, 40_000, 3000, 64),      # a CTA each, of up to 39,936 candidates
    (37, 2, 9000, 500, 7),          # clusters of 2
    (37, 1, 9000, 8000, 0),         # clusters of 4
    (9, 2, 40_000, 39_000, 38_000)  # clusters of 8, nearly all kept
])
def test_evict_of_long_runs(rt, B, Hkv, S, keep, recent):
    """Runs that do not fit shared memory beside short ones, and every size of cluster; a third of the weights are equal."""
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn(B, Hkv, S, device="cuda", generator=g)
    w = torch.where(torch.rand(B, Hkv, S, device="cuda", generator=g) < 0.3, 0.25, w)
    cache = tuple(torch.randint(-9, 9, (B, Hkv, S, 8), device="cuda", generator=g).bfloat16() for _ in "kv")
    lens = [S if b % 2 == 0 else max(1, keep // 2 if b % 4 == 1 else S - 17 * b) for b in range(B)]
    out = tuple(torch.full((B, Hkv, keep + 5, 8), 99.0, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    new_lens, w_out, kept = rt.kv_evict(cache, out, w, keep, recent=recent, kv_lens=_i32(*lens))
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    for b, n in enumerate(lens):
        m = min(n, keep)
        at = torch.arange(m, device="cuda").expand(Hkv, m)
        if n > keep:
            heavy = w[b, :, :n - recent].sort(dim=-1, descending=True, stable=True)[1][:, :keep - recent]
            at = torch.cat([heavy, torch.arange(n - recent, n, device="cuda").expand(Hkv, recent)], -1).sort(-1)[0]
        assert torch.equal(kept[b, :, :m].long(), at) and (kept[b, :, m:] == -1).all()
        assert torch.equal(w_out[b, :, :m], w[b].gather(1, at)) and not w_out[b, :, m:].any()
        for o, c in zip(out, cache):
            assert torch.equal(o[b, :, :m], c[b].gather(1, at[..., None].expand(Hkv, m, 8))) and (o[b, :, m:] == 99).all()
