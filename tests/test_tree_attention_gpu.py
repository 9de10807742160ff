"""GPU tests of attention for a tree of drafted tokens (btf_tree_attention) against its formula in 64 bits.

Tolerance of an output: with A = sum_j p_j |v_j| and eps that of the type,
  - p is rounded to the type before the product with v: eps / 2 of A; fp16 p below 2^-31 of the largest vanish:
    rows * 2^-31 of max |v|;
  - a score is a sum of D fp32 products, good to D 2^-24 sum |q k| scale (s_abs below), and its exponential to that
    plus 2^-21; numerator and denominator both move: 2 (s_abs + 2^-21) of A; their sums of up to 2^17 terms in
    fp32, pairwise in tiles: 2^-17 of A;
  - the output is rounded to the type: eps / 2 of it."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16]


def chain(n):
    return list(range(-1, n - 1))


def random_tree(rng, n, roots=0.1):
    return [-1 if j == 0 or rng.random() < roots else int(rng.integers(0, j)) for j in range(n)]


def seen(parents, count):
    m = np.zeros((len(parents), len(parents)), bool)
    for i in range(count):
        j = i
        while True:
            m[i, j] = True
            pj = int(parents[j])
            if not 0 <= pj < j:
                break
            j = pj
    return m


def _reference(q, k, v, lens, parents, counts, scale):
    """(out, tolerance without the terms of the type) per sequence, nodes of each only."""
    B, n, H, D = q.shape
    G = H // k.shape[2]
    res = []
    for b in range(B):
        c, L = int(counts[b]), int(lens[b])
        if c == 0:
            res.append(None)
            continue
        mask = torch.from_numpy(np.concatenate([np.ones((n, L), bool), seen(parents[b], c)[:, :c]], 1)[:c])
        kb, vb = (x[b, :L + c].double().repeat_interleave(G, 1) for x in (k, v))
        qb = q[b, :c].double()
        s = torch.einsum("ihd,jhd->hij", qb, kb) * scale
        sa = torch.einsum("ihd,jhd->hij", qb.abs(), kb.abs()).masked_fill(~mask, 0).nan_to_num().amax(-1) * scale
        p = torch.softmax(s.masked_fill(~mask, -torch.inf), -1)
        vb = vb.permute(1, 0, 2)
        o = torch.einsum("hij,hjd->ihd", p, vb)
        res.append((o, torch.einsum("hij,hjd->ihd", p, vb.abs()), sa.t()[..., None] * D * 2.0 ** -24,
                    vb.abs().amax(), L + c))
    return res


def _check(out, ref, t):
    eps = torch.finfo(t).eps / 2
    for b, r in enumerate(ref):
        if r is None:
            continue
        o, A, s, vmax, rows = r
        got = out[b, :o.shape[0]].double().cpu()
        tol = o.abs() * eps + A * (eps + 2 * (s + 2.0 ** -21) + 2.0 ** -17) + rows * 2.0 ** -31 * vmax
        err = (got - o).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()), got.isfinite().all())


def _inputs(B, n, ctx, H, HK, D, t, seed, qs=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, n, H, D, generator=g) * qs).to(t)
    k = (torch.randn(B, ctx, HK, D, generator=g) * 1.5).to(t)
    v = (torch.randn(B, ctx, HK, D, generator=g) + 0.3).to(t)
    return q, k, v


def _run(btf, cuda, q, k, v, lens, parents, counts=None, **kw):
    i = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(cuda)  # noqa: E731
    out = btf.tree_attention(q.to(cuda), k.to(cuda), v.to(cuda), i(lens), i(parents),
                             counts=None if counts is None else i(counts), **kw)
    assert btf.device_error() == 0
    return out


def _case(btf, cuda, B, n, H, HK, D, t, lens, parents, counts=None, ctx=None, seed=0, scale=None):
    ctx = ctx or max(lens) + n
    q, k, v = _inputs(B, n, ctx, H, HK, D, t, seed)
    out = _run(btf, cuda, q, k, v, lens, parents, counts, scale=scale)
    ref = _reference(q, k, v, lens, parents, [n] * B if counts is None else counts, scale or D ** -0.5)
    _check(out, ref, t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("H,HK,D", [(24, 4, 256), (8, 8, 64), (32, 4, 128), (6, 1, 192), (5, 1, 80), (4, 2, 8), (7, 7, 96),
                                    (64, 1, 128), (3, 1, 248)])
@pytest.mark.parametrize("n", [1, 7, 64])
def test_heads_sizes_and_types(cuda, btf, H, HK, D, n, t):
    rng = np.random.default_rng(n + D)
    _case(btf, cuda, 1, n, H, HK, D, t, [100], [random_tree(rng, n)], seed=D)


@pytest.mark.parametrize("length", [0, 1, 2, 31, 56, 62, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 1000, 4095])
@pytest.mark.parametrize("n", [1, 9, 64])
def test_lengths_around_the_tiles(cuda, btf, length, n):
    rng = np.random.default_rng(length)
    _case(btf, cuda, 1, n, 6, 2, 64, torch.float16, [length], [random_tree(rng, n)], seed=length, ctx=length + n + 5)


@pytest.mark.parametrize("parents", [chain(64), [-1] * 64, [-1] + [0] * 63, [-1, 0, 0, 1, 1, 2, 2] + list(range(6, 63)),
                                     [-5, 7, 2, 64, 99, 3] + [4] * 58], ids=["chain", "roots", "star", "mixed", "odd"])
def test_trees(cuda, btf, parents):
    """The deepest and the widest tree, and parents that are no earlier node (they hang on the cache)."""
    for length in (0, 50):
        _case(btf, cuda, 1, 64, 4, 1, 128, torch.bfloat16, [length], [parents], seed=3)


@pytest.mark.parametrize("t", TYPES)
def test_ragged_batch(cuda, btf, t):
    B, n = 9, 13
    rng = np.random.default_rng(5)
    lens, counts = [0, 1, 700, 64, 33, 511, 5, 2000, 128], [13, 1, 0, 5, 13, 2, 12, 7, 1]
    parents = [random_tree(rng, n) for _ in range(B)]
    q, k, v = _inputs(B, n, 2100, 12, 2, 128, t, 4)
    out = torch.full((B, n, 12, 128), 3.0, dtype=t, device=cuda)
    _run(btf, cuda, q, k, v, lens, parents, counts, out=out)
    _check(out, _reference(q, k, v, lens, parents, counts, 128 ** -0.5), t)
    for b in range(B):  # rows of no node stay as they were
        assert bool((out[b, counts[b]:] == 3).all())


@pytest.mark.parametrize("t", TYPES)
def test_long_cache(cuda, btf, t):
    rng = np.random.default_rng(8)
    _case(btf, cuda, 1, 20, 6, 1, 256, t, [40000], [random_tree(rng, 20)], seed=6)
    _case(btf, cuda, 2, 3, 2, 2, 64, t, [40000, 12345], [chain(3), [-1, 0, 0]], seed=7)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 256])
def test_nothing_behind_the_mask_matters(cuda, btf, t, D):
    """Rows behind the last node, and nodes that a node does not see, may hold NaN or infinities."""
    n, L, ctx = 8, 70, 300
    parents = [[-1, 0, 0, 1, 1, 2, 2, -1]]
    q, k, v = _inputs(1, n, ctx, 6, 2, D, t, 9)
    ref = _reference(q, k, v, [L], parents, [n], D ** -0.5)
    for x in (k, v):
        x[:, L + n:] = float("nan")
        x[:, L + n + 7:] = float("inf")
    out = _run(btf, cuda, q, k, v, [L], parents)
    _check(out, ref, t)
    bad = [3, 6]  # leaves: seen by themselves alone
    for kv, val in (("k", float("nan")), ("v", float("nan")), ("v", float("inf")), ("v", -float("inf"))):
        k2, v2 = k.clone(), v.clone()
        {"k": k2, "v": v2}[kv][:, [L + j for j in bad]] = val
        got = _run(btf, cuda, q, k2, v2, [L], parents)
        rest = [i for i in range(n) if i not in bad]
        assert torch.equal(got[:, rest], out[:, rest]), (kv, val)
        if val == val:
            assert bool((got[:, bad] == val).all())
        else:
            assert bool(got[:, bad].isnan().all())
    # in the cache itself everyone sees them
    v[0, 11, 1, 5] = float("inf")
    got = _run(btf, cuda, q, k, v, [L], parents)
    assert bool((got[0, :, 3:, 5] == float("inf")).all()) and bool(got[0, :, :3].isfinite().all())


def test_large_scores(cuda, btf):
    """Scores of hundreds, rising along the cache (the running maximum moves in every tile) and falling."""
    n, L, D = 5, 1000, 128
    q, k, v = _inputs(1, n, L + n, 4, 1, D, torch.bfloat16, 10)
    ramp = torch.linspace(-1, 1, L + n)[None, :, None, None]
    for sign in (1, -1):
        k2 = (q.float().mean((1, 2), keepdim=True) * ramp * sign * 3 + 0.02 * k.float()).to(k.dtype)
        q2 = (q.float().mean((1, 2), keepdim=True) * 4 + 0.05 * q.float()).to(q.dtype)
        parents = [[-1, 0, 1, 1, 0]]
        out = _run(btf, cuda, q2, k2, v, [L], parents, scale=1.0)
        _check(out, _reference(q2, k2, v, [L], parents, [n], 1.0), torch.bfloat16)


def test_scale(cuda, btf):
    for scale in (0.0, -0.3, 0.01):
        q, k, v = _inputs(1, 4, 90, 4, 2, 64, torch.float16, 11)
        out = _run(btf, cuda, q, k, v, [80], [[-1, 0, 1, 0]], scale=scale)
        ref = _reference(q, k, v, [80], [[-1, 0, 1, 0]], [4], scale)
        _check(out, [(o, A, s.abs(), m, r) for o, A, s, m, r in ref], torch.float16)


def test_strides(cuda, btf):
    """Heads outside tokens, a slice of a wider projection, and a cache interleaved with another."""
    t, B, n, H, HK, D, ctx = torch.float16, 2, 6, 8, 2, 64, 150
    q, k, v = _inputs(B, n, ctx, H, HK, D, t, 12)
    lens, parents = [100, 140], [[-1, 0, 0, 1, 2, 2]] * 2
    want = _run(btf, cuda, q, k, v, lens, parents)
    wide = torch.randn(B, n, H, 2 * D).to(t).to(cuda)
    wide[..., :D] = q.to(cuda)
    kv = torch.randn(B, HK, ctx, 2, D).to(t).to(cuda)
    kv[..., 0, :], kv[..., 1, :] = k.to(cuda).transpose(1, 2), v.to(cuda).transpose(1, 2)
    out = torch.zeros(B, H, n, D, dtype=t, device=cuda).transpose(1, 2)
    got = _run(btf, cuda, wide[..., :D], kv[..., 0, :].transpose(1, 2), kv[..., 1, :].transpose(1, 2), lens, parents,
               out=out)
    assert torch.equal(got, want)
    one = _run(btf, cuda, q[:1], k[:1, :, :1], v[:1, :, :1], lens[:1], parents[:1])  # dims of one entry
    _check(one, _reference(q[:1], k[:1, :, :1], v[:1, :, :1], lens[:1], parents[:1], [n], D ** -0.5), t)


def test_lens_are_bounded_by_the_cache(cuda, btf):
    q, k, v = _inputs(3, 4, 64, 2, 1, 64, torch.float16, 13)
    parents = [chain(4)] * 3
    out = _run(btf, cuda, q, k, v, [60, 1000, -7], parents)
    _check(out, _reference(q, k, v, [60, 60, 0], parents, [4] * 3, 0.125), torch.float16)
    out = _run(btf, cuda, q, k, v, [60, 60, 60], parents, counts=[9, -1, 4])  # more than n: n; less than 0: none
    ref = _reference(q, k, v, [60] * 3, parents, [4, 0, 4], 0.125)
    _check(out, ref, torch.float16)
    assert float(out[1].abs().max()) == 0


def test_large_offsets(cuda, btf):
    """The second sequence's cache lies behind 2^31 elements."""
    n, ctx, HK, D, t = 3, 2 ** 21 // 2 + 8, 8, 128, torch.float16
    k, v = (torch.empty(3, ctx, HK, D, dtype=t, device=cuda) for _ in range(2))
    q, ks, vs = _inputs(3, n, 200 + n, 16, HK, D, t, 14)
    k[:, :200 + n], v[:, :200 + n] = ks.to(cuda), vs.to(cuda)
    parents = [chain(n)] * 3
    got = btf.tree_attention(q.to(cuda), k, v, torch.tensor([200] * 3, dtype=torch.int32, device=cuda),
                             torch.tensor(parents, dtype=torch.int32, device=cuda))
    _check(got, _reference(q, ks, vs, [200] * 3, parents, [n] * 3, D ** -0.5), t)


def test_repeatable_streams_and_graph(cuda, btf):
    """The same bits on every call, on two streams at once (a workspace each), and from a graph whose lengths,
    trees and cache change between replays."""
    B, n, H, HK, D, ctx, t = 3, 12, 12, 2, 128, 900, torch.bfloat16
    q, k, v = (x.to(cuda) for x in _inputs(B, n, ctx, H, HK, D, t, 15))
    lens = torch.tensor([800, 3, 411], dtype=torch.int32, device=cuda)
    rng = np.random.default_rng(1)
    parents = torch.tensor([random_tree(rng, n) for _ in range(B)], dtype=torch.int32, device=cuda)
    want = btf.tree_attention(q, k, v, lens, parents)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        got.append([btf.tree_attention(q, k, v, lens, parents, stream=s) for _ in range(4)])
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for calls in got:
        for o in calls:
            assert torch.equal(o, want)
    out, work = torch.zeros_like(q), btf.tree_attention_work(q, k)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for gr in graphs:  # two graphs share one workspace; they run one after the other
        with torch.cuda.graph(gr):
            btf.tree_attention(q, k, v, lens, parents, out=out, work=work)
    for i in range(4):
        lens.copy_(torch.tensor([800 - i, 3 + 64 * i, 411], dtype=torch.int32))
        parents.copy_(torch.tensor([random_tree(rng, n) for _ in range(B)], dtype=torch.int32))
        k.mul_(0.9)
        graphs[i % 2].replay()
        assert torch.equal(out, btf.tree_attention(q, k, v, lens, parents))


def test_refusals(cuda, btf):
    q, k, v = (x.to(cuda) for x in _inputs(2, 4, 40, 4, 2, 64, torch.float16, 16))
    i = torch.zeros(2, dtype=torch.int32, device=cuda)
    par = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    for fn in (lambda: btf.tree_attention(q.float(), k.float(), v.float(), i, par),
               lambda: btf.tree_attention(q, k.bfloat16(), v, i, par), lambda: btf.tree_attention(q, k, v, i.long(), par),
               lambda: btf.tree_attention(q, k, v, i, par[:, :3]), lambda: btf.tree_attention(q, k, v, i[:1], par),
               lambda: btf.tree_attention(q, k[:, :3], v[:, :3], i, par), lambda: btf.tree_attention(q.cpu(), k, v, i, par),
               lambda: btf.tree_attention(q[..., :60], k[..., :60], v[..., :60], i, par),
               lambda: btf.tree_attention(q, k, v, i, par, work=torch.empty(16, dtype=torch.uint8, device=cuda)),
               lambda: btf.tree_attention(q, k, v, i, par, scale=float("nan")),
               lambda: btf.tree_attention(q[:, :, :3], k, v, i, par)):
        with pytest.raises(RuntimeError):
            fn()
    assert btf.tree_attention(q[:0], k[:0], v[:0], i[:0], par[:0]).shape == (0, 4, 4, 64)


@pytest.mark.parametrize("B,n,ctx", [(1, 1, 700), (3, 4, 2100), (40, 2, 600)])
def test_lengths_that_change_from_call_to_call(cuda, btf, B, n, ctx):
    """Calls one after another without a synchronisation, the lengths and counts rewritten in between by a kernel on the
    same stream: each call's outputs are those of a call by itself."""
    H, HK, D = 4, 2, 128
    g = torch.Generator(device=cuda).manual_seed(B)
    q, k, v = (torch.randn(s, generator=g, device=cuda).half() for s in ((B, n, H, D), (B, ctx, HK, D), (B, ctx, HK, D)))
    parents = (torch.arange(n, dtype=torch.int32, device=cuda) - 1).repeat(B, 1)
    calls = 40
    all_lens = torch.randint(0, ctx - n + 1, (calls, B), generator=g, device=cuda).int()
    all_counts = torch.randint(0, n + 1, (calls, B), generator=g, device=cuda).int()
    want = []
    for i in range(calls):
        torch.cuda.synchronize()
        want.append(btf.tree_attention(q, k, v, all_lens[i].clone(), parents, all_counts[i].clone()))
        torch.cuda.synchronize()
    lens, counts = torch.zeros(B, dtype=torch.int32, device=cuda), torch.zeros(B, dtype=torch.int32, device=cuda)
    work = btf.tree_attention_work(q, k)
    got = [torch.zeros_like(q) for _ in range(calls)]
    torch.cuda.synchronize()
    for i in range(calls):
        torch.add(all_lens[i], 0, out=lens)
        torch.add(all_counts[i], 0, out=counts)
        btf.tree_attention(q, k, v, lens, parents, counts, out=got[i], work=work)
    for i in range(calls):
        assert torch.equal(got[i], want[i]), i
    assert btf.device_error() == 0


@pytest.mark.parametrize("lengths", ["equal", "ragged", "short"])
@pytest.mark.parametrize("B,HK,D", [(10, 8, 256), (25, 3, 256), (18, 8, 200), (32, 4, 256), (31, 5, 256), (20, 8, 128), (32, 5, 64),
                                    (32, 8, 128), (33, 1, 128), (33, 8, 72)])
def test_pairs_beside_the_ranges(cuda, btf, B, HK, D, lengths):
    """About half as many, nearly as many and a few more (sequence, kv-head) pairs as the card takes ranges (148 above 128
    dims, 296 below), and more sequences than a warp has lanes."""
    n, rng = 3, np.random.default_rng(B * HK)
    lens = {"equal": [700] * B, "short": [int(x) for x in rng.integers(0, 70, B)],
            "ragged": [int(x) for x in np.exp(rng.uniform(0, np.log(900), B))]}[lengths]
    counts = [n] * B if lengths == "equal" else [int(x) for x in rng.integers(0, n + 1, B)]
    _case(btf, cuda, B, n, 2 * HK, HK, D, torch.float16, lens, [random_tree(rng, n) for _ in range(B)], counts,
          ctx=max(lens) + n + 1, seed=B)
