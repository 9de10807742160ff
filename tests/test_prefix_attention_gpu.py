"""GPU tests of attention for a batch that shares its first rows (btf_prefix_attention) against its formula in 64 bits:
the formula and the tolerance of the tree attention (test_tree_attention_gpu.py) over the shared and the own rows."""
import numpy as np
import pytest
import torch

from test_tree_attention_gpu import TYPES, _check, _inputs, _reference, chain, random_tree

pytestmark = pytest.mark.gpu


def _shared(P, HK, D, t, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    return ((torch.randn(P, HK, D, generator=g) * 1.5).to(t), (torch.randn(P, HK, D, generator=g) - 0.2).to(t))


def _joined(pk, pv, k, v, P):
    B = k.shape[0]
    return (torch.cat((pk[:P].expand(B, *pk[:P].shape), k), 1), torch.cat((pv[:P].expand(B, *pv[:P].shape), v), 1))


def _run(btf, cuda, q, pk, pv, k, v, lens, parents, counts=None, prefix_len=None, **kw):
    i = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(cuda)  # noqa: E731
    out = btf.prefix_attention(q.to(cuda), pk.to(cuda), pv.to(cuda), k.to(cuda), v.to(cuda), i(lens), i(parents),
                               counts=None if counts is None else i(counts),
                               prefix_len=None if prefix_len is None else i([prefix_len]), **kw)
    assert btf.device_error() == 0
    return out


def _case(btf, cuda, B, n, H, HK, D, t, P, lens, parents=None, counts=None, ctx=None, seed=0, scale=None, prefix_len=None):
    rng = np.random.default_rng(seed)
    parents = [random_tree(rng, n) for _ in range(B)] if parents is None else parents
    q, k, v = _inputs(B, n, ctx or max(lens) + n, H, HK, D, t, seed)
    pk, pv = _shared(P, HK, D, t, seed)
    out = _run(btf, cuda, q, pk, pv, k, v, lens, parents, counts, prefix_len, scale=scale)
    used = P if prefix_len is None else min(max(prefix_len, 0), P)
    kj, vj = _joined(pk, pv, k, v, used)
    _check(out, _reference(q, kj, vj, [used + x for x in lens], parents, [n] * B if counts is None else counts, scale or D ** -0.5), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("H,HK,D", [(24, 4, 256), (8, 8, 64), (32, 4, 128), (6, 1, 192), (5, 1, 80), (4, 2, 8), (7, 7, 96),
                                    (64, 1, 128), (3, 1, 248)])
@pytest.mark.parametrize("B,n", [(1, 1), (3, 7), (40, 1), (5, 64)])
def test_heads_sizes_and_types(cuda, btf, H, HK, D, B, n, t):
    _case(btf, cuda, B, n, H, HK, D, t, 150, [int(x) for x in np.random.default_rng(D).integers(0, 90, B)], seed=D + n)


@pytest.mark.parametrize("P", [0, 1, 2, 31, 63, 64, 65, 127, 128, 129, 1000, 4099])
@pytest.mark.parametrize("lens", [[0, 0], [1, 300], [64, 63]])
def test_lengths_around_the_tiles(cuda, btf, P, lens):
    _case(btf, cuda, 2, 3, 6, 2, 64, torch.float16, P, lens, seed=P, ctx=max(lens) + 9)
    _case(btf, cuda, 2, 1, 4, 1, 192, torch.bfloat16, P, lens, seed=P)


@pytest.mark.parametrize("prefix_len", [-5, 0, 1, 64, 100, 199, 200, 2 ** 30])
def test_length_on_the_device(cuda, btf, prefix_len):
    _case(btf, cuda, 4, 2, 8, 2, 128, torch.bfloat16, 200, [5, 0, 70, 3], prefix_len=prefix_len)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B", [7, 33, 100])
def test_ragged_batch(cuda, btf, t, B):
    """Sequences of unlike lengths and numbers of nodes, none among them: those take no place among the shared rows' M
    tiles, and rows of no node stay as they were."""
    n, H, HK, D, P = 11, 12, 2, 128, 700
    rng = np.random.default_rng(B)
    lens = [int(x) for x in np.exp(rng.uniform(0, 6.5, B)) - 1]
    counts = [int(x) for x in rng.integers(0, n + 1, B)]
    counts[0], counts[-1] = 0, n
    parents = [random_tree(rng, n) for _ in range(B)]
    q, k, v = _inputs(B, n, max(lens) + n, H, HK, D, t, 4)
    pk, pv = _shared(P, HK, D, t, 4)
    out = torch.full((B, n, H, D), 3.0, dtype=t, device=cuda)
    _run(btf, cuda, q, pk, pv, k, v, lens, parents, counts, out=out)
    kj, vj = _joined(pk, pv, k, v, P)
    _check(out, _reference(q, kj, vj, [P + x for x in lens], parents, counts, D ** -0.5), t)
    for b in range(B):
        assert bool((out[b, counts[b]:] == 3).all())
    none = torch.full((B, n, H, D), 3.0, dtype=t, device=cuda)
    _run(btf, cuda, q, pk, pv, k, v, lens, parents, [0] * B, out=none)
    assert bool((none == 3).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_rows_and_long_prefix(cuda, btf, D):
    """Several M tiles, stretches and turns of a CTA."""
    _case(btf, cuda, 30, 5, 12, 2, D, torch.float16, 9000, [int(x) for x in np.random.default_rng(1).integers(0, 40, 30)], seed=1)
    _case(btf, cuda, 300, 2, 8, 4, D, torch.bfloat16, 130, [int(x) for x in np.random.default_rng(2).integers(0, 70, 300)], seed=2)
    _case(btf, cuda, 1, 3, 2, 1, D, torch.bfloat16, 40000, [5], seed=3)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 256])
def test_nothing_behind_a_length_matters(cuda, btf, t, D):
    """Shared rows behind the length, own rows behind the last node and nodes that a node does not see may hold NaN or
    infinities."""
    n, L, ctx, P, rows = 8, 70, 300, 100, 230
    parents = [[-1, 0, 0, 1, 1, 2, 2, -1]]
    q, k, v = _inputs(1, n, ctx, 6, 2, D, t, 9)
    pk, pv = _shared(rows, 2, D, t, 9)
    want = _run(btf, cuda, q, pk, pv, k, v, [L], parents, prefix_len=P)
    k[:, L + n:], v[:, L + n:] = float("nan"), float("inf")
    pk[P:], pv[P:] = float("inf"), float("nan")
    assert torch.equal(_run(btf, cuda, q, pk, pv, k, v, [L], parents, prefix_len=P), want)
    v[0, L + 3], k[0, L + 4] = float("inf"), float("nan")  # nodes 3 and 4: seen by themselves alone
    got = _run(btf, cuda, q, pk, pv, k, v, [L], parents, prefix_len=P)
    others = [i for i in range(n) if i not in (3, 4)]
    assert torch.equal(got[:, others], want[:, others])


def test_no_shared_row_is_tree_attention(cuda, btf):
    B, n, H, HK, D = 5, 6, 8, 2, 96
    rng = np.random.default_rng(3)
    lens, parents = [0, 500, 64, 7, 1200], [random_tree(rng, n) for _ in range(B)]
    q, k, v = _inputs(B, n, 1300, H, HK, D, torch.float16, 3)
    ref = _reference(q, k, v, lens, parents, [n] * B, D ** -0.5)
    pk, pv = _shared(80, HK, D, torch.float16, 3)
    _check(_run(btf, cuda, q, pk[:0], pv[:0], k, v, lens, parents), ref, torch.float16)
    _check(_run(btf, cuda, q, pk, pv, k, v, lens, parents, prefix_len=0), ref, torch.float16)


def test_strides_scale_and_shared_heads(cuda, btf):
    """Views of larger tensors, one kv-head for all, a negative and a zero scale."""
    B, n, H, HK, D, P, ctx = 3, 4, 6, 3, 64, 90, 50
    t = torch.bfloat16
    rng = np.random.default_rng(6)
    parents, lens = [random_tree(rng, n) for _ in range(B)], [7, 0, 40]
    q, k, v = _inputs(B, n, ctx, H, HK, D, t, 6)
    pk, pv = _shared(P, HK, D, t, 6)
    i = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32).to(cuda)  # noqa: E731
    qw = torch.randn(B, H, n, 2 * D, device=cuda).to(t)
    kw, vw = torch.randn(B, HK, ctx, D + 8, device=cuda).to(t), torch.randn(B, HK, ctx, D + 8, device=cuda).to(t)
    pkw, pvw = torch.randn(HK, P + 5, D, device=cuda).to(t), torch.randn(HK, P + 5, D, device=cuda).to(t)
    ow = torch.full((n, B, H, D + 16), 3.0, dtype=t, device=cuda)
    qs, ks, vs = qw[..., D:].transpose(1, 2), kw[..., :D].transpose(1, 2), vw[..., :D].transpose(1, 2)
    pks, pvs, out = pkw[:, 2: 2 + P].transpose(0, 1), pvw[:, 2: 2 + P].transpose(0, 1), ow[..., 8: 8 + D].transpose(0, 1)
    qs.copy_(q), ks.copy_(k), vs.copy_(v), pks.copy_(pk), pvs.copy_(pv)
    for scale in (0.2, -0.2, 0.0):
        btf.prefix_attention(qs, pks, pvs, ks, vs, i(lens), i(parents), scale=scale, out=out)
        kj, vj = _joined(pk, pv, k, v, P)
        ref = _reference(q if scale >= 0 else -q, kj, vj, [P + x for x in lens], parents, [n] * B, abs(scale))
        _check(out, ref, t)
    assert bool((ow[..., :8] == 3).all()) and bool((ow[..., 8 + D:] == 3).all())
    one = pk[:, :1].to(cuda).expand(P, HK, D)
    onev = pv[:, :1].to(cuda).expand(P, HK, D)
    got = btf.prefix_attention(qs, one, onev, ks, vs, i(lens), i(parents))
    kj, vj = _joined(pk[:, :1].expand(P, HK, D), pv[:, :1].expand(P, HK, D), k, v, P)
    _check(got, _reference(q, kj, vj, [P + x for x in lens], parents, [n] * B, D ** -0.5), t)


def test_graph_workspace_and_streams(cuda, btf):
    """One captured call serves a growing batch; a workspace full of NaN; the same bits again and on another stream."""
    B, n, H, HK, D, P, ctx = 6, 1, 8, 2, 128, 300, 80
    t = torch.float16
    q, k, v = _inputs(B, n, ctx, H, HK, D, t, 2)
    pk, pv = _shared(P, HK, D, t, 2)
    dq, dk, dv, dpk, dpv = (x.to(cuda) for x in (q, k, v, pk, pv))
    lens, plen = torch.zeros(B, dtype=torch.int32, device=cuda), torch.full((1,), P, dtype=torch.int32, device=cuda)
    parents = torch.full((B, n), -1, dtype=torch.int32, device=cuda)
    out = torch.empty_like(dq)
    work = btf.prefix_attention_work(dq, dpk, dk)
    work.fill_(255)
    call = lambda o=out, **kw: btf.prefix_attention(dq, dpk, dpv, dk, dv, lens, parents, prefix_len=plen, out=o, **kw)  # noqa: E731
    call(work=work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(work=work)
    for length, shared in ((0, P), (13, P), (79, 65), (40, 0)):
        lens.fill_(length), plen.fill_(shared)
        graph.replay()
        torch.cuda.synchronize()
        kj, vj = _joined(pk, pv, k, v, shared)
        _check(out, _reference(q, kj, vj, [shared + length] * B, [[-1]] * B, [n] * B, D ** -0.5), t)
        again = call(torch.empty_like(out))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        other = call(torch.empty_like(out), stream=s)
        s.synchronize()
        assert torch.equal(again, out) and torch.equal(other, out)


def test_refusals(cuda, btf):
    B, n, H, HK, D, P, ctx = 2, 3, 4, 2, 64, 40, 30
    t = torch.float16
    q, k, v = (x.to(cuda) for x in _inputs(B, n, ctx, H, HK, D, t, 2))
    pk, pv = (x.to(cuda) for x in _shared(P, HK, D, t, 2))
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    parents = torch.tensor([chain(n)] * B, dtype=torch.int32, device=cuda)
    f = btf.prefix_attention
    for call in (
        lambda: f(q, pk[None], pv[None], k, v, lens, parents),
        lambda: f(q, pk[:, :1], pv[:, :1], k, v, lens, parents),
        lambda: f(q, pk, pv[:-1], k, v, lens, parents),
        lambda: f(q, pk.bfloat16(), pv.bfloat16(), k, v, lens, parents),
        lambda: f(q, pk.cpu(), pv.cpu(), k, v, lens, parents),
        lambda: f(q, pk, pv.transpose(0, 1).contiguous().transpose(0, 1), k, v, lens, parents),
        lambda: f(q, pk, pv, k, v, lens, parents, prefix_len=torch.tensor([4], device=cuda)),
        lambda: f(q, pk, pv, k, v, lens, parents, prefix_len=torch.tensor([4, 4], dtype=torch.int32, device=cuda)),
        lambda: f(q, pk, pv, k, v, lens, None),
        lambda: f(q, pk, pv, k, v, None, parents),
        lambda: f(q.float(), pk.float(), pv.float(), k.float(), v.float(), lens, parents),
        lambda: f(q, pk, pv, k, v, lens, parents, work=torch.empty(256, dtype=torch.uint8, device=cuda)),
        lambda: f(q, pk, pv, k, v, lens, parents, out=torch.empty_like(q)[:, :, :1].expand_as(q)),
        lambda: f(q, pk.clone().requires_grad_(), pv, k, v, lens, parents),
    ):
        with pytest.raises(RuntimeError):
            call()
