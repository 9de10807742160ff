"""GPU tests of the operators for many requests at the sizes that they take at most, or near them, against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,HK,D,ragged", [(1500, 8, 4, 64, True), (4099, 3, 1, 72, True), (65535, 2, 1, 16, False), (65535, 2, 1, 16, True)])
def test_prefix_attention_of_many_sequences(cuda, btf, B, H, HK, D, ragged):
    """One node each, over 70 shared rows and up to 9 own ones; of the ragged ones some have no node. The tolerance of
    test_tree_attention_gpu.py: p, eps / 2 of the mean of |v|; the scores (2 D 2^-24 of sums of |q k| that are below 10: less than
    2^-13) and the sums, together less than as much again; the output, eps / 2 and fp16's smallest step."""
    g = torch.Generator(device=cuda).manual_seed(B)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).half()  # noqa: E731
    P, ctx = 70, 10
    q, pk, pv, k, v = rn(B, 1, H, D), rn(P, HK, D), rn(P, HK, D), rn(B, ctx, HK, D), rn(B, ctx, HK, D)
    lens = torch.randint(0, ctx if ragged else 1, (B,), generator=g, device=cuda, dtype=torch.int32)
    counts = torch.randint(0, 2, (B,), generator=g, device=cuda, dtype=torch.int32) if ragged else None
    parents = torch.full((B, 1), -1, dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7.0)
    btf.prefix_attention(q, pk, pv, k, v, lens, parents, counts=counts, out=out)
    assert btf.device_error() == 0
    kj = torch.cat((pk.double().expand(B, P, HK, D), k.double()), 1).repeat_interleave(H // HK, 2)
    vj = torch.cat((pv.double().expand(B, P, HK, D), v.double()), 1).repeat_interleave(H // HK, 2)
    s = torch.einsum("bhd,bjhd->bhj", q[:, 0].double(), kj) * D ** -0.5
    s.masked_fill_((torch.arange(P + ctx, device=cuda) > P + lens[:, None])[:, None], -float("inf"))
    w = s.softmax(-1)
    want, size = torch.einsum("bhj,bjhd->bhd", w, vj), torch.einsum("bhj,bjhd->bhd", w, vj.abs())
    tol = (2.0 ** -10 + 2.0 ** -16) * size + 2.0 ** -11 * want.abs() + 2.0 ** -24
    there = torch.ones(B, dtype=torch.bool, device=cuda) if counts is None else counts > 0
    assert bool(((out[:, 0].double() - want).abs() <= tol)[there].all())
    assert bool((out[~there] == 7).all())


@pytest.mark.parametrize("n", [1, 1024])
def test_adapters_of_the_most_rows(cuda, btf, n):
    from test_adapters_gpu import BF16, F32, _check, _reference

    T, K, R, N = 1 << 20, 32, 8, 24
    g = torch.Generator(device=cuda).manual_seed(n)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x, base = rn(T, K).to(BF16), rn(T, N)
    a, b = (rn(n, R, K) * K ** -0.5).to(BF16), (rn(n, N, R) * 0.3).to(BF16)
    index = torch.randint(-1, n, (T,), generator=g, device=cuda, dtype=torch.int32)
    y = btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], btf.AdapterPlan(index, n))[0]
    assert btf.device_error() == 0
    _check(y, _reference(x, a, b, base, index, None, None, F32))
