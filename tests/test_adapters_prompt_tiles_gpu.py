"""GPU tests of btf_adapters on prompts whose tiles with and without an adapter (rank 0 among them) lie in any order: against
the formula in 64 bits, with the tolerance of test_adapters_gpu.py."""
import pytest
import torch

from test_adapters_gpu import BF16, F16, F32, _check, _inputs, _reference

pytestmark = pytest.mark.gpu


def _ranks(n, R, kind):
    if kind == "pattern":  # four tiles with an adapter two places apart, then one beside the last
        return torch.tensor([R, 0, R, 0, R, 0, R, R], dtype=torch.int32).repeat(n // 8)
    g = torch.Generator().manual_seed(5)
    return torch.where(torch.rand(n, generator=g) < 0.5, 0, R).int()


@pytest.mark.parametrize("kind", ["pattern", "random"])
@pytest.mark.parametrize("types,Ns", [((F32, BF16, F32), [64]), ((BF16, BF16, BF16), [64]), ((F16, F16, F32), [61]),
                                      ((BF16, BF16, BF16), [64, 40, 33])], ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_ranks_of_zero_between_the_tiles(cuda, btf, types, Ns, kind, in_place):
    """1024 adapters of 17 rows, half of them of rank 0, and rows without one: ten or so tiles of one 128-wide piece to a CTA,
    of which any are copied or, in place, passed over."""
    n, K, R = 1024, 64, 24
    T = 17 * n + 100000
    x, a, b, bases = _inputs(cuda, T, n, K, R, Ns, *types, 3)
    index = torch.full((T,), -1, dtype=torch.int32)
    index[torch.randperm(T, generator=torch.Generator().manual_seed(4))[: 17 * n]] = torch.arange(n, dtype=torch.int32).repeat(17)
    index = index.to(cuda)
    ranks = _ranks(n, R, kind).to(cuda)
    plan = btf.AdapterPlan(index, n)
    ys = [z.clone() if in_place else torch.full_like(z, 9.0) for z in bases]
    btf.adapters(x, [btf.AdapterSeg(p, q, y, y if in_place else z) for p, q, y, z in zip(a, b, ys, bases)], plan, ranks=ranks)
    assert btf.device_error() == 0
    for p, q, y, z in zip(a, b, ys, bases):
        _check(y, _reference(x, p, q, z, index, ranks, None, types[2]))
