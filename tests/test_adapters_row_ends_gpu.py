"""GPU tests that btf_adapters writes the N outputs of a row and nothing behind them, where the rows of a tile follow one another
(one adapter for all) and where they do not, for widths that end inside a 16-byte word and rows that are padded to whole ones."""
import pytest
import torch

from test_adapters_gpu import BF16, F16, F32, _check, _inputs, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [5, 150, 700, 1300])
@pytest.mark.parametrize("types", [(F16, F16, F32), (BF16, BF16, BF16), (F32, BF16, F32), (F32, F16, F16)], ids=str)
@pytest.mark.parametrize("N,width", [(1, 8), (17, 24), (19, 20), (19, 24), (61, 64), (61, 96), (129, 136), (131, 136), (132, 136), (33, 40), (887, 888), (250, 264)])
def test_nothing_behind_the_last_output_is_written(cuda, btf, types, N, width, T):
    K, R = 64, 16
    for adapters in (1, 3):
        index = (torch.arange(T, device=cuda) % adapters).int()
        x, (a,), (b,), (z,) = _inputs(cuda, T, adapters, K, R, [N], *types, N + T)
        plan = btf.AdapterPlan(index, adapters)
        for base in (None, torch.full((T, width), 5.0, dtype=types[2], device=cuda)[:, :N].copy_(z), "in place"):
            big = torch.full((T, width), 7.0, dtype=types[2], device=cuda)
            y = big[:, :N]
            if isinstance(base, str):
                base = y.copy_(z)
            want = _reference(x, a, b, None if base is None else z, index, None, None, types[2])
            btf.adapters(x, [btf.AdapterSeg(a, b, y, base)], plan)
            _check(y, want)
            assert bool((big[:, N:] == 7).all())
    assert btf.device_error() == 0


def test_projections_of_one_buffer(cuda, btf):
    """Two projections' outputs beside each other in the rows of one buffer, whose border lies inside a 16-byte word."""
    T, K, R, Ns = 700, 64, 16, [99, 157]
    x, a, b, _ = _inputs(cuda, T, 1, K, R, Ns, BF16, BF16, BF16, 1)
    index = torch.zeros(T, dtype=torch.int32, device=cuda)
    plan = btf.AdapterPlan(index, 1)
    for _ in range(5):
        y = torch.full((T, 256), 7.0, dtype=BF16, device=cuda)
        ys = [y[:, :99], y[:, 99:]]
        btf.adapters(x, [btf.AdapterSeg(*s) for s in zip(a, b, ys)], plan)
        for s in zip(a, b, ys):
            _check(s[2], _reference(x, s[0], s[1], None, index, None, None, BF16))
