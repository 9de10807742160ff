"""GPU tests of btf_adapters at the end of fp32's range, against the formula."""
import pytest
import torch

from test_adapters_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [5, 1100])
@pytest.mark.parametrize("w,y_type", [(BF16, F32), (BF16, BF16), (F16, F32)], ids=str)
def test_largest_finite_sums_and_infinities(cuda, btf, w, y_type, T):
    """h up to fp32's largest, which rounds to infinity in bf16, is finite all the same; infinite and NaN rows are so in y."""
    K, R, N = 32, 8, 16
    largest = torch.finfo(F32).max
    x = torch.zeros(T, K, device=cuda)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[4, 0] = largest, -3.4e38, 3.3953e38, float("inf"), float("nan")
    a = torch.zeros(1, R, K, dtype=w, device=cuda)
    a[0, :, 0] = 1.0  # h = x[:, 0], every one of its 8
    b = torch.zeros(1, N, R, dtype=w, device=cuda)
    b[0, :, 0] = 2.0 ** -10
    y = btf.adapters(x, [btf.AdapterSeg(a, b, torch.empty(T, N, dtype=y_type, device=cuda))],
                     btf.AdapterPlan(torch.zeros(T, dtype=torch.int32, device=cuda), 1))[0]
    assert btf.device_error() == 0
    want = x[:, :1].double() * 2.0 ** -10
    # terms of 22 bits or more, or (16-bit y) 16; the output's rounding: half of bf16's eps
    rtol = 2.0 ** -16 + 2.0 ** -8 if y_type == BF16 else 2.0 ** -21
    assert bool(((y[:3].double() - want[:3]).abs() <= rtol * want[:3].abs()).all()), y[:3, 0]
    assert not bool(y[3:5].isfinite().any()) and bool((y[5:] == 0).all())
