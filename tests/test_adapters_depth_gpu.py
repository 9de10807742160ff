"""Long sums of btf_adapters against 64 bits, with tolerances that grow like the error of sums of random signs (those of
test_adapters_gpu.py bound every order and sign, and beyond a few thousand elements leave room for mistakes).

With U = 2^-24, Q = root of sum_k (a x)^2 and E = root of sum_r (h b)^2, the sizes that sums of random signs have; a tensor-core sum
loses up to 2 U of its size, towards 0, in every MMA; 6 standard deviations of the rest:
  - h of an fp32 x: sums over 32 of K, 6 MMAs (8 of two tf32 terms): 16 U of Q and of |h|; K / 32 fp32 additions, each off by U / sqrt 3 of a
    running sum of 0.6 Q or so: 2 sqrt(K / 32) U of Q; two tf32 terms: 2^-21 of an element at most, 6 / sqrt 3 of that: 28 U of Q;
  - h of a 16-bit x: K / 16 MMAs, U of Q and |h| in each on average;
  - h's terms: 4 x 2^-24 (three bf16), 2^-22 (two fp16), 2^-17 (two bf16) of E, and 2^-39 of the row's largest h (fp16);
  - the sum over the rank: R / 16 + 1 MMAs of each of 2 or 3 terms, 2 U of E and of |B h|;
  - scale, base and output as in test_adapters_gpu.py."""
import pytest
import torch

from test_adapters_gpu import BF16, F16, F32, U, _index, _inputs

TYPES = [(F32, BF16, F32), (F32, F16, F32), (BF16, BF16, F32), (F16, F16, F32), (BF16, BF16, BF16), (F32, F16, F16)]


def _reference(x, a, b, base, index, scales, types):
    """(value, tolerance) in 64 bits of one projection."""
    T, K = x.shape
    n, N, R = b.shape
    half, x32 = types[1] == F16, types[0] == F32
    terms = 3 if not half and types[2] == F32 else 2
    split = 2.0 ** -22 if half else 2.0 ** -24 if terms == 3 else 2.0 ** -17
    y = torch.zeros(T, N, dtype=torch.float64, device=x.device) if base is None else base.double()
    tol = 4 * U * y.abs()
    for j in range(n):
        rows = (index == j).nonzero()[:, 0]
        if not rows.numel():
            continue
        xs, A, B, s = x[rows].double(), a[j].double(), b[j].double(), 1.0 if scales is None else float(scales[j])
        h, Q = xs @ A.T, (xs.square() @ A.square().T).sqrt()
        if x32:
            of_q, of_h = 2 * (K / 32) ** 0.5 + 16 + 28 * half, 16
        else:
            of_q = of_h = K / 16
        E, d = (h.square() @ B.square().T).sqrt(), h @ B.T
        t = ((of_q * U * Q).square() @ B.square().T).sqrt() + of_h * U * (d.abs() + E) + 4 * split * E
        t += 2 * U * terms * (R / 16 + 1) * (E + d.abs())
        if half:
            t += 2.0 ** -39 * h.abs().amax(1, keepdim=True) * B.square().sum(1).sqrt()
        y[rows] += d * s
        tol[rows] += (t + 4 * U * d.abs()) * abs(s)
    tol += 4 * U * y.abs() + (torch.finfo(types[2]).eps / 2 * y.abs() if types[2] != F32 else 0)
    return y, tol + (2.0 ** -25 if types[2] == F16 else 0)


@pytest.mark.parametrize("K", [5120, 17408])
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_the_tolerance_finds_mistakes(types, K):
    """On the CPU: 32 of K left out, and an fp32 x cut to one bf16 term (or one of tf32's size), are beyond it almost
    everywhere that there is a delta larger than the output's rounding."""
    torch.manual_seed(K)
    T, R, N = 24, 48, 72
    x, a, b = torch.randn(T, K).to(types[0]), (torch.randn(1, R, K) * K ** -0.5).to(types[1]), (torch.randn(1, N, R) * 0.3).to(types[1])
    index = torch.zeros(T, dtype=torch.int32)
    y, tol = _reference(x, a, b, None, index, None, types)
    mistakes = [x.clone().index_fill_(1, torch.arange(64, 96), 0)]
    if types[0] == F32:
        mistakes += [x.bfloat16().float(), (x.view(torch.int32) & -0x2000).view(torch.float32)] if types[2] == F32 else [x.bfloat16().float()]
    for wrong in mistakes:
        z, _ = _reference(wrong, a, b, None, index, None, types)
        part = 0.9 if types[2] == F32 or wrong is mistakes[0] else 0.05
        assert float(((z - y).abs() > tol).double().mean()) > part


@pytest.mark.gpu
@pytest.mark.parametrize("T", [9, 300, 1024, 6007])
@pytest.mark.parametrize("K", [5120, 17408])
@pytest.mark.parametrize("types", TYPES, ids=str)
def test_long_sums(cuda, btf, types, K, T):
    n, R, N = 2, 48, 72
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], *types, K + T)
    index, scales = _index(cuda, T, n, T), torch.tensor([1.5, -0.75], device=cuda)
    y = btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], btf.AdapterPlan(index, n), scales=scales)[0]
    want, tol = _reference(x, a, b, base, index, scales, types)
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 48, 1024, 1025, 6007])
@pytest.mark.parametrize("K", [512, 5120, 17408])
@pytest.mark.parametrize("w", [BF16, F16], ids=str)
def test_fp32_rows_are_served_to_fp32(cuda, btf, w, K, T):
    """Root mean square of the error at most 16 U of y's: about U for each of the 2 MMAs of a 32 of K's first terms and of the
    5 of the rank's, 5 for K / 32 additions, 4 for the terms' bits."""
    x, (a,), (b,), _ = _inputs(cuda, T, 1, K, 64, [256], F32, w, F32, K + T)
    index = torch.zeros(T, dtype=torch.int32, device=cuda)
    y = btf.adapters(x, [btf.AdapterSeg(a, b)], btf.AdapterPlan(index, 1))[0]
    want = x.double() @ a[0].double().T @ b[0].double().T
    assert float((y - want).square().mean().sqrt() / want.square().mean().sqrt()) <= 16 * U
