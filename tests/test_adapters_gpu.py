"""GPU tests of low-rank adapters of many requests (btf_adapters, btf_adapter_plan) against their formula in 64 bits.

Tolerance of an output, with U = 2^-24, h = A x and sums of magnitudes S = sum_k |a x|, D = sum_r |h| |b|:
  - h is a sum of K fp32 products in whatever order, on tensor cores that may cut off instead of rounding:
    (K + 64) U of S; an fp32 x enters with at least 22 bits (2^-21 covers the two roundings of its terms): 2^-21 of S;
  - h's terms: 24 bits (bf16 weights, fp32 y), 22 bits and 2^-39 of the row's largest (fp16 weights), or 16 bits
    (bf16 weights and y: two roundings to 2^-9 of what is left, 2^-18, doubled): of D;
  - the sum over the rank: (R + 64) U of D; scale, base and the output's own rounding: 4 U of |delta| + |base|, eps / 2 of
    the output (and half of fp16's smallest step)."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
TYPES = [(F32, F16, F32), (F32, BF16, F32), (F32, BF16, BF16), (F32, F16, F16), (F16, F16, F16), (F16, F16, F32),
         (BF16, BF16, BF16), (BF16, BF16, F32)]


def _inputs(cuda, T, n, K, R, Ns, x_type, w_type, y_type, seed, base=True):
    g = torch.Generator(device=cuda).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    x = rn(T, K).to(x_type)
    a = [(rn(n, R, K) * K ** -0.5).to(w_type) for _ in Ns]
    b = [(rn(n, N, R) * 0.3).to(w_type) for N in Ns]
    bases = [rn(T, N).to(y_type) if base else None for N in Ns]
    return x, a, b, bases


def _reference(x, a, b, base, index, ranks, scales, y_type):
    """(value, tolerance) in 64 bits of one projection."""
    T, K = x.shape
    n, N, R = b.shape
    y = torch.zeros(T, N, dtype=torch.float64, device=x.device) if base is None else base.double()
    tol = torch.zeros_like(y)
    half = a.dtype == F16
    for j in range(n):
        rows = (index == j).nonzero()[:, 0]
        r = R if ranks is None else min(max(int(ranks[j]), 0), R)
        if not rows.numel() or not r:
            continue
        xs, A, B = x[rows].double(), a[j, :r].double(), b[j, :, :r].double()
        s = 1.0 if scales is None else float(scales[j])
        h, S = xs @ A.T, xs.abs() @ A.abs().T
        eh = ((K + 64) * U + 2.0 ** -21) * S
        split = 2.0 ** -22 if half else 2.0 ** -24 if y_type == F32 else 2.0 ** -17
        D = h.abs() @ B.abs().T
        d = h @ B.T * s
        t = eh @ B.abs().T + D * (split + (R + 64) * U)
        if half:
            t = t + 2.0 ** -39 * h.abs().amax(1, keepdim=True) * B.abs().sum(1)
        y[rows] += d
        tol[rows] = t * abs(s) + 4 * U * d.abs()
    tol += 4 * U * y.abs() + (torch.finfo(y_type).eps / 2 * y.abs() if y_type != F32 else 0)
    if base is not None:
        tol += 4 * U * base.double().abs()
    return y, tol + (2.0 ** -25 if y_type == F16 else 0)


def _check(y, ref):
    want, tol = ref
    err = (y.double() - want).abs()
    assert bool((err <= tol + 1e-30).all()), (float((err / (tol + 1e-30)).max()), y.isfinite().all())


def _index(cuda, T, n, seed, none=0.1):
    g = torch.Generator().manual_seed(seed)
    i = torch.randint(0, n, (T,), generator=g, dtype=torch.int32)
    i[torch.rand(T, generator=g) < none] = -1
    return i.to(cuda)


def _case(btf, cuda, T, n, K, R, Ns, types, seed=0, base=True, ranks="mixed", index=None, scaled=True):
    x, a, b, bases = _inputs(cuda, T, n, K, R, Ns, *types, seed, base)
    index = _index(cuda, T, n, seed) if index is None else index
    g = torch.Generator().manual_seed(seed + 1)
    ranks = torch.randint(0, R + 1, (n,), generator=g, dtype=torch.int32).to(cuda) if ranks == "mixed" else ranks
    scales = (torch.rand(n, generator=g) * 3 - 1).to(cuda) if scaled else None
    plan = btf.AdapterPlan(index, n)
    out = btf.adapters(x, [btf.AdapterSeg(p, q, torch.full((T, N), 9.0, dtype=types[2], device=cuda), z)
                           for p, q, N, z in zip(a, b, Ns, bases)], plan, ranks=ranks, scales=scales)
    assert btf.device_error() == 0
    for y, p, q, z in zip(out, a, b, bases):
        _check(y, _reference(x, p, q, z, index, ranks, scales, types[2]))


# ---------------------------------------------------------------- the plan
@pytest.mark.parametrize("T,n", [(1, 1), (5, 3), (31, 2), (32, 40), (33, 1), (257, 9), (1000, 1024), (5000, 7), (70001, 300)])
def test_plan_sorts_the_rows(cuda, btf, T, n):
    index = _index(cuda, T, n, T, none=0.2)
    index[:: 7] = n + 5  # no adapter either
    plan = btf.AdapterPlan(index, n)
    words = plan.plan.view(torch.int32).cpu()
    key = torch.where((index < 0) | (index >= n), n, index).cpu()
    order = words[8: 8 + T].long()
    assert torch.equal(order, torch.sort(key, stable=True).indices)
    assert torch.equal(words[8 + T: 8 + 2 * T], key[order])
    assert words[:2].tolist() == [T, n] and int(words[4]) == int((key < n).sum())
    small = (32 + 8 * T + 15) // 16 * 4
    lists = min(n + 1, T) + 1
    for word, size, width, first in ((2, 16, 20, small), (3, 128, 4, small + 20 * (T // 16 + lists))):
        tiles = words[first: first + width * int(words[word])].view(-1, width)
        want, at = [], 0
        for j, c in enumerate(torch.bincount(key, minlength=n + 1).tolist()):
            want += [[j if j < n else -1, at + i, min(size, c - i)] for i in range(0, c, size)]
            at += c
        assert tiles[:, :3].tolist() == want
        if size == 16:  # with their rows
            assert all(t[4: 4 + t[2]] == order[t[1]: t[1] + t[2]].tolist() for t in tiles.tolist())


# ---------------------------------------------------------------- the call
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("T", [1, 7, 300, 1100])
def test_types(cuda, btf, types, T):
    _case(btf, cuda, T, 3, 264, 64, [200], types, seed=T)


@pytest.mark.parametrize("types", [(F32, BF16, F32), (F16, F16, F16)], ids=str)
@pytest.mark.parametrize("R", [8, 16, 24, 32, 40, 64, 72, 96, 128])
def test_ranks(cuda, btf, R, types):
    for T in (20, 1100):
        _case(btf, cuda, T, 5, 512, R, [96, 33], types, seed=R)
        _case(btf, cuda, T, 5, 512, R, [96], types, seed=R, ranks=None, scaled=False)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 385, 511, 512, 513, 1024, 1025, 2111])
def test_rows(cuda, btf, T):
    _case(btf, cuda, T, 4, 128, 16, [64, 8, 129], (F32, F16, F32), seed=T)
    _case(btf, cuda, T, 1, 128, 16, [64], (BF16, BF16, BF16), seed=T, base=False, index=torch.zeros(T, dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("K", [8, 16, 24, 32, 40, 1000, 5120, 17408])
def test_depths(cuda, btf, K):
    _case(btf, cuda, 9, 2, K, 32, [72], (F32, BF16, F32), seed=K)
    _case(btf, cuda, 600, 2, K, 32, [72], (BF16, BF16, BF16), seed=K)
    _case(btf, cuda, 300, 2, K, 48, [72], (F16, F16, F32), seed=K)
    _case(btf, cuda, 1100, 2, K, 48, [72], (F32, F16, F32), seed=K)


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 257, 1000])
def test_widths(cuda, btf, N):
    _case(btf, cuda, 6, 2, 64, 24, [N, 1, N + 1], (F32, F16, F16), seed=N)
    _case(btf, cuda, 570, 2, 64, 24, [N], (F16, F16, F16), seed=N, base=False)
    _case(btf, cuda, 1070, 2, 64, 24, [N], (F32, BF16, F32), seed=N)


def test_many_adapters(cuda, btf):
    _case(btf, cuda, 700, 1024, 64, 8, [40], (F32, BF16, F32), seed=1)
    _case(btf, cuda, 130, 1024, 64, 8, [40], (BF16, BF16, BF16), seed=2)
    _case(btf, cuda, 1300, 1024, 64, 8, [40], (F32, BF16, F32), seed=3)


@pytest.mark.parametrize("T", [200, 700, 1500, 3000])
def test_one_request_among_many(cuda, btf, T):
    """How K is split follows the tiles that there are, not those that could be."""
    index = torch.full((T,), 17, dtype=torch.int32, device=cuda)
    for types in ((F32, BF16, F32), (F16, F16, F16)):
        _case(btf, cuda, T, 24, 2056, 40, [70, 64, 9], types, seed=T, index=index, ranks=None)
    _case(btf, cuda, T, 24, 2056, 40, [70], (BF16, BF16, BF16), seed=T, index=torch.arange(T, dtype=torch.int32, device=cuda) % 3)


def test_no_row_has_an_adapter(cuda, btf):
    for T in (3, 500, 1100):
        for base in (True, False):
            _case(btf, cuda, T, 4, 64, 16, [50, 64], (F32, BF16, F32), index=torch.full((T,), -1, dtype=torch.int32, device=cuda), base=base)
            _case(btf, cuda, T, 4, 64, 16, [50, 64], (BF16, BF16, BF16), index=torch.full((T,), 4, dtype=torch.int32, device=cuda), base=base)
    x = torch.zeros(0, 64, device=cuda)
    a, b = torch.zeros(1, 8, 64, dtype=F16, device=cuda), torch.zeros(1, 5, 8, dtype=F16, device=cuda)
    out = btf.adapters(x, [btf.AdapterSeg(a, b)], btf.AdapterPlan(torch.zeros(0, dtype=torch.int32, device=cuda), 1))
    assert out[0].shape == (0, 5)


@pytest.mark.parametrize("T", [5, 301, 1101])
@pytest.mark.parametrize("w", [F16, BF16])
def test_nothing_behind_a_rank_matters(cuda, btf, T, w):
    """What lies behind an adapter's rank, and other rows' NaN and infinities, touch nothing."""
    n, K, R, N = 3, 96, 40, 70
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, w, F32, 5)
    index = _index(cuda, T, n, 6)
    ranks = torch.tensor([13, 0, 33], dtype=torch.int32, device=cuda)
    plan = btf.AdapterPlan(index, n)
    want = btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, ranks=ranks)[0]
    for j, r in enumerate((13, 0, 33)):
        a[j, r:], b[j, :, r:] = float("nan"), float("inf")
    assert torch.equal(btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, ranks=ranks)[0], want)
    with_one = (index == 0).nonzero()[:, 0]
    x[with_one[0], 3], x[with_one[-1], 5] = float("nan"), float("inf")
    got = btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, ranks=ranks)[0]
    spoiled = torch.zeros(T, dtype=torch.bool, device=cuda)
    spoiled[with_one[0]] = spoiled[with_one[-1]] = True
    assert torch.equal(got[~spoiled], want[~spoiled]) and not bool(got[spoiled].isfinite().any())
    for bad in (-3, 99):  # ranks are taken as 0 .. R
        r = torch.full((n,), bad, dtype=torch.int32, device=cuda)
        a2, b2 = a.nan_to_num(0, 0, 0), b.nan_to_num(0, 0, 0)
        _check(btf.adapters(x.nan_to_num(0, 0, 0), [btf.AdapterSeg(a2, b2, base=base)], plan, ranks=r)[0],
               _reference(x.nan_to_num(0, 0, 0), a2, b2, base, index, r, None, F32))


@pytest.mark.parametrize("T", [20, 1030])
def test_range_of_magnitudes(cuda, btf, T):
    """fp32 rows far from 1, with fp16 and bf16 weights: h leaves fp16's range, and its rows differ by 2^80."""
    n, K, R, N = 2, 64, 16, 40
    for w in (F16, BF16):
        x, (a,), (b,), _ = _inputs(cuda, T, n, K, R, [N], F32, w, F32, 8)
        x *= 2.0 ** torch.linspace(-60, 60, T, device=cuda).round()[:, None]
        a[:, ::2] *= 2.0 ** -8
        index = _index(cuda, T, n, 9, none=0)
        out = btf.adapters(x, [btf.AdapterSeg(a, b)], btf.AdapterPlan(index, n))[0]
        _check(out, _reference(x, a, b, None, index, None, None, F32))


@pytest.mark.parametrize("T", [11, 333, 1111])
@pytest.mark.parametrize("y_type", [F32, BF16])
def test_strides_and_in_place(cuda, btf, T, y_type):
    n, K, R, N = 4, 128, 16, 61
    x0, (a0,), (b0,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, BF16, y_type, 3)
    xw, aw, bw = torch.zeros(T, K + 12, device=cuda), torch.zeros(n, R + 3, K + 8, dtype=BF16, device=cuda), torch.zeros(n, N, 3 * R, dtype=BF16, device=cuda)
    x, a, b = xw[:, 4: 4 + K], aw[:, :R, :K], bw[:, :, R: 2 * R]
    x.copy_(x0), a.copy_(a0), b.copy_(b0)
    index = _index(cuda, T, n, 4)
    plan = btf.AdapterPlan(index, n)
    ref = _reference(x, a, b, base, index, None, None, y_type)
    for first, width in ((0, N), (8, 96), (1, N + 2), (3, 72)):  # aligned rows and others
        big = torch.full((T, width), 5.0, dtype=y_type, device=cuda) if width > N else torch.full((T, N), 5.0, dtype=y_type, device=cuda)
        first = min(first, width - N)
        y = big[:, first: first + N]
        btf.adapters(x, [btf.AdapterSeg(a, b, y, base)], plan)
        _check(y, ref)
        y.copy_(base)
        btf.adapters(x, [btf.AdapterSeg(a, b, y, y)], plan)  # in place
        _check(y, ref)
        assert bool((big[:, :first] == 5).all()) and bool((big[:, first + N:] == 5).all())
    # one row of base for all rows; one adapter's matrices for all adapters
    one = base[:1].expand(T, N)
    got = btf.adapters(x, [btf.AdapterSeg(a[:1].expand(n, R, K), b[:1].expand(n, N, R), base=one)], plan)[0]
    same = torch.where(index < 0, index, 0)
    _check(got, _reference(x, a[:1], b[:1], one, same, None, None, y_type))


@pytest.mark.parametrize("T", [200, 900])
def test_results_do_not_depend_on_the_run_and_rows_stand_alone(cuda, btf, T):
    """The same call gives the same bits; a row's result does not depend on the rows beside it in a tile."""
    n, K, R, N = 6, 1024, 32, 300
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], BF16, BF16, F32, 11)
    index = _index(cuda, T, n, 12)
    plan = btf.AdapterPlan(index, n)
    work = btf.adapters_work(x, [btf.AdapterSeg(a, b)], plan)
    first = btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, work=work)[0]
    work.fill_(255)  # NaN: nothing of the workspace is read before it is written
    for _ in range(3):
        assert torch.equal(btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, work=work)[0], first)
    p = torch.randperm(T, generator=torch.Generator().manual_seed(1)).to(cuda)
    again = btf.adapters(x[p], [btf.AdapterSeg(a, b, base=base[p])], btf.AdapterPlan(index[p].contiguous(), n))[0]
    assert torch.equal(again, first[p])


@pytest.mark.parametrize("T", [40, 1200])
def test_graph_and_streams(cuda, btf, T):
    """Plan and call captured in one graph and replayed with other rows; another stream."""
    n, K, R, N = 5, 256, 16, 128
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, F16, F32, 2)
    index = _index(cuda, T, n, 3)
    plan = btf.AdapterPlan(index, n)
    y = torch.empty(T, N, device=cuda)
    seg = [btf.AdapterSeg(a, b, y, base)]
    work = btf.adapters_work(x, seg, plan)
    ranks = torch.tensor([16, 3, 8, 0, 16], dtype=torch.int32, device=cuda)
    btf.adapters(x, seg, plan, ranks=ranks, work=work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(index)
        btf.adapters(x, seg, plan, ranks=ranks, work=work)
    for seed in (4, 5):
        index.copy_(_index(cuda, T, n, seed))
        x.copy_(torch.randn(T, K, generator=torch.Generator().manual_seed(seed)))
        y.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        _check(y, _reference(x, a, b, base, index, ranks, None, F32))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    z = btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, ranks=ranks, stream=s)[0]
    s.synchronize()
    assert torch.equal(z, y)
    assert btf.device_error() == 0


@pytest.mark.parametrize("T", [8, 1100])
def test_plan_of_other_sizes_is_reported(cuda, btf, T):
    """The C call with a plan that was made for other sizes writes nothing and says so."""
    n, K, R, N = 2, 64, 8, 16
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, F16, F32, 2)
    plan = btf.AdapterPlan(torch.zeros(T + 1, dtype=torch.int32, device=cuda), n)
    plan.T = T
    y = torch.full((T, N), 3.0, device=cuda)
    btf.adapters(x, [btf.AdapterSeg(a, b, y, base)], plan)
    torch.cuda.synchronize()
    assert btf.lib().btf_device_error(1) == 2 and bool((y == 3).all())
    assert btf.device_error() == 0


def test_refusals(cuda, btf):
    T, n, K, R, N = 8, 2, 64, 8, 16
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, F16, F32, 2)
    plan = btf.AdapterPlan(torch.zeros(T, dtype=torch.int32, device=cuda), n)
    S, i32 = btf.AdapterSeg, torch.int32
    y = torch.empty(T, N, device=cuda)
    for call in (
        lambda: btf.adapters(x, [], plan),
        lambda: btf.adapters(x, [S(a, b)] * 4, plan),
        lambda: btf.adapters(x[:7], [S(a, b)], plan),
        lambda: btf.adapters(x[:, :32], [S(a, b)], plan),
        lambda: btf.adapters(x.half().t().contiguous().t(), [S(a, b)], plan),
        lambda: btf.adapters(x.bfloat16(), [S(a, b)], plan),
        lambda: btf.adapters(x, [S(a.float(), b.float())], plan),
        lambda: btf.adapters(x, [S(a, b.bfloat16())], plan),
        lambda: btf.adapters(x, [S(a, b, y.bfloat16(), base.bfloat16())], plan),
        lambda: btf.adapters(x, [S(a, b, y, base.half())], plan),
        lambda: btf.adapters(x, [S(a, b, y[:, :15], base)], plan),
        lambda: btf.adapters(x, [S(a, b, y[:1].expand(T, N))], plan),
        lambda: btf.adapters(x, [S(a[:, :7], b[:, :, :7])], plan),
        lambda: btf.adapters(x, [S(a, b)], plan, ranks=torch.zeros(n, device=cuda)),
        lambda: btf.adapters(x, [S(a, b)], plan, ranks=torch.zeros(n + 1, dtype=i32, device=cuda)),
        lambda: btf.adapters(x, [S(a, b)], plan, scales=torch.zeros(n, dtype=torch.float64, device=cuda)),
        lambda: btf.adapters(x, [S(a, b)], plan, work=torch.empty(16, dtype=torch.uint8, device=cuda)),
        lambda: btf.adapters(x.cpu(), [S(a, b)], plan),
        lambda: btf.adapters(x, [S(a.cpu(), b)], plan),
        lambda: btf.adapters(x, [S(a, b.clone().requires_grad_())], plan),
        lambda: btf.adapters(x.clone().requires_grad_(), [S(a, b)], plan),
        lambda: btf.AdapterPlan(torch.zeros(T, device=cuda), n),
        lambda: btf.AdapterPlan(torch.zeros(T, dtype=i32), n),
        lambda: btf.AdapterPlan(torch.zeros(T, dtype=i32, device=cuda), 0),
        lambda: btf.AdapterPlan(torch.zeros(T, dtype=i32, device=cuda), 1025),
        lambda: plan.update(torch.zeros(T + 1, dtype=i32, device=cuda)),
        lambda: plan.update(None),
    ):
        with pytest.raises(RuntimeError):
            call()
    assert ctypes.sizeof(btf.AdapterSegC) == btf._ADAPTER_SEG.size
    assert ctypes.sizeof(btf.AdaptersArgsC) == btf._ADAPTERS_HEAD.size + 3 * btf._ADAPTER_SEG.size + btf._ADAPTERS_TAIL.size
