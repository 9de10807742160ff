"""GPU tests of the rotary positions (btf_rope) against the formula in 64 bits.

Tolerance of a rotated value, from a and b of its pair and the factor m: an angle's fraction of a turn is rounded to
fp32 (|f| <= 1/2: 2^-25 of a turn, 2 pi 2^-25 rad), sincospif is good to 2 ulp of 1 (2^-23) and the product with m and
the two fused products round thrice (3 * 2^-24); so (|a| + |b|) m (2 pi 2^-25 + 2^-23 + 3 * 2^-24) < (|a| + |b|) m 8 * 2^-24.
A norm before it multiplies by 1 / sqrt(mean + eps): D terms summed in fp32 (D 2^-24 of the mean at most, half of
that on the root), division, root and two products: (D / 2 + 5) 2^-24 more. Rounding to the output type adds eps / 2."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SCALINGS = {"none": {}, "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=2.5),
            "yarn": dict(scaling="yarn", factor=8.0, orig_ctx=2048)}


def _reference(x, turns, m, pos, inter, inverse=False, normw=None, eps=1e-6):
    """(value, |a| + |b| of its pair times m) in 64 bits."""
    x = x.double().cpu()
    if normw is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * normw.double().cpu()
    R = 2 * len(turns)
    ang = (pos.double().cpu()[:, None] * torch.from_numpy(turns))
    ang = ((ang - ang.round()) * 2 * np.pi)[:, None]
    c, s = ang.cos() * m, ang.sin() * (-m if inverse else m)
    y, size = x.clone(), x.abs()
    sa, sb = (slice(0, R, 2), slice(1, R, 2)) if inter else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., sa], x[..., sb]
    y[..., sa], y[..., sb] = a * c - b * s, a * s + b * c
    size[..., sa] = size[..., sb] = (a.abs() + b.abs()) * m
    return y, size


def _check(y, ref, size, normed_D=0):
    eps = torch.finfo(y.dtype).eps
    tol = size * (8 + (normed_D / 2 + 5 if normed_D else 0)) * U + (ref.abs() * eps / 2 if eps > 1e-6 else 0)
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of the smallest numbers
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= tol + 1e-30).all()), float((err - tol).max())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 64, 64), (3, 5, 256, 64), (257, 2, 128, 128), (5, 3, 80, 40), (7, 2, 100, 50),
                                     (2, 3, 72, 72), (4, 1, 2, 2), (3, 2, 7, 4), (2, 2, 1024, 1024), (6, 2, 96, 0),
                                     (33, 40, 128, 96), (2, 3, 1000, 998), (1, 1, 1, 0)])
def test_shapes(cuda, btf, T, H, D, R, inter):
    g = torch.Generator().manual_seed(T * 1000 + D)
    x = torch.randn(T, H, D, generator=g)
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
    if R:
        table = btf.RopeTable(R, base=1e6, interleaved=inter)
        ref, size = _reference(x, table.host, table.mscale, pos, inter)
    else:
        table = btf.RopeTable(2, interleaved=inter)
        table.n_rot = 0  # nothing rotated: the dims are copied
        ref, size = x.double(), x.double().abs()
    for t in TYPES:
        xt = x.to(t)
        if t != torch.float32 and R:
            ref, size = _reference(xt, table.host, table.mscale, pos, inter)
        elif t != torch.float32:
            ref, size = xt.double(), xt.double().abs()
        y = torch.full((T, H, D), 7.0, dtype=t, device=cuda)
        btf.rope([btf.RopeSeg(xt.to(cuda), y)], table, pos.to(cuda))
        _check(y, ref, size)


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("inter", [False, True])
def test_scalings_and_far_positions(cuda, btf, scaling, inter):
    T, H, D, R = 9, 2, 128, 64
    table = btf.RopeTable(R, base=1e4, interleaved=inter, **SCALINGS[scaling])
    pos = torch.tensor([0, 1, -1, 4095, 131071, 1000003, 2 ** 31 - 1, -2 ** 31, 77], dtype=torch.int32)
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(1))
    ref, size = _reference(x, table.host, table.mscale, pos, inter)
    y = torch.empty(T, H, D, device=cuda)
    btf.rope([btf.RopeSeg(x.to(cuda), y)], table, pos.to(cuda))
    # 2^31 / 2 pi turns in 64 bits are rounded by 2^-25 of a turn: another 2 pi 2^-25 rad, on top of the same of the
    # fp32 fraction, in the reference and in the kernel: 2 * 2 pi 2^-25 < 7 * 2^-24
    _check(y, ref, size * (15 / 8))


@pytest.mark.parametrize("x_type", TYPES)
@pytest.mark.parametrize("y_type", TYPES)
def test_types_norm_and_cache_rows(cuda, btf, x_type, y_type):
    """The decoder's q/k norm, rotation and append: q out of (q, gate) rows, k and v into slots of a cache."""
    T, H, HK, D, R, ctx = 6, 6, 2, 256, 64, 40
    g = torch.Generator().manual_seed(3)
    qg = torch.randn(T, H, 2 * D, generator=g).to(x_type)
    k, v = (torch.randn(T, HK, D, generator=g).to(x_type) for _ in range(2))
    qn, kn = (1.2 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
    pos = torch.tensor([9, 10, 10, 11, 11, 12], dtype=torch.int32)
    rows = torch.tensor([39, 0, 1, -1, 3, 40], dtype=torch.int32)  # two tokens without a slot
    table = btf.RopeTable(R, base=1e7)
    yq = torch.zeros(T, H, D, dtype=y_type, device=cuda)
    kc, vc = (torch.full((ctx, HK, D), 5.0, dtype=y_type, device=cuda) for _ in range(2))
    btf.rope([btf.RopeSeg(qg.to(cuda)[..., :D], yq, normw=qn.to(cuda)),
              btf.RopeSeg(k.to(cuda), kc, normw=kn.to(cuda), rows=rows.to(cuda)),
              btf.RopeSeg(v.to(cuda), vc, rotate=False, rows=rows.to(cuda))], table, pos.to(cuda))
    ref, size = _reference(qg[..., :D], table.host, 1.0, pos, False, normw=qn)
    _check(yq, ref, size, normed_D=D)
    there = [0, 1, 2, 4]
    slots = rows[there].long()
    ref, size = _reference(k, table.host, 1.0, pos, False, normw=kn)
    _check(kc[slots], ref[there], size[there], normed_D=D)
    _check(vc[slots], v.double()[there], v.double().abs()[there])
    other = [i for i in range(ctx) if i not in slots.tolist()]
    assert bool((kc[other] == 5).all()) and bool((vc[other] == 5).all())


@pytest.mark.parametrize("D,R,inter", [(128, 128, False), (100, 60, True), (1024, 512, False)])
def test_norm_alone_and_odd_sizes(cuda, btf, D, R, inter):
    x = torch.randn(3, 2, D, generator=torch.Generator().manual_seed(2)) * 3
    w = torch.rand(D, generator=torch.Generator().manual_seed(4)) + 0.5
    pos = torch.tensor([1, 2, 3], dtype=torch.int32)
    table = btf.RopeTable(R, interleaved=inter)
    y = torch.empty(3, 2, D, device=cuda)
    btf.rope([btf.RopeSeg(x.to(cuda), y, normw=w.to(cuda))], table, pos.to(cuda), eps=1e-5)
    ref, size = _reference(x, table.host, 1.0, pos, inter, normw=w, eps=1e-5)
    _check(y, ref, size, normed_D=D)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_in_place_strided_slices(cuda, btf, t, inter):
    """q and k are slices of a fused projection's rows, rotated where they lie; v between them stays."""
    T, H, HK, D = 5, 4, 2, 64
    rows = torch.randn(T, (H + 2 * HK) * D, generator=torch.Generator().manual_seed(5)).to(t)
    pos = torch.arange(100, 100 + T, dtype=torch.int32)
    table = btf.RopeTable(D, interleaved=inter)
    d = rows.to(cuda)
    cut = lambda x: (x[:, : H * D].unflatten(1, (H, D)), x[:, H * D:(H + HK) * D].unflatten(1, (HK, D)))  # noqa: E731
    q, k = cut(d)
    btf.rope([btf.RopeSeg(q), btf.RopeSeg(k)], table, pos.to(cuda))
    for got, x in zip(cut(d), cut(rows)):
        _check(got, *_reference(x, table.host, 1.0, pos, inter))
    assert torch.equal(d[:, (H + HK) * D:].cpu(), rows[:, (H + HK) * D:])


@pytest.mark.parametrize("off,stride", [(1, 131), (2, 130), (4, 132), (3, 200)])
def test_any_alignment(cuda, btf, off, stride):
    T, D = 4, 64
    for t in TYPES:
        buf = torch.randn(8 + T * stride * 2, generator=torch.Generator().manual_seed(6)).to(t)
        x = buf[off:].as_strided((T, 2, D), (2 * stride, stride, 1))
        pos = torch.arange(T, dtype=torch.int32) * 50
        table = btf.RopeTable(32, interleaved=True)
        out = torch.zeros(8 + T * stride * 2, dtype=t, device=cuda)
        y = out[off:].as_strided((T, 2, D), (2 * stride, stride, 1))
        btf.rope([btf.RopeSeg(buf.to(cuda)[off:].as_strided((T, 2, D), (2 * stride, stride, 1)), y)], table, pos.to(cuda))
        _check(y, *_reference(x, table.host, 1.0, pos, True))
        y.zero_()
        assert float(out.abs().max()) == 0  # nothing else was written


@pytest.mark.parametrize("scaling", ["none", "yarn"])
@pytest.mark.parametrize("inter", [False, True])
def test_inverse_is_the_gradient(cuda, btf, scaling, inter):
    """The transposed map: against its formula, <R x, g> == <x, R^T g>, and differences of the forward pass."""
    T, H, D, R = 6, 3, 48, 32
    gen = torch.Generator().manual_seed(7)
    x, gy = torch.randn(T, H, D, generator=gen), torch.randn(T, H, D, generator=gen)
    pos = torch.randint(0, 9000, (T,), generator=gen, dtype=torch.int32)
    table = btf.RopeTable(R, interleaved=inter, **SCALINGS[scaling])
    out = [torch.empty(T, H, D, device=cuda) for _ in range(3)]
    btf.rope([btf.RopeSeg(gy.to(cuda), out[0])], table, pos.to(cuda), inverse=True)
    _check(out[0], *_reference(gy, table.host, table.mscale, pos, inter, inverse=True))
    btf.rope([btf.RopeSeg(x.to(cuda), out[1])], table, pos.to(cuda))
    lhs, rhs = (out[1].double().cpu() * gy.double()).sum(), (x.double() * out[0].double().cpu()).sum()
    n = T * H * D
    assert abs(float(lhs - rhs)) <= 2 * n * 9 * U * 4 * table.mscale  # n products of |x||g| < 16, each 8 + 1 units off
    # a linear map: a step of 2^3 in one entry shows its column, each side within the forward tolerance
    e = torch.zeros_like(x)
    e[2, 1, 5] = 8.0
    btf.rope([btf.RopeSeg((x + e).to(cuda), out[2])], table, pos.to(cuda))
    diff = ((out[2] - out[1]).double().cpu() * gy.double()).sum() / 8.0
    assert abs(float(diff) - float(out[0][2, 1, 5])) <= 2 * 16 * 9 * U * 16


def test_streams_graph_and_large_offsets(cuda, btf):
    T, H, D = 32, 8, 128
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(8)).to(cuda)
    pos = torch.arange(T, dtype=torch.int32, device=cuda)
    table = btf.RopeTable(D)
    ys = [torch.empty_like(x) for _ in range(3)]
    btf.rope([btf.RopeSeg(x, ys[0])], table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    btf.rope([btf.RopeSeg(x, ys[1])], table, pos, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        btf.rope([btf.RopeSeg(x, ys[2])], table, pos)
    for k in range(2):
        pos.copy_(torch.arange(T, dtype=torch.int32) + 10 * k)
        x.copy_(x + k)
        graph.replay()
        if k == 0:
            assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])
    btf.rope([btf.RopeSeg(x, ys[0])], table, pos)
    assert torch.equal(ys[0], ys[2])
    # a cache row behind 2^31 elements
    cache = torch.empty((2 ** 21 + 40) * H * D, dtype=torch.float16, device=cuda).view(-1, H, D)
    rows = torch.arange(2 ** 21 + 8, 2 ** 21 + 8 + T, dtype=torch.int32, device=cuda)
    cache[rows.long()] = 0
    btf.rope([btf.RopeSeg(x, cache, rows=rows)], table, pos)
    assert torch.equal(cache[rows.long()], ys[0].half())


def test_refusals(cuda, btf):
    x = torch.zeros(4, 2, 64, device=cuda)
    pos = torch.zeros(4, dtype=torch.int32, device=cuda)
    table = btf.RopeTable(64)
    bad = [
        lambda: btf.rope([btf.RopeSeg(x)], table, pos.long()),
        lambda: btf.rope([btf.RopeSeg(x)], table, pos[:3]),
        lambda: btf.rope([btf.RopeSeg(x)], table, pos.cpu()),
        lambda: btf.rope([btf.RopeSeg(x.double())], table, pos),
        lambda: btf.rope([btf.RopeSeg(x[..., ::2])], btf.RopeTable(32), pos),
        lambda: btf.rope([btf.RopeSeg(x[..., :32])], table, pos),
        lambda: btf.rope([btf.RopeSeg(x, torch.zeros(3, 2, 64, device=cuda))], table, pos),
        lambda: btf.rope([btf.RopeSeg(x, normw=torch.ones(64, device=cuda))], table, pos, inverse=True),
        lambda: btf.rope([btf.RopeSeg(x, normw=torch.ones(63, device=cuda))], table, pos),
        lambda: btf.rope([btf.RopeSeg(x, x, rows=pos)], table, pos),
    ]
    for fn in bad:
        with pytest.raises(RuntimeError):
            fn()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t", [torch.float16, torch.float32])
def test_many_tokens(cuda, btf, t, inter):
    """Enough of them that a thread takes several batches of heads, the last one short; rows checked here and there."""
    T, H, D = 16001, 41, 128
    g = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(T, H, D, generator=g, device=cuda).to(t)
    y = torch.empty_like(x)
    pos = torch.arange(70000, 70000 + T, dtype=torch.int32, device=cuda)
    table = btf.RopeTable(D, base=1e6, interleaved=inter)
    btf.rope([btf.RopeSeg(x, y)], table, pos)
    at = torch.cat([torch.arange(0, T, 97), torch.tensor([T - 2, T - 1])]).to(cuda)
    ref, size = _reference(x[at], table.host, 1.0, pos[at], inter)
    _check(y[at], ref, size)
    # every row keeps its length: an element is off by (|a| + |b|) 8 * 2^-24 + |y| eps / 2 at most, and |a| + |b| is
    # at most sqrt 2 of its pair's length, so the square by 2 sqrt 2 * 8 * 2^-24 + eps of it, below 2^-19 + 2 eps
    a, b = x.double().square().sum(-1), y.double().square().sum(-1)
    assert float(((a - b).abs() / a).max()) <= 2 * torch.finfo(t).eps + 2.0 ** -19


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,H,D,R,off", [(5, 3, 100, 100, 0), (5, 3, 100, 50, 0), (4, 2, 80, 20, 0), (3, 5, 72, 36, 0),
                                         (2, 3, 1024, 512, 0), (6, 2, 128, 128, 1), (3, 2, 65, 0, 0), (4, 3, 256, 64, 0),
                                         (3001, 33, 100, 100, 0), (1201, 33, 1024, 1024, 0)])
def test_norm_in_place(cuda, btf, T, H, D, R, off, t, inter):
    """A head's norm is that of its values before any of them is replaced, however many rounds of lanes it takes: the
    same bits as a call into another tensor of the same layout, and the formula's values."""
    g = torch.Generator(device=cuda).manual_seed(T + D + R)
    x = (torch.randn(T * H * D + off, generator=g, device=cuda) * 2).to(t)[off:].view(T, H, D)
    w = torch.rand(D, generator=g, device=cuda) + 0.5
    pos = torch.randint(0, 5000, (T,), generator=g, device=cuda, dtype=torch.int32)
    table = btf.RopeTable(max(R, 2), base=1e6, interleaved=inter)
    table.n_rot = R
    y = torch.zeros(T * H * D + off, dtype=t, device=cuda)[off:].view(T, H, D)
    btf.rope([btf.RopeSeg(x, y, normw=w)], table, pos)
    given = x.cpu()
    btf.rope([btf.RopeSeg(x, normw=w)], table, pos)
    assert torch.equal(x, y)
    at = list(range(T))[:: max(1, T // 50)]
    ref, size = _reference(given[at], table.host[: R // 2], 1.0, pos[at], inter, normw=w)
    _check(x[at], ref, size, normed_D=D)
