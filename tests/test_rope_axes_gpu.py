"""GPU tests of rotary positions with several axes (btf_rope_axes) against the formula in 64 bits; the tolerance is that
of the positions with one axis (test_rope_gpu.py), whose arithmetic it shares."""
import numpy as np
import pytest
import torch

from test_rope_gpu import TYPES, _check

pytestmark = pytest.mark.gpu


def _reference(x, table, pos, inverse=False, normw=None, eps=1e-6):
    """(value, |a| + |b| of its pair times m) in 64 bits; pos [axes][T]."""
    x = x.double().cpu()
    if normw is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * normw.double().cpu()
    R, m = table.n_rot, table.mscale
    ang = pos.double().cpu().numpy()[table.axis_host[: R // 2]].T * table.host[: R // 2]
    ang = torch.from_numpy((ang - np.round(ang)) * 2 * np.pi)[:, None]
    c, s = ang.cos() * m, ang.sin() * (-m if inverse else m)
    y, size = x.clone(), x.abs()
    sa, sb = (slice(0, R, 2), slice(1, R, 2)) if table.interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., sa], x[..., sb]
    y[..., sa], y[..., sb] = a * c - b * s, a * s + b * c
    size[..., sa] = size[..., sb] = (a.abs() + b.abs()) * m
    return y, size


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("axes", ["split", "turns", "own"])
@pytest.mark.parametrize("T,H,D,sections", [(1, 1, 64, [32]), (3, 5, 256, [11, 11, 10]), (257, 2, 128, [24, 20, 20]),
                                            (5, 3, 80, [20, 20]), (7, 2, 100, [5, 12, 3, 5]), (33, 40, 128, [16, 0, 24, 8]),
                                            (4, 1, 6, [1, 1, 1]), (2, 2, 1024, [500, 12]), (9, 3, 72, [0, 36])])
def test_layouts_and_types(cuda, btf, T, H, D, sections, axes, inter):
    g = torch.Generator().manual_seed(T * 1000 + D)
    table = btf.RopeTable(2 * sum(sections), base=1e6, interleaved=inter, sections=sections, axes=axes)
    pos = torch.randint(-50, 5000, (len(sections), T), generator=g, dtype=torch.int32)
    for t in TYPES:
        x = torch.randn(T, H, D, generator=g).to(t)
        y = torch.full((T, H, D), 7.0, dtype=t, device=cuda)
        btf.rope([btf.RopeSeg(x.to(cuda), y)], table, pos.to(cuda))
        _check(y, *_reference(x, table, pos))


def test_norm_append_and_padding(cuda, btf):
    """The decoder's q/k norm, rotation and append, more rounds than lanes too; tokens without a slot are not written."""
    for D, sections in ((256, [11, 11, 10]), (1024, [100, 100, 56])):
        T, H, HK, ctx = 6, 6, 2, 40
        g = torch.Generator().manual_seed(3)
        qg = torch.randn(T, H, 2 * D, generator=g)
        k, v = (torch.randn(T, HK, D, generator=g) for _ in range(2))
        qn, kn = (1.2 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
        pos = torch.tensor([[9, 10, 10, 10, 11, 12], [9, 10, 11, 12, 13, 13], [9, 10, 10, 11, 10, 14]], dtype=torch.int32)
        rows = torch.tensor([39, 0, 1, -1, 3, 40], dtype=torch.int32)
        table = btf.RopeTable(2 * sum(sections), base=1e7, sections=sections, axes="turns")
        yq = torch.zeros(T, H, D, dtype=torch.float16, device=cuda)
        kc, vc = (torch.full((ctx, HK, D), 5.0, dtype=torch.float16, device=cuda) for _ in range(2))
        btf.rope([btf.RopeSeg(qg.to(cuda)[..., :D], yq, normw=qn.to(cuda)),
                  btf.RopeSeg(k.to(cuda), kc, normw=kn.to(cuda), rows=rows.to(cuda)),
                  btf.RopeSeg(v.to(cuda), vc, rotate=False, rows=rows.to(cuda))], table, pos.to(cuda))
        _check(yq, *_reference(qg[..., :D], table, pos, normw=qn), normed_D=D)
        there = [0, 1, 2, 4]
        slots = rows[there].long()
        ref, size = _reference(k, table, pos, normw=kn)
        _check(kc[slots], ref[there], size[there], normed_D=D)
        _check(vc[slots], v.double()[there], v.double().abs()[there])
        untouched = [i for i in range(ctx) if i not in slots.tolist()]
        assert bool((kc[untouched] == 5).all()) and bool((vc[untouched] == 5).all())


def test_equal_positions_are_the_positions_of_one_axis(cuda, btf):
    """Text has one position on every axis: the same bits as the call of one axis, by one shared row of positions too."""
    T, H, D = 31, 4, 128
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(1)).to(cuda)
    pos = torch.randint(0, 200000, (T,), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(cuda)
    kw = dict(base=5e5, scaling="yarn", factor=4.0, orig_ctx=4096)
    want = torch.empty_like(x)
    btf.rope([btf.RopeSeg(x, want)], btf.RopeTable(96, **kw), pos)
    for axes in ("split", "turns"):
        table = btf.RopeTable(96, sections=[20, 14, 14], axes=axes, **kw)
        for p in (pos.repeat(3, 1), pos.expand(3, T), torch.stack([pos] * 7)[2:5]):
            y = torch.empty_like(x)
            btf.rope([btf.RopeSeg(x, y)], table, p)
            assert torch.equal(y, want)


@pytest.mark.parametrize("axes", ["split", "turns", "own"])
def test_inverse_is_the_gradient(cuda, btf, axes):
    """<rope(x), g> = <x, inverse(g)>, and the inverse against differences of the formula."""
    T, H, D, sections = 11, 3, 80, [15, 10, 15]
    gen = torch.Generator().manual_seed(5)
    x, g = (torch.randn(T, H, D, generator=gen) for _ in range(2))
    pos = torch.randint(0, 3000, (3, T), generator=gen, dtype=torch.int32)
    table = btf.RopeTable(80, base=1e4, scaling="yarn", factor=2.0, orig_ctx=512, interleaved=True, sections=sections, axes=axes)
    dx = torch.empty(T, H, D, device=cuda)
    btf.rope([btf.RopeSeg(g.to(cuda), dx)], table, pos.to(cuda), inverse=True)
    _check(dx, *_reference(g, table, pos, inverse=True))
    # the map is linear: a difference over a step of 1 is the derivative
    for (t, h, d) in [(0, 0, 0), (3, 1, 41), (10, 2, 79)]:
        e = torch.zeros(T, H, D, dtype=torch.float64)
        e[t, h, d] = 1
        diff = (_reference(x.double() + e, table, pos)[0] - _reference(x, table, pos)[0])
        want = float((diff * g.double()).sum())
        # two terms of the sum, each off by what _check allows of |a| + |b| <= 8, and the differences' own rounding
        assert abs(float(dx[t, h, d]) - want) <= 8 * 8 * 2.0 ** -24 * table.mscale + 1e-12


def test_graph_other_stream_and_in_place(cuda, btf):
    T, H, D = 5, 4, 64
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(T, H, D, generator=gen).to(cuda)
    table = btf.RopeTable(64, base=1e4, sections=[12, 10, 10], axes="turns")
    pos = torch.randint(0, 3000, (3, T), generator=gen, dtype=torch.int32).to(cuda)
    y = torch.empty_like(x)
    btf.rope([btf.RopeSeg(x, y)], table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    z = x.clone()
    torch.cuda.synchronize()
    btf.rope([btf.RopeSeg(z)], table, pos, stream=s)
    s.synchronize()
    assert torch.equal(z, y)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        btf.rope([btf.RopeSeg(x, out)], table, pos)
    pos += 17
    graph.replay()
    btf.rope([btf.RopeSeg(x, y)], table, pos)
    assert torch.equal(out, y)


def test_refusals(cuda, btf):
    x = torch.zeros(4, 2, 64, device=cuda)
    table = btf.RopeTable(64, sections=[12, 10, 10])
    pos = torch.zeros(3, 4, dtype=torch.int32, device=cuda)
    for bad in (None, pos[0], pos[:2], pos.long(), pos.t().contiguous().t(), pos.cpu(), pos[:, :3]):
        with pytest.raises(RuntimeError):
            btf.rope([btf.RopeSeg(x)], table, bad)
    with pytest.raises(RuntimeError):  # a table of one axis takes one position per token
        btf.rope([btf.RopeSeg(x)], btf.RopeTable(64), pos)
    table.axis = table.axis[:-1]
    with pytest.raises(RuntimeError):
        btf.rope([btf.RopeSeg(x)], table, pos)
