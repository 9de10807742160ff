"""The operators of many requests as they are used together: the adapters' part of q, k and v beside the shared projection,
positions of three axes with the append to each sequence's cache, attention over the shared prompt and the own rows, the
adapters' part of the output; captured in one graph and replayed as the batch changes. Each stage is held to its formula in
64 bits on what the stage before it gave."""
import gc

import pytest
import torch

from test_adapters_gpu import _check as check_adapters, _reference as adapters_reference
from test_prefix_attention_gpu import _joined
from test_rope_axes_gpu import _reference as axes_reference
from test_rope_gpu import _check as check_rope
from test_tree_attention_gpu import _check as check_attention, _reference as attention_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
def test_adapters_rope_attention_adapters(cuda, btf, t):
    B, H, HK, D, K, R, n, ctx, P = 21, 6, 2, 128, 264, 24, 5, 90, 333
    g = torch.Generator(device=cuda).manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    i32 = lambda a: torch.as_tensor(list(a) if isinstance(a, range) else a, dtype=torch.int32).to(cuda)  # noqa: E731
    widths = [H * D, HK * D, HK * D]
    x, proj = rn(B, K), [rn(B, N) for N in widths]
    a, b = [(rn(n, R, K) * K ** -0.5).to(t) for _ in widths], [(rn(n, N, R) * 0.3).to(t) for N in widths]
    oa, ob = (rn(n, R, H * D) * (H * D) ** -0.5).to(t), (rn(n, K, R) * 0.3).to(t)
    ranks, scales = i32([24, 0, 7, 16, 24]), torch.rand(n, generator=g, device=cuda) + 0.5
    pk, pv = (rn(P, HK, D) * 1.5).to(t), rn(P, HK, D).to(t)
    kc, vc = (torch.full((B, ctx, HK, D), float("nan"), dtype=t, device=cuda) for _ in range(2))
    table = btf.RopeTable(96, base=1e6, sections=[16, 20, 12], axes="turns")
    index, lens, used = i32([0] * B), i32([0] * B), i32([P])
    pos, rows, parents, counts = i32([[0] * B] * 3), i32(range(0, B * ctx, ctx)), i32([[-1]] * B), i32([1] * B)
    y = [torch.empty(B, N, device=cuda) for N in widths]
    q16, o = torch.empty(B, H, D, dtype=t, device=cuda), torch.zeros(B, 1, H, D, dtype=t, device=cuda)
    out = torch.empty(B, K, device=cuda)
    qkv = [btf.AdapterSeg(p, q, z, c) for p, q, z, c in zip(a, b, y, proj)]
    plan = btf.AdapterPlan(index, n)
    last = [btf.AdapterSeg(oa, ob, out, x)]
    work = btf.adapters_work(x, qkv, plan)
    work_o = btf.adapters_work(o.view(B, H * D), last, plan)
    work_p = btf.prefix_attention_work(q16[:, None], pk, kc)

    def forward():
        plan.update(index)
        btf.adapters(x, qkv, plan, ranks=ranks, scales=scales, work=work)
        q, k, v = (z.view(B, -1, D) for z in y)
        btf.rope([btf.RopeSeg(q, q16), btf.RopeSeg(k, kc.view(B * ctx, HK, D), rows=rows),
                  btf.RopeSeg(v, vc.view(B * ctx, HK, D), rotate=False, rows=rows)], table, pos)
        btf.prefix_attention(q16[:, None], pk, pv, kc, vc, lens, parents, prefix_len=used, counts=counts, out=o, work=work_p)
        btf.adapters(o.view(B, H * D).float(), last, plan, ranks=ranks, scales=scales, work=work_o)

    forward()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forward()
    gh = torch.Generator().manual_seed(7)
    for step in range(4):
        lens.copy_(torch.randint(0, ctx, (B,), generator=gh, dtype=torch.int32))
        index.copy_(torch.randint(-1, n, (B,), generator=gh, dtype=torch.int32))
        counts.copy_(torch.rand(B, generator=gh) < (0.7, 1.0, 0.1, 0.0)[step])
        used.fill_((P, 100, 0, 1)[step])
        pos.copy_(lens + used + i32([[0], [3], [-2]]))
        rows.copy_(torch.arange(B, device=cuda, dtype=torch.int32) * ctx + lens)
        for s in range(B):  # what lies before the new row must have been written
            kc[s, : lens[s]], vc[s, : lens[s]] = rn(int(lens[s]), HK, D).to(t), rn(int(lens[s]), HK, D).to(t)
        x.copy_(rn(B, K))
        graph.replay()
        torch.cuda.synchronize()
        for z, p, q, c in zip(y, a, b, proj):
            check_adapters(z, adapters_reference(x, p, q, c, index, ranks, scales, torch.float32))
        check_rope(q16, *axes_reference(y[0].view(B, H, D), table, pos))
        at = torch.arange(B, device=cuda), lens.long()
        check_rope(kc[at], *axes_reference(y[1].view(B, HK, D), table, pos))
        assert torch.equal(vc[at], y[2].view(B, HK, D).to(t))
        kj, vj = _joined(pk.cpu(), pv.cpu(), kc.cpu(), vc.cpu(), int(used))
        check_attention(o, attention_reference(q16[:, None].cpu(), kj, vj, (lens + used).tolist(), [[-1]] * B,
                                               counts.tolist(), D ** -0.5), t)
        check_adapters(out, adapters_reference(o.view(B, H * D).float(), oa, ob, x, index, ranks, scales, torch.float32))
    assert btf.device_error() == 0


def _calls(cuda, btf):
    g = torch.Generator(device=cuda).manual_seed(8)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    i32 = lambda a: torch.as_tensor(list(a) if isinstance(a, range) else a, dtype=torch.int32).to(cuda)  # noqa: E731
    T, K, R, n, N, H, HK, D, ctx, P = 9, 64, 16, 3, 40, 6, 2, 64, 30, 70
    x, base, index = rn(T, K), rn(T, N), i32([0, 1, 2, -1, 0, 2, 2, 1, 0])
    a, b = rn(n, R, K).half(), rn(n, N, R).half()
    ranks, scales = i32([16, 3, 9]), rn(n)
    plan = btf.AdapterPlan(index, n)
    rx, kc = rn(T, H, D), rn(ctx, H, D).half()
    pos, rows = i32([list(range(7, 7 + T)), list(range(T)), [5] * T]), i32(list(range(3, 3 + T)))
    table = btf.RopeTable(32, sections=[4, 4, 8], axes="own", interleaved=True)
    q, k, v, pk, pv = rn(2, 3, H, D).half(), rn(2, ctx, HK, D).half(), rn(2, ctx, HK, D).half(), rn(P, HK, D).half(), rn(P, HK, D).half()
    lens, parents, counts, used = i32([27, 5]), i32([[-1, 0, 1], [-1, -1, 0]]), i32([3, 2]), i32([50])

    def all_calls(**kw):
        y, c = base.clone(), kc.clone()
        btf.adapters(x, [btf.AdapterSeg(a, b, y, y)], plan, ranks=ranks, scales=scales, **kw)
        h = btf.adapters(x, [btf.AdapterSeg(a, b), btf.AdapterSeg(a, b, base=base)], plan, **kw)
        btf.rope([btf.RopeSeg(rx, c, rows=rows)], table, pos, **kw)
        o = btf.prefix_attention(q, pk, pv, k, v, lens, parents, **kw)
        o2 = btf.prefix_attention(q, pk, pv, k, v, lens, parents, used, counts, 0.3, torch.zeros_like(q), **kw)
        return [y, *h, c, o, o2]

    bad = (lambda: btf.adapters(x[:3], [btf.AdapterSeg(a, b)], plan), lambda: btf.adapters(x, [btf.AdapterSeg(a, b.float())], plan),
           lambda: btf.adapters(x, [btf.AdapterSeg(a, b)], plan, ranks=scales), lambda: btf.rope([btf.RopeSeg(rx)], table, pos[:2]),
           lambda: btf.rope([btf.RopeSeg(rx)], table, pos[0]), lambda: btf.prefix_attention(q, pk.float(), pv, k, v, lens, parents),
           lambda: btf.prefix_attention(q, pk, pv, k, v, lens, parents, lens),
           lambda: btf.prefix_attention(q, pk, pv, k, v, lens, parents, work=torch.empty(256, dtype=torch.uint8, device=cuda)))
    return all_calls, bad


def test_short_and_long_way_of_a_call_agree(cuda, btf, monkeypatch):
    """The binding of ordinary calls does them itself, on the current stream too; what it leaves to the Python mirror (a
    stream that is given, an error) ends the same way, and neither keeps a reference."""
    all_calls, bad = _calls(cuda, btf)
    btf.ensure_init(0)
    calls, taken = btf._calls, []
    assert calls is not None

    class Seen:
        def __getattr__(self, name):
            def call(*a):
                r = getattr(calls, name)(*a)
                taken.append(r is not None)
                return r
            return call

    monkeypatch.setattr(btf, "_calls", Seen())
    short = all_calls()
    assert len(taken) == 5 and all(taken)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = all_calls()
    side.synchronize()
    given = all_calls(stream=side)
    side.synchronize()
    assert len(taken) == 10 and all(taken)
    for fn in bad:
        with pytest.raises(RuntimeError):
            fn()
    assert not any(taken[10:])
    monkeypatch.setattr(btf, "_calls", None)
    for fn in bad:
        with pytest.raises(RuntimeError):
            fn()
    long = all_calls()
    for other in (on_side, given, long):
        for p, q in zip(short, other):
            assert p.dtype == q.dtype and torch.equal(p, q)
    monkeypatch.setattr(btf, "_calls", calls)
    torch.cuda.synchronize()
    del short, on_side, given, long, other, p, q
    gc.collect()
    before = torch.cuda.memory_allocated()
    for _ in range(50):
        all_calls()
    gc.collect()
    assert torch.cuda.memory_allocated() <= before


def test_two_graphs_share_one_workspace(cuda, btf):
    """Captured calls with one workspace, replayed after one another: none reads what the other left there."""
    g = torch.Generator(device=cuda).manual_seed(9)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    i32 = lambda a: torch.as_tensor(list(a) if isinstance(a, range) else a, dtype=torch.int32).to(cuda)  # noqa: E731
    n, K, N, R = 4, 128, 72, 32
    a, b = rn(n, R, K).bfloat16(), rn(n, N, R).bfloat16()
    pk, pv = rn(300, 2, 64).half(), rn(300, 2, 64).half()
    runs = []
    for T, B in ((700, 3), (40, 17)):
        x, index = rn(T, K).bfloat16(), torch.randint(-1, n, (T,), generator=g, device=cuda, dtype=torch.int32)
        q, k = rn(B, 2, 4, 64).half(), rn(B, 90, 2, 64).half()
        lens, parents = torch.randint(0, 88, (B,), generator=g, device=cuda, dtype=torch.int32), i32([[-1, 0]] * B)
        runs.append((x, [btf.AdapterSeg(a, b, torch.empty(T, N, device=cuda, dtype=torch.bfloat16))], btf.AdapterPlan(index, n), q, k,
                     lens, parents, torch.empty_like(q)))
    work = max((btf.adapters_work(r[0], r[1], r[2]) for r in runs), key=len)
    work_p = max((btf.prefix_attention_work(r[3], pk, r[4]) for r in runs), key=len)
    graphs, want = [], []
    for x, segs, plan, q, k, lens, parents, out in runs:
        def call():
            btf.adapters(x, segs, plan, work=work)
            btf.prefix_attention(q, pk, pv, k, k, lens, parents, out=out, work=work_p)
        call()
        want.append((segs[0].y.clone(), out.clone()))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
    for order in ((0, 1, 0), (1, 1, 0, 1)):
        work.fill_(255), work_p.fill_(255)
        for r in runs:
            r[1][0].y.zero_(), r[7].zero_()
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        for r, (y, o) in zip(runs, want):
            assert torch.equal(r[1][0].y, y) and torch.equal(r[7], o)


@pytest.mark.parametrize("short", [True, False])
def test_autograd_learns_what_is_written(cuda, btf, monkeypatch, short):
    if not short:
        monkeypatch.setattr(btf, "_calls", None)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    x, a, b = torch.randn(4, 64, device=cuda), torch.randn(2, 8, 64, device=cuda).half(), torch.randn(2, 24, 8, device=cuda).half()
    plan = btf.AdapterPlan(i32(0, 1, -1, 0), 2)
    q, k = (torch.randn(*s, device=cuda).half() for s in ((1, 2, 4, 64), (1, 9, 2, 64)))
    table, pos = btf.RopeTable(64, sections=[16, 16]), i32(3, 4).expand(2, 2)
    h = torch.randn(2, 3, 64, device=cuda)

    def each(want):
        w = lambda t: t.clone().requires_grad_() if want else t  # noqa: E731
        yield lambda: btf.adapters(w(x), [btf.AdapterSeg(a, b)], plan)
        yield lambda: btf.adapters(x, [btf.AdapterSeg(a, w(b))], plan)
        yield lambda: btf.adapters(x, [btf.AdapterSeg(a, b, base=w(torch.zeros(4, 24, device=cuda)))], plan)
        yield lambda: btf.prefix_attention(q, w(k[0]), k[0], k, k, i32(7), i32(-1, 0)[None])
        yield lambda: btf.prefix_attention(w(q), k[0], k[0], k, k, i32(7), i32(-1, 0)[None])
        yield lambda: btf.rope([btf.RopeSeg(h, w(torch.zeros(2, 3, 64, device=cuda)))], table, pos)

    for fn in each(True):
        with pytest.raises(RuntimeError, match="gradient"):
            fn()
    with torch.no_grad():
        for fn in each(True):
            fn()
    with torch.inference_mode():
        for fn in each(False):
            fn()
    y, out, z = torch.zeros(4, 24, device=cuda), torch.zeros_like(q), torch.zeros(2, 3, 64, device=cuda)
    versions = [t._version for t in (y, out, z, k, a)]
    btf.adapters(x, [btf.AdapterSeg(a, b, y)], plan)
    btf.prefix_attention(q, k[0], k[0], k, k, i32(7), i32(-1, 0)[None], out=out)
    btf.rope([btf.RopeSeg(h, z)], table, pos)
    assert [t._version for t in (y, out, z, k, a)] == [v + 1 for v in versions[:3]] + versions[3:]
