"""The operators of new tokens as they are used together: rotate the drafted tokens' q and k and append k and v to the
cache, attend over the cache and the tree, project, draw a token per node; captured in one graph and replayed as the
cache grows. Each stage is held to its formula in 64 bits on what the stage before it gave."""
import numpy as np
import pytest
import torch

from test_rope_gpu import _check as check_rope, _reference as rope_reference
from test_sample_gpu import _reference as sample_reference
from test_tree_attention_gpu import _check as check_tree, _reference as tree_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
def test_rope_attention_sampling(cuda, btf, t):
    n, H, HK, D, R, ctx, V = 9, 6, 2, 128, 64, 700, 5003
    g = torch.Generator(device="cuda").manual_seed(3)
    randn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    parents = [-1, 0, 0, 1, 1, 2, 5, 5, 7]
    depth = [0]
    for p in parents[1:]:
        depth.append(depth[p] + 1)
    kc, vc = (torch.zeros(ctx, HK, D, dtype=t, device=cuda) for _ in range(2))
    kc[:600], vc[:600] = randn(600, HK, D).to(t), randn(600, HK, D).to(t)
    kc[600:], vc[600:] = float("nan"), float("inf")  # rows that nothing has written yet
    qg, k, v = randn(n, H, 2 * D), randn(n, HK, D), randn(n, HK, D)
    qn, kn = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
    head = randn(H * D, V) * 0.05
    table = btf.RopeTable(R, base=1e6, scaling="yarn", factor=4.0, orig_ctx=512)
    par = torch.tensor([parents], dtype=torch.int32, device=cuda)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    lens, pos, rows = i32([0]), i32([0] * n), i32([0] * n)
    q16 = torch.empty(n, H, D, dtype=t, device=cuda)
    out = torch.empty(1, n, H, D, dtype=t, device=cuda)
    u, temp, topp = torch.rand(n, generator=g, device=cuda), torch.full((n,), 0.8, device=cuda), torch.full((n,), 0.9, device=cuda)
    topk = torch.full((n,), 100, dtype=torch.int32, device=cuda)
    tok, lp = torch.empty(n, dtype=torch.int32, device=cuda), torch.empty(n, device=cuda)
    work = btf.tree_attention_work(q16[None], kc[None])
    logits = torch.empty(n, V, device=cuda)

    def forward():
        btf.rope([btf.RopeSeg(qg[..., :D], q16, normw=qn), btf.RopeSeg(k, kc, normw=kn, rows=rows),
                  btf.RopeSeg(v, vc, rotate=False, rows=rows)], table, pos)
        btf.tree_attention(q16[None], kc[None], vc[None], lens, par, out=out, work=work)
        torch.matmul(out.view(n, H * D).float(), head, out=logits)
        btf.sample(logits, u, temperature=temp, top_k=topk, top_p=topp, tokens=tok, logprobs=lp)

    def place(length):
        lens.fill_(length)
        pos.copy_(i32([length + d for d in depth]))
        rows.copy_(i32([length + j for j in range(n)]))

    place(600)
    forward()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forward()
    for length in (600, 603, 0, 691):
        place(length)
        if length > 603:  # what lies before must have been written
            kc[600:length], vc[600:length] = randn(length - 600, HK, D).to(t), randn(length - 600, HK, D).to(t)
        u.copy_(torch.rand(n, generator=g, device=cuda))
        qg.copy_(randn(n, H, 2 * D))
        graph.replay()
        torch.cuda.synchronize()
        ref, size = rope_reference(qg[..., :D], table.host, table.mscale, pos.cpu(), False, normw=qn)
        check_rope(q16, ref, size, normed_D=D)
        ref, size = rope_reference(k, table.host, table.mscale, pos.cpu(), False, normw=kn)
        check_rope(kc[rows.long()], ref, size, normed_D=D)
        check_tree(out, tree_reference(q16[None].cpu(), kc[None].cpu(), vc[None].cpu(), [length], [parents], [n], D ** -0.5), t)
        x = logits.cpu().numpy()
        for j in range(n):
            want, wlp = sample_reference(x[j], np.float32(u[j].item()), np.float32(0.8), 100, np.float32(0.9))
            assert int(tok[j]) == want
            assert abs(float(lp[j]) - wlp) <= 2.0 ** -15
    assert btf.device_error() == 0


def test_short_and_long_way_of_a_call_agree(cuda, btf, monkeypatch):
    """The binding of ordinary calls does them itself, on the current stream too; what it leaves to the Python mirror
    (another type, a stream that is given, an error) ends the same way."""
    import gc

    g = torch.Generator(device=cuda).manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    T, H, HK, D, ctx = 5, 6, 2, 64, 40
    q, k, kc, w = rn(T, H, 2 * D)[..., :D], rn(T, HK, D), rn(ctx, HK, D).half(), rn(D)
    pos, rows = torch.arange(7, 7 + T, dtype=torch.int32, device=cuda), torch.arange(3, 3 + T, dtype=torch.int32, device=cuda)
    table = btf.RopeTable(32, base=1e5, scaling="linear", factor=2.0, interleaved=True)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    tq, tk, tv = rn(2, 3, H, D).half(), rn(2, ctx, HK, D).half(), rn(2, ctx, HK, D).half()
    lens, parents, counts = i32(37, 5), torch.tensor([[-1, 0, 1], [-1, -1, 0]], dtype=torch.int32, device=cuda), i32(3, 2)
    x, u = rn(4, 999), torch.rand(4, generator=g, device=cuda)
    par = dict(temperature=torch.full((4,), 0.7, device=cuda), top_k=i32(9, 0, 30, 1), top_p=torch.full((4,), 0.9, device=cuda))

    def all_calls(**kw):
        y, c = torch.zeros(T, H, D, device=cuda), kc.clone()
        btf.rope([btf.RopeSeg(q, y, normw=w), btf.RopeSeg(k, c, rows=rows, rotate=False)], table, pos, **kw)
        z = y.clone()
        btf.rope([btf.RopeSeg(z)], table, pos, True, **kw)
        o = btf.tree_attention(tq, tk, tv, lens, parents, counts, scale=0.3, **kw)
        o2 = btf.tree_attention(tq, tk, tv, lens, parents, out=torch.zeros_like(tq), **kw)
        return [y, c, z, o, o2, *btf.sample(x, u, **par, **kw), *btf.sample(x, u, **kw)]

    btf.ensure_init(0)
    assert btf._calls is not None
    taken = []
    calls = btf._calls

    class Seen:
        def __getattr__(self, name):
            def call(*a):
                r = getattr(calls, name)(*a)
                taken.append(r is not None)
                return r
            return call

    monkeypatch.setattr(btf, "_calls", Seen())
    short = all_calls()
    assert len(taken) == 6 and all(taken)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = all_calls()
    side.synchronize()
    given = all_calls(stream=side)
    side.synchronize()
    assert len(taken) == 12 and all(taken)
    for bad in (lambda: btf.rope([btf.RopeSeg(x)], table, pos), lambda: btf.sample(x.double(), u),
                lambda: btf.sample(x, u[:3]), lambda: btf.tree_attention(tq, tk.float(), tv, lens, parents),
                lambda: btf.rope([btf.RopeSeg(k.cpu())], table, pos), lambda: btf.rope([], table, pos),
                lambda: btf.tree_attention(tq, tk, tv, lens, parents, work=torch.empty(256, dtype=torch.uint8, device=cuda)),
                lambda: btf.sample(x, u, tokens=torch.zeros(4, device=cuda))):
        with pytest.raises(RuntimeError):
            bad()
    assert not any(taken[12:])
    monkeypatch.setattr(btf, "_calls", None)
    long = all_calls()
    for other in (on_side, given, long):
        for a, b in zip(short, other):
            assert a.dtype == b.dtype and torch.equal(a, b)
    # the short way keeps no reference
    monkeypatch.setattr(btf, "_calls", calls)
    torch.cuda.synchronize()
    del short, on_side, given, long, other, a, b
    gc.collect()
    before = torch.cuda.memory_allocated()
    for _ in range(50):
        all_calls()
    gc.collect()
    assert torch.cuda.memory_allocated() <= before


def test_tables_and_workspaces_that_are_too_small(cuda, btf):
    """A table with fewer frequencies than it says, and a workspace whose bytes are one byte over and over."""
    x, pos = torch.zeros(2, 1, 64, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    table = btf.RopeTable(16)
    table.n_rot = 64
    with pytest.raises(RuntimeError):
        btf.rope([btf.RopeSeg(x)], table, pos)
    q, k = torch.zeros(1, 1, 2, 64, device=cuda).half(), torch.zeros(1, 300, 2, 64, device=cuda).half()
    work = btf.tree_attention_work(q, k)
    for bad in (work[:1].expand(len(work)), torch.empty(2 * len(work), dtype=torch.uint8, device=cuda)[::2]):
        with pytest.raises(RuntimeError):
            btf.tree_attention(q, k, k, pos[:1], pos[:1, None], work=bad)


@pytest.mark.parametrize("short", [True, False])
def test_autograd_learns_what_is_written(cuda, btf, monkeypatch, short):
    """No graph is recorded: what wants a gradient is refused while one would be, and what a call writes counts as
    changed in place, so that a backward pass that saved it says so."""
    if not short:
        monkeypatch.setattr(btf, "_calls", None)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table, pos = btf.RopeTable(64), i32(3, 4)
    x = torch.randn(2, 3, 64, device=cuda, requires_grad=True)
    q, k = (torch.randn(*s, device=cuda).half() for s in ((1, 2, 4, 64), (1, 9, 2, 64)))
    logits, u = torch.randn(2, 50, device=cuda, requires_grad=True), torch.rand(2, device=cuda)

    def each(a, ka, lp):
        yield lambda: btf.rope([btf.RopeSeg(a)], table, pos)
        yield lambda: btf.tree_attention(q, ka, k, i32(7), i32(-1, 0)[None])
        yield lambda: btf.sample(logits.detach(), u, logprobs=lp)

    wants = (x * 1, k.clone().requires_grad_(), torch.zeros(2, device=cuda, requires_grad=True))
    for fn in each(*wants):
        with pytest.raises(RuntimeError, match="gradient"):
            fn()
    with torch.no_grad():
        for fn in each(*wants):
            fn()
    with torch.inference_mode():
        for fn in each(x.clone(), k.clone(), torch.zeros(2, device=cuda)):
            fn()
    tok, lp = btf.sample(logits, u)  # drawing has no gradient: values
    assert not lp.requires_grad
    h = x * 2
    y = (h * h).sum()  # saves h
    with torch.no_grad():
        btf.rope([btf.RopeSeg(h)], table, pos)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out, cache = torch.zeros_like(q), torch.zeros(5, 3, 64, device=cuda)
    tok, lp = torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(2, device=cuda)
    versions = [t._version for t in (out, cache, tok, lp, k)]
    btf.tree_attention(q, k, k, i32(7), i32(-1, 0)[None], out=out)
    btf.rope([btf.RopeSeg(x.detach(), cache, rows=i32(1, 2))], table, pos)
    btf.sample(logits, u, tokens=tok, logprobs=lp)
    assert [t._version for t in (out, cache, tok, lp, k)] == [v + 1 for v in versions[:4]] + versions[4:]


def test_segments_that_make_their_tensors_when_asked(cuda, btf):
    """Objects with a segment's attributes, each a view made anew when it is read: used to the call's end."""
    base, out = torch.randn(4, 3, 128, device=cuda), torch.zeros(4, 3, 64, device=cuda)
    table, pos = btf.RopeTable(64), torch.arange(4, dtype=torch.int32, device=cuda)

    class Seg:
        x = property(lambda self: base[..., 64:])
        y = property(lambda self: out[:])
        normw = rows = None
        rotate = True

    version = out._version
    for _ in range(20):
        btf.rope([Seg(), Seg()], table, pos)
    assert out._version == version + 40
    want = torch.empty_like(out)
    btf.rope([btf.RopeSeg(base[..., 64:], want)], table, pos)
    assert torch.equal(out, want)
