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
