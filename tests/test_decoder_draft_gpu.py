"""GPU tests of the decoder's drawn tokens and drafted trees (btf_decoder_step_sampled, _run_sampled, _verify,
_accept) on seeded synthetic models: both layer kinds, every node of a tree against stepping along its path.

A draft and a step compute the same in two orders (rotary angles in 64 bits and in fp32 steps, fp16 attention outputs and
probabilities: 2^-11). Where there is no attention layer the difference is that of the batched products, rel-RMS 1e-5
as between prompt chunks and steps. After one, a Q8 code may fall to either side: an activation whose two values
differ by delta gets codes one apart with probability delta / d, d = amax / 127 its block's step, so a difference of r
relative becomes sqrt(d delta): r' = sqrt(c r / 127), with amax = c times the block's rms, c <= 3 for 32 Gaussian values.
  - With one attention layer, the last one: r = 2 * 2^-11.5 of its outputs, then the products with wo, gate and up, down
    and the head: 0.0028 -> 0.0081; the SwiGLU product of two such has sqrt 2 of that, 0.016 -> 0.019: 2e-2, the
    decoder's own tolerance between two implementations.
  - Whatever r begins with, repeated products settle at r = c / 127 = 0.024, a SwiGLU product of two branches at sqrt 2
    of that, 0.034; the residual's difference and the head's own rounding add up to sqrt 2 * 0.034 < 0.05.
A wrong parent, row or state changes logits by their own size."""
import numpy as np
import pytest

from conftest import rel_rms

pytestmark = pytest.mark.gpu

SMALL = dict(n_layer=8, n_embd=512, n_ff=1024, n_vocab=1000, n_head=4, n_head_kv=2, head_dim=128, n_rot=64,
             d_state=64, n_group=2, dt_rank=4, conv_kernel=4, hadamard_block=128, rope_base=1e7, rms_eps=1e-6)
DIMS = {
    "small": SMALL,
    "model heads": dict(n_layer=4, n_embd=1024, n_ff=2048, n_vocab=3001, n_head=4, n_head_kv=1, head_dim=256, n_rot=64,
                        d_state=128, n_group=2, dt_rank=8, conv_kernel=4, hadamard_block=1024, rope_base=1e7,
                        rms_eps=1e-6),
    "recurrent layers": dict(SMALL, n_layer=3),
    "one attention layer": dict(SMALL, n_layer=4),
}


def _tol(dims):
    return {3: 1e-5, 4: 2e-2}.get(dims["n_layer"], 5e-2)


PROMPT = [7, 3, 500, 42, 9, 11]


@pytest.fixture(params=list(DIMS))
def dims(request):
    return DIMS[request.param]


def _open(btf, dims, **kw):
    return btf.Decoder(dims=dims, seed=5, n_ctx=64, **kw)


def _along(btf, dims, tokens):
    """Logits after each of `tokens` behind the prompt, one step at a time."""
    with _open(btf, dims) as d:
        d.prefill(PROMPT)
        return [d.step(t, logits=True)[1] for t in tokens]


def test_chain_equals_steps(cuda, btf, dims):
    draft = [5, 17, 256, 3, 99, 1, 640, 2]
    want = _along(btf, dims, draft + [77, 78])
    with _open(btf, dims) as d:
        d.prefill(PROMPT)
        nxt, lg = d.verify(draft, list(range(-1, 7)), logits=True)
        for j in range(8):
            assert rel_rms(lg[j], want[j]) <= _tol(dims), (j, rel_rms(lg[j], want[j]))
            assert nxt[j] == int(np.argmax(lg[j]))
        assert d.info()["pos"] == len(PROMPT)
        d.accept(7)
        assert d.info()["pos"] == len(PROMPT) + 8
        for j, t in enumerate((77, 78)):  # decoding goes on from the draft's states and rows
            assert rel_rms(d.step(t, logits=True)[1], want[8 + j]) <= _tol(dims)
    assert btf.device_error() == 0


def test_every_path_of_a_tree(cuda, btf, dims):
    tokens, parents = [5, 17, 18, 19, 256, 257, 3, 640], [-1, 0, 0, 1, 1, 4, -1, 6]
    with _open(btf, dims) as d:
        d.prefill(PROMPT)
        _, lg = d.verify(tokens, parents, logits=True)
        _, again = d.verify(tokens, parents, logits=True)
        assert np.array_equal(lg, again)  # a draft leaves nothing behind
    for node in range(8):
        path, j = [], node
        while j >= 0:
            path.insert(0, j)
            j = parents[j]
        want = _along(btf, dims, [tokens[j] for j in path] + [33])
        assert rel_rms(lg[node], want[-2]) <= _tol(dims), (node, rel_rms(lg[node], want[-2]))
        with _open(btf, dims) as d:
            d.prefill(PROMPT)
            nxt, _ = d.verify(tokens, parents)
            d.accept(node)
            assert d.info()["pos"] == len(PROMPT) + len(path)
            got = d.step(33, logits=True)[1]
            assert rel_rms(got, want[-1]) <= _tol(dims), (node, rel_rms(got, want[-1]))


def test_a_dropped_draft_changes_nothing(cuda, btf, dims):
    with _open(btf, dims) as d, _open(btf, dims) as plain:
        for x in (d, plain):
            x.prefill(PROMPT)
        d.verify([1, 2, 3], [-1, 0, 0])
        for t in (5, 6):
            assert np.array_equal(d.step(t, logits=True)[1], plain.step(t, logits=True)[1])
            d.verify([t, 2], [-1, -1])


def test_accepted_draft_feeds_run(cuda, btf, dims):
    """Greedy decoding by drafts of the model's own tokens gives what run() gives."""
    import torch

    with _open(btf, dims) as a, _open(btf, dims) as b:
        first, _ = a.prefill(PROMPT)
        b.prefill(PROMPT)
        chain = [first]
        for _ in range(4):
            chain.append(a.step(chain[-1])[0])
        nxt, _ = b.verify(chain[:4], [-1, 0, 1, 2])
        assert nxt.tolist() == chain[1:]
        b.accept(3)
        a.run(3)
        b.run(3)
        torch.cuda.synchronize()
        assert a.info()["pos"] == b.info()["pos"] == len(PROMPT) + 7


@pytest.mark.parametrize("graph", [True, False])
def test_sampled_steps(cuda, btf, dims, graph):
    """The drawn token is btf_sample's of the same logits; temperature 0 is the greedy step; run_sampled draws as
    steps do."""
    import torch

    params = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    us = [0.05, 0.5, 0.93, 0.31, 0.77]
    f = lambda v, t=torch.float32: torch.tensor([v], dtype=t, device=cuda)  # noqa: E731
    with _open(btf, dims, cuda_graph=graph) as d, _open(btf, dims, cuda_graph=graph) as plain:
        t, toks = PROMPT[0], []
        for u in us:
            nxt, lp, lg = d.step_sampled(t, u, logits=True, **params)
            g, lg2 = plain.step(t, logits=True)
            assert np.array_equal(lg, lg2)
            tok, lps = btf.sample(torch.from_numpy(lg)[None].to(cuda), f(u), f(0.9), f(40, torch.int32), f(0.95), f(0.01))
            assert nxt == int(tok[0]) and lp == float(lps[0])
            assert g == int(np.argmax(lg))
            toks.append(nxt)
            t = nxt
        d.reset()
        d.step_sampled(PROMPT[0], us[0], **params)
        d.run_sampled(us[1:], **params)
        torch.cuda.synchronize()
        assert d.info()["pos"] == len(us) and d.stats()["steps"] == 2 * len(us)
        # the last token run_sampled drew is the one the next device step takes
        d.run(1)
        plain.step(toks[-1])
        lg = _device_logits(btf, d)
        assert np.array_equal(lg, plain.step(0, logits=True)[1]) is False  # (another token's logits)
        plain.reset()
        for x in [PROMPT[0]] + toks[:-1]:
            plain.step(x)
        assert np.array_equal(lg, plain.step(toks[-1], logits=True)[1])
        assert d.step_sampled(3, 0.4, temperature=0.0)[0] == plain.step(3)[0]


def _device_logits(btf, d):
    import torch

    torch.cuda.synchronize()
    i = d.info()

    class Held:
        __cuda_array_interface__ = dict(shape=(i["n_vocab"],), typestr="<f4", data=(i["logits"], False), version=3)

    return torch.as_tensor(Held(), device="cuda").cpu().numpy()


def test_sampled_drafts(cuda, btf, dims):
    import torch

    us = [0.2, 0.5, 0.9]
    with _open(btf, dims) as d:
        d.prefill(PROMPT)
        nxt, lg = d.verify([4, 5, 6], [-1, 0, 0], sampling=dict(temperature=1.3, top_p=0.9), us=us, logits=True)
        n = len(us)
        tok, _ = btf.sample(torch.from_numpy(lg).to(cuda), torch.tensor(us, device=cuda),
                            torch.full((n,), 1.3, device=cuda), top_p=torch.full((n,), 0.9, device=cuda))
        assert nxt.tolist() == tok.tolist()


def test_refusals(cuda, btf):
    dims = DIMS["small"]
    with btf.Decoder(dims=dims, seed=1, n_ctx=10) as d:
        before = d.info()["device_bytes"]
        bad = [([1] * 9, [-1] * 9), ([], []), ([1, 2], [-1, 1]), ([1, 2], [-2, 0]), ([1000], [-1]), ([-1], [-1])]
        for t, p in bad:
            with pytest.raises(RuntimeError):
                d.verify(t, p)
        with pytest.raises(RuntimeError):
            d.verify([1, 2], [-1])
        with pytest.raises(RuntimeError):
            d.verify([1], [-1], sampling=dict(temperature=1.0))
        with pytest.raises(RuntimeError):
            d.accept(0)
        assert d.info()["device_bytes"] == before  # nothing was allocated for them
        d.verify([1, 2], [-1, 0])
        assert d.info()["device_bytes"] > before
        for node in (-1, 2):
            with pytest.raises(RuntimeError):
                d.accept(node)
        d.accept(1)
        with pytest.raises(RuntimeError):
            d.accept(0)  # taken already
        d.verify([1], [-1])
        d.step(1)
        with pytest.raises(RuntimeError):
            d.accept(0)  # dropped by the step
        d.verify([1] * 7, [-1] * 7)
        with pytest.raises(RuntimeError):
            d.verify([1] * 8, [-1] * 8)  # 3 + 8 > 10
        with pytest.raises(RuntimeError):
            d.step_sampled(1000, 0.5)
        d.reset()
        with pytest.raises(RuntimeError):
            d.accept(0)


def test_a_long_drawn_run(cuda, btf):
    """More steps than random numbers are copied at a time: the run ends where as many drawn steps end."""
    dims = dict(SMALL, n_layer=3)
    us = np.random.default_rng(8).random(4100, dtype=np.float32)
    params = dict(temperature=1.1, top_k=30)
    with btf.Decoder(dims=dims, seed=5, n_ctx=4200) as d, btf.Decoder(dims=dims, seed=5, n_ctx=4200) as steps:
        t = d.step_sampled(3, 0.5, **params)[0]
        d.run_sampled(us, **params)
        assert t == steps.step_sampled(3, 0.5, **params)[0]
        for u in us:
            t = steps.step_sampled(t, float(u), **params)[0]
        assert np.array_equal(_device_logits(btf, d), _device_logits(btf, steps))
        assert d.info()["pos"] == steps.info()["pos"] == 4101
        with pytest.raises(RuntimeError):
            d.run_sampled(us[:100], **params)  # past the context
    assert btf.device_error() == 0


def test_a_drawn_run_copies_its_numbers(cuda, btf):
    """The random numbers belong to the caller again when run_sampled returns, in pinned memory too."""
    import torch

    dims = dict(SMALL, n_layer=3)
    params = dict(temperature=1.1, top_k=30)
    us = torch.rand(4300, generator=torch.Generator().manual_seed(8)).pin_memory()
    kept = us.numpy().copy()
    with btf.Decoder(dims=dims, seed=5, n_ctx=4400) as d, btf.Decoder(dims=dims, seed=5, n_ctx=4400) as other:
        for x, u in ((d, us.numpy()), (other, kept)):
            x.step_sampled(3, 0.5, **params)
            x.run_sampled(u, **params)
            us.zero_()
        assert np.array_equal(_device_logits(btf, d), _device_logits(btf, other))
    assert btf.device_error() == 0


TREE = ([5, 17, 18, 19, 256, 257, 3, 640], [-1, 0, 0, 1, 1, 4, -1, 6])


@pytest.mark.parametrize("node", [0, 2, 4, 7])
def test_run_continues_from_the_accepted_node(cuda, btf, dims, node):
    """btf_decoder_run takes the token after the accepted node of a branching tree, whichever node that is."""
    tokens, parents = TREE
    path, j = [], node
    while j >= 0:
        path.insert(0, tokens[j])
        j = parents[j]
    with _open(btf, dims) as d:
        d.prefill(PROMPT)
        nxt, _ = d.verify(tokens, parents)
        assert len(set(nxt.tolist())) > 1
        d.accept(node)
        d.run(1)
        got = _device_logits(btf, d)
        assert d.info()["pos"] == len(PROMPT) + len(path) + 1
    want = _along(btf, dims, path + [int(nxt[node])])[-1]
    assert rel_rms(got, want) <= _tol(dims), rel_rms(got, want)
    if dims["n_layer"] == 3:  # to 1e-5: a token from another node would be seen, and so is a run of several steps
        with _open(btf, dims) as a, _open(btf, dims) as b:
            a.prefill(PROMPT)
            b.prefill(PROMPT)
            for t in path:
                a.step(t)
            b.verify(tokens, parents)
            b.accept(node)
            a.run(3)
            b.run(3)
            la, lb = _device_logits(btf, a), _device_logits(btf, b)
            assert rel_rms(lb, la) <= _tol(dims), rel_rms(lb, la)


@pytest.mark.parametrize("node", [0, 3, 7])
def test_accepted_node_has_the_decoders_logits(cuda, btf, dims, node):
    """After an acceptance the decoder's logits are those behind its last token, as after a step."""
    with _open(btf, dims) as d:
        d.prefill(PROMPT)
        _, lg = d.verify(*TREE, logits=True)
        d.accept(node)
        assert np.array_equal(_device_logits(btf, d), lg[node])


def test_a_draft_that_found_no_memory_leaves_none_behind(cuda, btf):
    """A decoder whose first draft fails for want of device memory holds after the next one what it would have held."""
    import ctypes

    dims = DIMS["model heads"]  # a draft allocates 13 MB of states, the attention's small buffers, its workspace of 39 MB

    def opened():
        return btf.Decoder(dims=dims, seed=5, n_ctx=9600)

    def take(size, held):
        p = ctypes.c_void_p()
        if btf.lib().btf_alloc(size, ctypes.byref(p)):
            return False
        held.append(p)
        return True

    def give(held):
        while held:
            assert btf.lib().btf_free(held.pop()) == 0

    with opened() as plain:
        plain.verify([1], [-1])
        want = plain.info()["device_bytes"]
    with opened() as d:
        spare, rest, size = [], [], 1 << 38
        try:
            for _ in range(12):
                assert take(2 << 20, spare)
            while size >= 2 << 20:
                if not take(size, rest):
                    size //= 2
            give(spare)  # 24 MB, and less than 2 beside them
            with pytest.raises(RuntimeError, match="memory"):
                d.verify([1], [-1])
            # the workspace, 148 ranges x 2 x 128 rows x (256 + 2) floats, is what was not to be had
            assert want - d.info()["device_bytes"] > 39 * 10 ** 6
        finally:
            give(spare)
            give(rest)
        d.verify([1], [-1])
        assert d.info()["device_bytes"] == want
    assert btf.device_error() == 0


@pytest.mark.parametrize("n_layer", [4, 8])
def test_a_draft_rounds_q_whatever_a_step_does(cuda, btf, n_layer):
    """The tree attention's q is fp16: a decoder opened with round_q_f16 = 0 checks the same tree to the same bits, and
    to the bounds above against its own steps, whose q is fp32 (2^-12 of it, beside the 2 * 2^-11.5 there)."""
    dims = dict(SMALL, n_layer=n_layer)
    with _open(btf, dims) as a, _open(btf, dims, round_q_f16=False) as b, _open(btf, dims, round_q_f16=False) as steps:
        got = []
        for d in (a, b):
            for t in PROMPT[:1]:  # one token: attention to itself alone, the same states and rows in both
                d.step(t)
            got.append(d.verify(*TREE, logits=True)[1])
        assert np.array_equal(*got)
        steps.step(PROMPT[0])
        for j, t in ((0, 5), (1, 17), (3, 19)):
            want = steps.step(t, logits=True)[1]
            assert rel_rms(got[1][j], want) <= _tol(dims), (j, rel_rms(got[1][j], want))
