"""Eager steps without a host synchronisation between them: a step's first kernel is resident before the last one's
argmax has written the token, and must read it only after."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DIMS = dict(n_embd=512, n_ff=1024, n_vocab=1000, n_head=4, n_head_kv=2, head_dim=128, n_rot=64, d_state=64, n_group=2,
            dt_rank=4, conv_kernel=4, hadamard_block=128, rope_base=1e7, rms_eps=1e-6)


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("n_layer", [3, 4])
def test_run_equals_steps(cuda, btf, n_layer, graph):
    dims = dict(DIMS, n_layer=n_layer)
    with btf.Decoder(dims=dims, seed=5, n_ctx=64, cuda_graph=graph) as a, \
            btf.Decoder(dims=dims, seed=5, n_ctx=64, cuda_graph=graph) as b:
        t = a.step(7)[0]
        for _ in range(20):
            t = a.step(t)[0]
        want = a.step(t, logits=True)
        b.step(7)
        b.run(20)
        got = b.step(t, logits=True)
        assert np.array_equal(got[1], want[1]) and got[0] == want[0]
