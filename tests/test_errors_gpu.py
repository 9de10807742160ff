"""A call that failed has reported its error: the calls after it are not told of it again."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _fail(btf):
    p = ctypes.c_void_p()
    assert btf.lib().btf_alloc(1 << 60, ctypes.byref(p)) == 2  # BTF_ERR_CUDA: no such device has that much memory
    assert b"memory" in btf.lib().btf_last_error()


def test_a_failed_allocation_does_not_fail_the_next_launch(cuda, btf):
    import torch

    x = torch.randn(2, 256, device=cuda)
    act = btf.quant_q8(x)
    torch.cuda.synchronize()
    q = act.q.cpu()
    _fail(btf)
    act = btf.quant_q8(x)
    torch.cuda.synchronize()
    assert torch.equal(act.q.cpu(), q)


@pytest.mark.parametrize("graph", [True, False])
def test_nor_a_decoders_step(cuda, btf, graph):
    dims = dict(n_layer=4, n_embd=512, n_ff=1024, n_vocab=1000, n_head=4, n_head_kv=2, head_dim=128, n_rot=64, d_state=64,
                n_group=2, dt_rank=4, conv_kernel=4, hadamard_block=128, rope_base=1e7, rms_eps=1e-6)
    with btf.Decoder(dims=dims, seed=5, n_ctx=64, cuda_graph=graph) as d, \
            btf.Decoder(dims=dims, seed=5, n_ctx=64, cuda_graph=graph) as plain:
        for t in (3, 4):
            _fail(btf)
            assert np.array_equal(d.step(t, logits=True)[1], plain.step(t, logits=True)[1])
        _fail(btf)
        a = d.verify([5, 6], [-1, 0], logits=True)[1]
        assert np.array_equal(a, plain.verify([5, 6], [-1, 0], logits=True)[1])
