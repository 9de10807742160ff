"""btf_adapters with one row, one adapter or one output, whose strides do not matter: the C ABI's checks on the CPU (each call is
refused for its missing workspace, before anything is launched), results on the GPU."""
import pytest
import torch

from test_batch_ops_cpu import _adapters

ONE = [dict(T=1, x_row=1), dict(T=1, x_row=0), dict(T=1, x_row=-3), dict(n_adapters=1, seg=dict(a_adapter=3, b_adapter=5)),
       dict(seg=dict(N=1, b_row=7)), dict(T=1, seg=dict(y_row=0, base_row=-1)), dict(T=1, x_type=1, x_row=9)]


@pytest.mark.parametrize("kw", ONE, ids=str)
def test_strides_of_one_entry_are_not_refused(btf, kw):
    assert _adapters(btf, work=None, **kw) != 0
    message = btf.lib().btf_last_error()
    assert b"stride" not in message and b"rows" not in message, message


@pytest.mark.parametrize("kw", [dict(x_row=1), dict(n_adapters=2, seg=dict(a_adapter=3)), dict(seg=dict(b_row=7)),
                                dict(T=1, seg=dict(a_row=7)), dict(seg=dict(base_row=-1))], ids=str)
def test_strides_that_matter_are(btf, kw):
    assert _adapters(btf, work=None, **kw) == 1
    assert b"stride" in btf.lib().btf_last_error() or b"rows" in btf.lib().btf_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("direct", [True, False])
def test_results_with_odd_strides_of_one_entry(cuda, btf, direct):
    from test_adapters_gpu import F16, F32, _check, _inputs, _reference

    kw = {} if direct else dict(stream=torch.cuda.current_stream())  # the ordinary calls' way, and the mirror's
    K, R = 64, 8
    for T, n, N in ((1, 3, 20), (1, 1, 1), (5, 1, 20), (600, 1, 20), (5, 2, 1), (600, 2, 1)):
        x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, F16, F32, T + N)
        index = torch.arange(T, dtype=torch.int32, device=cuda) % n
        want = _reference(x, a, b, base, index, None, None, F32)
        if T == 1:
            x = x.view(K, 1).t()
            assert x.stride(0) == 1
        if n == 1:
            a, b = a.as_strided((1, R, K), (3, K, 1)), b.as_strided((1, N, R), (5, R, 1))
        if N == 1:
            b = b.as_strided((n, 1, R), (b.stride(0), 7, 1))
        _check(btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], btf.AdapterPlan(index, n), **kw)[0], want)
    assert btf.device_error() == 0
