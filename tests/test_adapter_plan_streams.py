"""An AdapterPlan's memory belongs to the stream that it is made on: on the CPU by a stand-in for the launch, on the GPU by
plans made and used on a side stream while the current one takes and gives back blocks of the same size."""
import types

import pytest
import torch


def test_the_plan_is_allocated_where_it_is_launched(btf, monkeypatch):
    inside, allocated = [], []
    real_lib, real_empty = btf.lib(), torch.empty

    def launch(dev, stream, fn, args):
        inside.append(stream)
        try:
            return fn(None, args)
        finally:
            inside.pop()

    def empty(*args, **kw):
        allocated.append(list(inside))
        return real_empty(*args, **kw)

    fake = types.SimpleNamespace(btf_adapter_plan_bytes=real_lib.btf_adapter_plan_bytes, btf_adapter_plan=lambda *a: 0)
    monkeypatch.setattr(btf, "lib", lambda: fake)
    monkeypatch.setattr(btf, "_launch", launch)
    monkeypatch.setattr(btf, "_cuda_device", lambda what, t: t.device)
    monkeypatch.setattr(torch, "empty", empty)
    plan = btf.AdapterPlan(torch.zeros(20, dtype=torch.int32), 3, stream="side")
    assert allocated == [["side"]] and plan.plan.nbytes == real_lib.btf_adapter_plan_bytes(20, 3)
    plan.update(torch.ones(20, dtype=torch.int32), stream="other")  # into the same memory
    assert allocated == [["side"]]
    for index in (torch.zeros(19, dtype=torch.int32), torch.zeros(20), None):
        with pytest.raises((RuntimeError, AttributeError)):
            plan.update(index)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [48, 1500])
def test_plans_on_a_side_stream(cuda, btf, T):
    """Each plan is made and used on the side stream and dropped, while the current stream fills blocks of its size."""
    from test_adapters_gpu import F16, F32, _check, _index, _inputs, _reference

    n, K, R, N = 5, 256, 16, 96
    x, (a,), (b,), (base,) = _inputs(cuda, T, n, K, R, [N], F32, F16, F32, 1)
    index = [_index(cuda, T, n, seed) for seed in range(12)]
    side, busy = torch.cuda.Stream(), torch.zeros(4096, 4096, device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    size = btf.lib().btf_adapter_plan_bytes(T, n)
    out = []
    for i in index:
        busy @ busy  # the current stream is behind, so that what it fills below is filled while the side stream runs
        for _ in range(4):
            torch.empty(size, dtype=torch.uint8, device=cuda).fill_(255)
        plan = btf.AdapterPlan(i, n, stream=side)
        where = [s["stream"] for s in torch.cuda.memory_snapshot()
                 if s["address"] <= plan.plan.data_ptr() < s["address"] + s["total_size"]]
        assert where == [side.cuda_stream]
        out.append(btf.adapters(x, [btf.AdapterSeg(a, b, base=base)], plan, stream=side)[0])
        del plan
        torch.empty(size, dtype=torch.uint8, device=cuda).fill_(255)
    torch.cuda.synchronize()
    assert btf.device_error() == 0
    for i, y in zip(index, out):
        _check(y, _reference(x, a, b, base, i, None, None, F32))
