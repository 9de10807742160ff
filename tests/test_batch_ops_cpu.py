"""Host side of the operators for many requests at once: the table of rotary positions with several axes against its
formulas, and the argument checks of the C ABI. Nothing is launched: every refused call returns before it looks for a
device."""
import ctypes

import numpy as np
import pytest

from test_new_token_ops_cpu import P, _freqs


# ---------------------------------------------------------------- rotary positions with several axes
@pytest.mark.parametrize("sections,axes,want", [
    ([3, 2, 1], "split", [0, 0, 0, 1, 1, 2]), ([3, 2, 1], "own", [0, 0, 0, 1, 1, 2]),
    ([3, 2, 1], "turns", [0, 1, 2, 0, 1, 0]), ([1, 4], "turns", [0, 1, 1, 1, 1]), ([0, 2, 0, 1], "turns", [1, 3, 1]),
    ([0, 2, 0, 1], "split", [1, 1, 3]), ([5], "turns", [0] * 5),
])
def test_axes_of_the_pairs(btf, sections, axes, want):
    t = btf.RopeTable(2 * sum(sections), sections=sections, axes=axes, device=None)
    assert t.axis_host.tolist() == want and t.n_axes == len(sections)


@pytest.mark.parametrize("kw", [{}, dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=2.0),
                                dict(scaling="yarn", factor=8.0, orig_ctx=4096)])
def test_axes_table_follows_its_formulas(btf, kw):
    sections = [20, 12, 32]
    args = (kw.get("scaling", "none"), kw.get("factor", 1.0), kw.get("orig_ctx", 0))
    one = btf.RopeTable(128, base=1e6, device=None, **kw)
    for axes in ("split", "turns"):
        t = btf.RopeTable(128, base=1e6, sections=sections, axes=axes, device=None, **kw)
        assert np.array_equal(t.host, one.host) and t.mscale == one.mscale
    t = btf.RopeTable(128, base=1e6, sections=sections, axes="own", device=None, **kw)
    want = np.concatenate([_freqs(2 * s, 1e6, *args) for s in sections])
    # as the table of one axis: x ln b < 17, so 17 * 2^-53 and two roundings
    np.testing.assert_allclose(t.host * 2 * np.pi, want, rtol=24 * 2.0 ** -53)
    assert t.mscale == one.mscale


@pytest.mark.parametrize("n_rot,sections,kw", [
    (64, [16, 15], {}), (64, [32, 1], {}), (64, [40, -8], {}), (64, [], {}), (64, [8, 8, 8, 4, 4], {}), (0, [0], {}),
    (64, [32], dict(axes="mixed")), (64, [31, 1], dict(axes="own", scaling="ntk", factor=2.0)), (1026, [513], {}),
    (64, [16, 16], dict(base=1.0)), (64, [2 ** 30, 2 ** 30, 2 ** 30, 32], {}),
])
def test_axes_table_refuses(btf, n_rot, sections, kw):
    with pytest.raises(RuntimeError):
        btf.RopeTable(n_rot, sections=sections, device=None, **kw)


def _axes(btf, seg=None, T=2, D=64, R=64, turns=P, axis=P, n_axes=3, pos=P, stride=2):
    base = dict(x=P, y=P + 1024, x_type=0, y_type=0, heads=1, rotate=1, x_token=64, x_head=64, y_token=64, y_head=64,
                normw=None, rows=None, n_rows=0)
    base.update(seg or {})
    return btf.lib().btf_rope_axes((btf.RopeSegC * 1)(btf.RopeSegC(**base)), 1, T, D, R, turns, axis, n_axes, 1.0, 0, 0,
                                   1e-6, pos, stride, None)


@pytest.mark.parametrize("kw", [dict(n_axes=0), dict(n_axes=5), dict(axis=None), dict(pos=None), dict(turns=None),
                                dict(stride=-1), dict(T=-1), dict(R=66), dict(R=63), dict(seg=dict(x=None)),
                                dict(seg=dict(y_token=0))])
def test_rope_axes_refuses(btf, kw):
    assert _axes(btf, **kw) == 1, kw
    assert btf.lib().btf_last_error()


def test_rope_axes_of_nothing_is_done(btf):
    assert _axes(btf, T=0, axis=None) == 0 and _axes(btf, seg=dict(heads=0)) == 0


# ---------------------------------------------------------------- low-rank adapters
def _adapters(btf, seg=None, **kw):
    s = dict(a=P, a_adapter=8 * 64, a_row=64, b=P, b_adapter=16 * 8, b_row=8, N=16, base=P, base_row=16, y=P + 1024, y_row=16)
    s.update(seg or {})
    a = dict(x=P, x_row=64, x_type=0, w_type=1, y_type=0, T=4, K=64, R=8, n_adapters=2, nseg=1, ranks=None, scales=None,
             plan=P, plan_bytes=1 << 40, work=P, work_bytes=1 << 40)
    a.update(kw)
    args = btf.AdaptersArgsC(**a)
    for i in range(3):
        args.segs[i] = btf.AdapterSegC(**s)
    return btf.lib().btf_adapters(ctypes.byref(args), None)


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(T=(1 << 20) + 1), dict(K=0), dict(K=60), dict(R=0), dict(R=12), dict(R=136), dict(n_adapters=0),
    dict(n_adapters=1025), dict(nseg=0), dict(nseg=4), dict(w_type=0), dict(w_type=3), dict(x_type=2), dict(y_type=2),
    dict(y_type=3), dict(x=None), dict(x=P + 8), dict(x_row=62), dict(x_row=-64), dict(x_type=1, x_row=68), dict(plan=None),
    dict(plan=P + 8), dict(plan_bytes=64),
    dict(seg=dict(a=None)), dict(seg=dict(b=None)), dict(seg=dict(y=None)), dict(seg=dict(a=P + 8)), dict(seg=dict(b=P + 4)),
    dict(seg=dict(a_row=60)), dict(seg=dict(b_row=-8)), dict(seg=dict(a_adapter=4)), dict(seg=dict(N=0)), dict(seg=dict(y=P + 2)),
    dict(seg=dict(base=P + 1)), dict(seg=dict(y_row=15)), dict(seg=dict(base_row=-1)), dict(seg=dict(base=P + 1024, base_row=32)),
])
def test_adapters_refuses(btf, kw):
    assert _adapters(btf, **kw) == 1, kw
    assert btf.lib().btf_last_error()


def test_adapters_of_no_row_are_done_and_plans_refuse(btf):
    L = btf.lib()
    assert _adapters(btf, T=0) == 0
    assert L.btf_adapters(None, None) == 1
    for T, n in ((-1, 1), (1, 0), (1, 1025), ((1 << 20) + 1, 1)):
        assert L.btf_adapter_plan_bytes(T, n) == -1 and L.btf_adapter_plan(P, T, n, P, 1 << 40, None) == 1
    size = L.btf_adapter_plan_bytes(100, 7)
    assert size > 400
    for args in ((None, 100, 7, P, size), (P, 100, 7, None, size), (P, 100, 7, P + 8, size), (P, 100, 7, P, size - 1)):
        assert L.btf_adapter_plan(*args, None) == 1
    assert L.btf_adapters_work(4, 60, 8, 1, 2) == -1


# ---------------------------------------------------------------- attention behind shared rows
def _prefix(btf, tree=None, **kw):
    a = dict(q=P, q_batch=1024, q_node=512, q_head=64, k=P, v=P, kv_batch=4096, kv_row=64, kv_head=64, o=P, o_batch=1024,
             o_node=512, o_head=64, type=1, B=1, n=2, H=8, HK=1, D=64, n_ctx=64, lens=P, parents=P, counts=None,
             scale=0.125, work=P, work_bytes=1 << 40)
    a.update(tree or {})
    s = dict(k=P, v=P, row=64, head=64, rows=100, len=None)
    s.update(kw)
    return btf.lib().btf_prefix_attention(ctypes.byref(btf.TreeAttnC(**a)), ctypes.byref(btf.PrefixC(**s)), None)


@pytest.mark.parametrize("kw", [
    dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(row=63), dict(row=-64), dict(row=0), dict(head=4),
    dict(rows=-1), dict(rows=(1 << 30) + 1), dict(tree=dict(n=65)), dict(tree=dict(q=None)), dict(tree=dict(type=0)),
    dict(tree=dict(lens=None)), dict(tree=dict(o_head=0)), dict(tree=dict(kv_row=60)), dict(tree=dict(work=None)),
])
def test_prefix_attention_refuses(btf, kw):
    assert _prefix(btf, **kw) == 1, kw
    assert btf.lib().btf_last_error()


def test_prefix_attention_of_no_sequence_is_done(btf):
    assert _prefix(btf, tree=dict(B=0)) == 0
    assert btf.lib().btf_prefix_attention(None, None, None) == 1
    assert btf.lib().btf_prefix_attention_work(1, 65, 8, 1, 64, 64, 10) == -1
    assert btf.lib().btf_prefix_attention_work(1, 1, 8, 1, 64, 64, -1) == -1
    assert ctypes.sizeof(btf.PrefixC) == btf._PREFIX.size
