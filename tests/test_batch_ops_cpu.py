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
