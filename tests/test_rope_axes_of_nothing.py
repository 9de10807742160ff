"""A table of rotary positions with several axes and no pair at all is refused, whatever its layout, as one of one axis is."""
import ctypes

import pytest


@pytest.mark.parametrize("axes", ["split", "turns", "own"])
@pytest.mark.parametrize("sections", [[0], [0, 0, 0]])
def test_no_pair_is_refused(btf, axes, sections):
    with pytest.raises(RuntimeError):
        btf.RopeTable(0, sections=sections, axes=axes, device=None)


def test_what_it_refuses_does_not_depend_on_the_pairs(btf):
    """The C call with frequencies of its own for every axis: the base and the scaling are looked at whatever the sections."""
    out = (ctypes.c_double * 4)(), (ctypes.c_uint8 * 4)(), ctypes.c_float(7)
    for kw in (dict(base=0.5), dict(scaling=9), dict(scaling=1, factor=0.5), dict(scaling=3, factor=2.0)):
        cfg = btf.RopeCfgC(**dict(dict(n_rot=0, scaling=0, base=1e4, factor=1.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=0), **kw))
        assert btf.lib().btf_rope_axes_table(ctypes.byref(cfg), (ctypes.c_int * 2)(0, 0), 2, 2, out[0], out[1],
                                             ctypes.byref(out[2])) == 1
