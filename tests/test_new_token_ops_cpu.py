"""Host side of the rotary, tree-attention and sampling operators: the frequency
table against its formulas, and the argument checks of the C ABI. Nothing is
launched: every refused call returns before it looks for a device."""
import ctypes
import math
import os
import subprocess
import sys

import numpy as np
import pytest


# ---------------------------------------------------------------- rotary table
def _freqs(R, base, scaling="none", factor=1.0, ctx=0, fast=32.0, slow=1.0):
    i = np.arange(R // 2, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (R / (R - 2))
    f = np.exp(-2.0 * i / R * np.log(base))
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        lo, hi = (R * math.log(ctx / (2 * math.pi * b)) / (2 * math.log(base)) for b in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        f = f * (1 - r) + f / factor * r
    return f


@pytest.mark.parametrize("R,base,kw", [
    (64, 1e7, {}), (2, 1e4, {}), (128, 1e4, dict(scaling="linear", factor=4.0)), (1024, 5e5, {}),
    (80, 1e4, dict(scaling="ntk", factor=2.0)), (128, 1e6, dict(scaling="yarn", factor=8.0, orig_ctx=4096)),
    (64, 1e4, dict(scaling="yarn", factor=16.0, orig_ctx=64, beta_fast=4.0, beta_slow=4.0)),
])
def test_rope_table_follows_its_formulas(btf, R, base, kw):
    t = btf.RopeTable(R, base=base, device=None, **kw)
    want = _freqs(R, base, kw.get("scaling", "none"), kw.get("factor", 1.0), kw.get("orig_ctx", 0),
                  kw.get("beta_fast", 32.0), kw.get("beta_slow", 1.0))
    # exp(-x ln b) against pow(b, -x): x ln b < 17, so 17 * 2^-53 and two roundings
    np.testing.assert_allclose(t.host * 2 * math.pi, want, rtol=24 * 2.0 ** -53)
    assert t.mscale == pytest.approx(0.1 * math.log(kw["factor"]) + 1 if kw.get("scaling") == "yarn" else 1.0, rel=2e-7)


@pytest.mark.parametrize("kw", [
    dict(n_rot=0), dict(n_rot=3), dict(n_rot=1026), dict(n_rot=64, base=1.0), dict(n_rot=64, base=math.nan),
    dict(n_rot=64, base=math.inf), dict(n_rot=64, scaling="linear", factor=0.5),
    dict(n_rot=64, scaling="linear", factor=math.inf), dict(n_rot=2, scaling="ntk", factor=2.0),
    dict(n_rot=64, scaling="yarn", factor=2.0), dict(n_rot=64, scaling="yarn", factor=2.0, orig_ctx=512, beta_slow=0.0),
    dict(n_rot=64, scaling="yarn", factor=2.0, orig_ctx=512, beta_fast=1.0, beta_slow=2.0),
    dict(n_rot=64, scaling="dynamic"),
])
def test_rope_table_refuses(btf, kw):
    with pytest.raises(RuntimeError):
        btf.RopeTable(device=None, **kw)


# ---------------------------------------------------------------- refusals
BUF = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(BUF) + 255) // 256 * 256  # a plausible aligned address; nothing reads it


def _rope(btf, seg=None, nseg=1, T=2, D=64, R=64, turns=P, pos=P, inverse=0):
    base = dict(x=P, y=P + 1024, x_type=0, y_type=0, heads=1, rotate=1, x_token=64, x_head=64, y_token=64, y_head=64,
                normw=None, rows=None, n_rows=0)
    base.update(seg or {})
    arr = (btf.RopeSegC * 4)(*[btf.RopeSegC(**base)] * 4)
    return btf.lib().btf_rope(arr, nseg, T, D, R, turns, 1.0, 0, inverse, 1e-6, pos, None)


@pytest.mark.parametrize("kw", [
    dict(nseg=0), dict(nseg=4), dict(T=-1), dict(D=0), dict(D=1025), dict(R=63), dict(R=66), dict(R=-2),
    dict(turns=None), dict(pos=None), dict(seg=dict(x=None)), dict(seg=dict(y=None)), dict(seg=dict(x_type=3)),
    dict(seg=dict(y_type=-1)), dict(seg=dict(heads=-1)), dict(seg=dict(x=P + 2)), dict(seg=dict(y=P + 1, y_type=1)),
    dict(seg=dict(rows=P)), dict(seg=dict(normw=P), inverse=1), dict(seg=dict(y=P, y_type=1)),
    dict(seg=dict(y=P, y_token=128)), dict(seg=dict(y=P, rows=P, n_rows=2)),
])
def test_rope_refuses(btf, kw):
    assert _rope(btf, **kw) == 1, kw
    assert btf.lib().btf_last_error()


def test_rope_of_nothing_is_done(btf):
    assert _rope(btf, T=0) == 0 and _rope(btf, seg=dict(heads=0)) == 0


def _tree(btf, **kw):
    a = dict(q=P, q_batch=1024, q_node=512, q_head=64, k=P, v=P, kv_batch=4096, kv_row=64, kv_head=64, o=P, o_batch=1024,
             o_node=512, o_head=64, type=1, B=1, n=2, H=8, HK=1, D=64, n_ctx=64, lens=P, parents=P, counts=None,
             scale=0.125, work=P, work_bytes=1 << 40)
    a.update(kw)
    return btf.lib().btf_tree_attention(ctypes.byref(btf.TreeAttnC(**a)), None)


@pytest.mark.parametrize("kw", [
    dict(B=-1), dict(n=0), dict(n=65), dict(H=0), dict(HK=0), dict(HK=3), dict(D=0), dict(D=60), dict(D=264),
    dict(n_ctx=1), dict(type=0), dict(type=3), dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(lens=None),
    dict(parents=None), dict(q=P + 2), dict(k=P + 8), dict(o=P + 4), dict(kv_row=63), dict(q_head=4), dict(o_node=-8),
    dict(scale=math.nan), dict(scale=math.inf), dict(work=None), dict(work=P + 16), dict(work_bytes=0),
])
def test_tree_attention_refuses(btf, kw):
    assert _tree(btf, **kw) == 1, kw


def test_tree_attention_of_no_sequence_is_done(btf):
    assert _tree(btf, B=0) == 0


def test_tree_attention_null_arguments(btf):
    assert btf.lib().btf_tree_attention(None, None) == 1
    assert btf.lib().btf_tree_attention_work(1, 65, 8, 1, 64, 64) == -1


@pytest.mark.parametrize("kw", [dict(B=-1), dict(V=0), dict(V=524289), dict(ld=99), dict(type=3), dict(logits=None),
                                dict(u=None), dict(tokens=None), dict(logits=P + 2), dict(B=(1 << 24) + 1)])
def test_sample_refuses(btf, kw):
    a = dict(logits=P, type=0, ld=100, B=2, V=100, u=P, tokens=P)
    a.update(kw)
    if "V" in kw and kw["V"] > 100:
        a["ld"] = kw["V"]
    assert btf.lib().btf_sample(a["logits"], a["type"], a["ld"], a["B"], a["V"], a["u"], None, None, None, None,
                                a["tokens"], None, None) == 1, kw


def test_sample_of_no_row_is_done(btf):
    assert btf.lib().btf_sample(None, 0, 100, 0, 100, None, None, None, None, None, None, None, None) == 0


def test_python_wrappers_refuse_host_tensors(btf):
    import torch

    t = btf.RopeTable(64, device="cpu")
    x, p = torch.zeros(2, 1, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        btf.rope([btf.RopeSeg(x)], t, p)
    with pytest.raises(RuntimeError, match="1..3"):
        btf.rope([], t, p)
    q, k = torch.zeros(1, 2, 4, 64).half(), torch.zeros(1, 9, 2, 64).half()
    with pytest.raises(RuntimeError, match="CUDA"):
        btf.tree_attention(q, k, k, p[:1], p[None])
    with pytest.raises(RuntimeError, match="expected"):
        btf.tree_attention(q, k, k[:, :8], p[:1], p[None])
    with pytest.raises(RuntimeError, match="CUDA"):
        btf.sample(torch.zeros(2, 10), torch.zeros(2))
    with pytest.raises(RuntimeError, match="contiguous"):
        btf.sample(torch.zeros(10, 2).t(), torch.zeros(2))


def test_packed_arguments_are_the_structs(btf):
    """The wrappers fill the argument structs by struct.pack: the same bytes as the ctypes fields."""
    v = list(range(1, 14))
    v[5] = 1
    assert btf._ROPE_SEG.pack(*v) == bytes(btf.RopeSegC(*v))
    v = list(range(1, 27))
    assert len(v) == len(btf.TreeAttnC._fields_)
    a, b = btf._TREE_ATTN.pack(*v), btf.TreeAttnC(*v)
    assert btf.TreeAttnC.from_buffer_copy(a).work_bytes == 26 and len(a) == ctypes.sizeof(b)
    for name, _ in btf.TreeAttnC._fields_:
        assert getattr(btf.TreeAttnC.from_buffer_copy(a), name) == getattr(b, name), name


def test_rope_refuses_more_tokens_than_it_counts(btf):
    assert _rope(btf, T=(1 << 30) + 1) == 1


def test_cpp_mirror_of_drafts_compiles():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-I", os.path.join(root, "include"),
                        "-I", "/usr/local/cuda/include", os.path.join(root, "tests", "shim_draft.cpp")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_binding_leaves_what_is_not_ordinary(btf):
    """Without CUDA tensors the binding of ordinary calls declines, whatever it is given."""
    torch = pytest.importorskip("torch")
    if not os.path.exists(os.path.join(btf.HERE, "btf_b200_calls.so")):
        pytest.skip("built without torch")
    btf.lib()
    btf._bind_calls()
    x, v = torch.zeros(2, 3, 8), torch.zeros(2, dtype=torch.int32)
    table = btf.RopeTable(8, device=None)
    for segs in ([], [btf.RopeSeg(x)], [btf.RopeSeg(None)], [None], (btf.RopeSeg(x),), [btf.RopeSeg(x)] * 4, None):
        assert btf._calls.rope(segs, table, v, False, 1e-6) is None
    q = torch.zeros(1, 1, 2, 64).half()
    for a in (q, None, 3):
        assert btf._calls.tree_attention(a, q, q, v, v, None, None, None, None) is None
        assert btf._calls.sample(a, v, None, None, None, None, None, None) is None
    assert btf._calls.sample(x) is None  # (too few arguments)


def _rebound(btf, monkeypatch, here):
    monkeypatch.setattr(btf, "HERE", str(here))
    monkeypatch.setattr(btf, "_calls", None)
    monkeypatch.setattr(btf, "_bind_tried", False)
    btf._bind_calls()
    return btf._calls


def test_a_binding_that_does_not_load_leaves_the_mirror(btf, tmp_path, monkeypatch):
    """A library of another torch, or no library at all, is no reason for set-up or a call to fail."""
    btf.lib()
    assert _rebound(btf, monkeypatch, tmp_path) is None  # none there
    (tmp_path / "btf_b200_calls.so").write_bytes(b"not a shared object")
    assert _rebound(btf, monkeypatch, tmp_path) is None
    src = tmp_path / "m.c"  # loads, and is not the module; then one that wants a symbol that is not there
    for code in ("int x;", "extern int no_such_symbol(void); int (*f)(void) = no_such_symbol;"):
        src.write_text(code)
        so = tmp_path / "other" / "btf_b200_calls.so"
        so.parent.mkdir(exist_ok=True)
        subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
        assert _rebound(btf, monkeypatch, so.parent) is None
    torch = pytest.importorskip("torch")
    with pytest.raises(RuntimeError, match="CUDA"):  # the mirror does the call
        btf.sample(torch.zeros(2, 10), torch.zeros(2))


def test_a_binding_of_another_torch_is_not_used(btf, monkeypatch):
    torch = pytest.importorskip("torch")
    if not os.path.exists(os.path.join(btf.HERE, "btf_b200_calls.so")):
        pytest.skip("built without torch")
    assert _rebound(btf, monkeypatch, btf.HERE) is not None
    monkeypatch.setattr(torch, "__version__", "1.0.0+cu1")
    assert _rebound(btf, monkeypatch, btf.HERE) is None


@pytest.mark.parametrize("before", ["", "sys.modules['torch'] = None"], ids=["installed", "not to be had"])
def test_set_up_needs_no_torch(before):
    """kernels_init neither imports torch nor needs it (the device is not looked for here)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ["import sys", "sys.path.insert(0, 'bonsai-ternary-fast_b200')", before, "import btf_b200 as b",
            "b.check = lambda *a: None", "b.kernels_init(0)", "assert not sys.modules.get('torch') and b._calls is None"]
    r = subprocess.run([sys.executable, "-c", "\n".join(code)], cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_tensors_that_want_a_gradient_are_refused(btf):
    """The calls record no graph, so a gradient would be missing in silence: refused as torch's own out= calls are."""
    torch = pytest.importorskip("torch")
    t, p = btf.RopeTable(64, device="cpu"), torch.zeros(2, dtype=torch.int32)
    x, w = torch.zeros(2, 1, 64), torch.ones(64)
    g = lambda a: a.clone().requires_grad_()  # noqa: E731
    q, k = torch.zeros(1, 2, 4, 64).half(), torch.zeros(1, 9, 2, 64).half()
    b = torch.zeros(2, 10)
    calls = [lambda: btf.rope([btf.RopeSeg(g(x))], t, p), lambda: btf.rope([btf.RopeSeg(x, g(x))], t, p),
             lambda: btf.rope([btf.RopeSeg(x), btf.RopeSeg(x, x, normw=g(w))], t, p),
             lambda: btf.tree_attention(g(q), k, k, p[:1], p[None]), lambda: btf.tree_attention(q, g(k), k, p[:1], p[None]),
             lambda: btf.tree_attention(q, k, g(k), p[:1], p[None]),
             lambda: btf.tree_attention(q, k, k, p[:1], p[None], out=g(q)),
             lambda: btf.sample(b, b[:, 0], logprobs=g(b[:, 0]))]
    for fn in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            fn()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            fn()


@pytest.mark.parametrize("seg", [dict(heads=2, y_head=0), dict(y_token=0), dict(y_token=0, rows=P, n_rows=2)])
def test_rope_refuses_rows_that_share_their_memory(btf, seg):
    """An expanded output, whose rows would overwrite one another."""
    assert _rope(btf, seg=seg) == 1
    assert b"strides" in btf.lib().btf_last_error()


@pytest.mark.parametrize("kw", [dict(B=2, o_batch=0), dict(o_node=0), dict(o_head=0)])
def test_tree_attention_refuses_rows_that_share_their_memory(btf, kw):
    assert _tree(btf, **kw) == 1
    assert b"strides" in btf.lib().btf_last_error()
