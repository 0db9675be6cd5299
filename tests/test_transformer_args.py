"""What the transformer operators refuse, and the frequencies of rotary
positions: on the CPU, nothing is launched."""
import ctypes

import numpy as np
import pytest

import tinytorch_amd
from tinytorch_amd import Attention, Rope, Strides
from transformer_ref import frequencies

P = 0x1000  # a pointer that no refused call reads


@pytest.fixture(scope="module")
def L():
    return tinytorch_amd.lib()


def rope(**kw):
    d = dict(head_dim=64, rot_dim=64, interleaved=0, scaling=0, base=10000.0, factor=1.0, trained=0.0, low=0.0,
             high=0.0, magnitude=0.0)
    d.update(kw)
    return Rope(**d)


@pytest.mark.parametrize("kw", [dict(), dict(rot_dim=2), dict(rot_dim=32, base=500000.0),
                                dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0),
                                dict(scaling=2, factor=8.0, rot_dim=2),
                                dict(scaling=3, factor=8.0, trained=8192.0, low=1.0, high=32.0)])
def test_frequencies(L, kw):
    r = rope(**kw)
    f = (ctypes.c_double * (r.rot_dim // 2))()
    assert L.tt_rope_frequencies(r, f) == 0
    want = frequencies(r.rot_dim, r.base, ("plain", "linear", "ntk", "parts")[r.scaling], r.factor, r.trained,
                       r.low, r.high)
    np.testing.assert_allclose(np.array(f), want, rtol=1e-13)


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=66),
                                dict(head_dim=1024, rot_dim=514), dict(base=0.0), dict(base=float("inf")),
                                dict(base=float("nan")), dict(scaling=4), dict(scaling=-1),
                                dict(scaling=1, factor=0.0), dict(scaling=2, factor=float("inf")),
                                dict(scaling=3, factor=2.0, trained=0.0, high=1.0),
                                dict(scaling=3, factor=2.0, trained=10.0, low=1.0, high=1.0),
                                dict(magnitude=-1.0), dict(magnitude=float("nan"))])
def test_rope_refuses(L, kw):
    f = (ctypes.c_double * 512)()
    assert L.tt_rope_frequencies(rope(**kw), f) == -1
    assert L.tt_k_rope(rope(**kw), P, P, None, 4, 4, 2, 0, 0, 0) == -1


@pytest.mark.parametrize("args", [(None, P, None, 4, 4, 2, 0, 0), (P, None, None, 4, 4, 2, 0, 0),
                                  (P, P, None, 0, 4, 2, 0, 0), (P, P, None, 4, 0, 2, 0, 0),
                                  (P, P, None, 4, 4, 0, 0, 0), (P, P, None, 4, 4, 2, 127, 0),
                                  (P, P, None, 4, 4, 2, 0, 127), (P, P, None, 4, 4, 2, 128, 132),
                                  (P, P, None, 1 << 60, 4, 2, 0, 0), (P, P, None, 4, 4, 1 << 30, 0, 0)])
def test_rope_refuses_layouts(L, args):
    x, y, pos, rows, seq, heads, ldx, ldy = args
    assert L.tt_k_rope(rope(), x, y, pos, rows, seq, heads, ldx, ldy, 0) == -1


def attention(**kw):
    d = dict(batch=2, q_rows=8, k_rows=8, q_heads=4, kv_heads=2, head_dim=64)
    d.update(kw)
    return Attention(**d)


BAD_ATTENTION = [dict(batch=0), dict(q_rows=0), dict(k_rows=0), dict(q_heads=0), dict(kv_heads=0),
                 dict(kv_heads=3), dict(head_dim=0), dict(head_dim=129), dict(window=-1),
                 dict(scale=float("nan")), dict(scale=float("inf")), dict(q_rows=1 << 31),
                 dict(k_rows=1 << 31), dict(batch=1 << 40), dict(batch=1 << 20, q_rows=1 << 20),
                 dict(batch=1 << 20, k_rows=1 << 20), dict(q=Strides(row=-4)), dict(o=Strides(batch=-1)),
                 dict(k=Strides(row=63)), dict(v=Strides(head=63)), dict(k=Strides(row=(1 << 23) + 1)),
                 dict(q=Strides(head=(1 << 27) + 1)), dict(q_heads=1 << 18, kv_heads=1 << 18)]


@pytest.mark.parametrize("kw", BAD_ATTENTION)
def test_attention_refuses(L, kw):
    a = attention(**kw)
    assert L.tt_k_attention_fwd(a, P, P, P, P, None, None) == -1
    assert L.tt_k_attention_bwd(a, P, P, P, P, P, P, P, P, P, None) == -1
    assert L.tt_k_attention_fwd_ws(a) == 0 and L.tt_k_attention_bwd_ws(a) == 0


@pytest.mark.parametrize("kw", [dict(batch=1, q_rows=1 << 17, k_rows=1 << 17, q_heads=64, kv_heads=8),
                                dict(batch=1, q_rows=1 << 22, k_rows=1 << 20, q_heads=1, kv_heads=1),
                                dict(batch=64, q_rows=4096, k_rows=1 << 17, q_heads=64, kv_heads=8),
                                dict(batch=1, q_rows=1 << 28, k_rows=1 << 28, q_heads=1, kv_heads=1)])
def test_attention_workspaces_stay_small(L, kw):
    """Next to operands of gigabytes: 4 GiB at most for each of two kinds of
    images and for the parts of the gradients, and two floats a row."""
    a = attention(head_dim=128, **kw)
    rows = kw["batch"] * kw["q_heads"] * kw["q_rows"]
    assert L.tt_k_attention_fwd_ws(a) <= 4.01 * 2**30
    assert 4 * rows <= L.tt_k_attention_bwd_ws(a) <= 12.01 * 2**30 + 4 * rows


def test_attention_workspace_sizes_stand(L):
    """The size asked for is that of the call, whatever was asked before."""
    kinds = [attention(batch=2, q_rows=r, k_rows=900, q_heads=2, kv_heads=2, head_dim=d)
             for d in (16, 64, 80, 96, 112, 128) for r in (1, 16, 17, 32, 33, 100, 1100)]
    sizes = [(L.tt_k_attention_fwd_ws(a), L.tt_k_attention_bwd_ws(a)) for a in kinds]
    assert min(min(s) for s in sizes) > 0
    for i in np.random.default_rng(0).permutation(len(kinds) * 4) % len(kinds):
        a = kinds[i]
        assert (L.tt_k_attention_fwd_ws(a), L.tt_k_attention_bwd_ws(a)) == sizes[i]


def test_attention_refuses_missing_operands(L):
    a = attention()
    for i in range(4):
        args = [P] * 4
        args[i] = None
        assert L.tt_k_attention_fwd(a, *args, None, None) == -1
    for i in range(6):
        args = [P] * 6
        args[i] = None
        assert L.tt_k_attention_bwd(a, *args, P, P, P, None) == -1
    assert L.tt_k_attention_bwd(a, *[P] * 6, P, P, None, None) == -1  # dk without dv
    assert L.tt_k_attention_bwd(a, *[P] * 6, None, None, None, None) == 0  # nothing asked for
    assert L.tt_k_attention_fwd(None, P, P, P, P, None, None) == -1


@pytest.mark.parametrize("args", [(None, P, 4, 8, 1e-5), (P, None, 4, 8, 1e-5), (P, P, 0, 8, 1e-5),
                                  (P, P, 4, 0, 1e-5), (P, P, -1, 8, 1e-5), (P, P, 4, 8, -1e-5),
                                  (P, P, 4, 8, float("nan")), (P, P, 4, 8, float("inf")),
                                  (P, P, 1 << 40, 1 << 20, 1e-5), (P, P, 4, 1 << 31, 1e-5)])
def test_layernorm_refuses(L, args):
    x, y, rows, cols, eps = args
    assert L.tt_k_layernorm_fwd(x, None, None, y, None, None, rows, cols, eps) == -1


def test_layernorm_backward_refuses(L):
    for i in range(4):
        args = [P] * 4  # x, dy, mean, rstd
        args[i] = None
        assert L.tt_k_layernorm_bwd(args[0], P, args[1], args[2], args[3], P, P, P, 4, 8, None) == -1
    assert L.tt_k_layernorm_bwd(P, P, P, P, P, P, P, P, 0, 8, None) == -1
    assert L.tt_k_layernorm_bwd(P, P, P, P, P, None, None, None, 4, 8, None) == 0
    assert L.tt_k_layernorm_bwd_ws(0, 8) == 0 and L.tt_k_layernorm_bwd_ws(4, 8) > 0


@pytest.mark.parametrize("kw", [dict(z=None), dict(ids=None), dict(teacher=None), dict(loss=None), dict(rows=0),
                                dict(cols=0), dict(top=0), dict(top=1025), dict(T=0.0), dict(T=-1.0),
                                dict(T=float("nan")), dict(T=float("inf")), dict(scale=float("nan")),
                                dict(rows=1 << 40), dict(dz=P)])
def test_distill_refuses(L, kw):
    d = dict(z=P, ids=P, teacher=P, loss=P, dz=2 * P, rows=4, cols=10, top=3, T=1.0, scale=1.0)
    d.update(kw)
    assert L.tt_k_distill(d["z"], d["ids"], d["teacher"], d["top"], d["T"], d["loss"], d["dz"], d["rows"],
                          d["cols"], d["scale"]) == -1


def test_nodes_refuse_missing_inputs(L):
    assert not L.ag_layernorm(None, None, None, 1e-5)
    assert not L.ag_rope(None, rope(), 2, None, 4)
    assert not L.ag_attention(None, None, None, attention())
    assert not L.ag_distill(None, None, None, 3, 1.0)


def test_node_methods_exist():
    import importlib
    import os
    import sys
    from tinytorch_amd.torch_py import Node
    sys.path.insert(0, os.path.join(tinytorch_amd.ROOT, "build"))
    try:
        m = importlib.import_module("tinytorch_pybind")
    finally:
        sys.path.pop(0)
    for meth in ("layernorm", "rope", "attention", "distill"):
        assert hasattr(m.Node, meth) and hasattr(Node, meth)


@pytest.mark.parametrize("kw", [dict(low=float("-inf"), high=1.0), dict(low=float("-inf"), high=float("inf"))])
def test_rope_refuses_a_ramp_without_a_start(L, kw):
    """r = clamp((n - low) / (high - low)) has no value there: NaN frequencies."""
    f = (ctypes.c_double * 32)()
    r = rope(scaling=3, factor=8.0, trained=8192.0, **kw)
    assert L.tt_rope_frequencies(r, f) == -1
    assert L.tt_k_rope(r, P, P, None, 4, 4, 2, 0, 0, 0) == -1


@pytest.mark.parametrize("kw", [dict(scaling=2, factor=1e-200, rot_dim=4), dict(base=5e-324),
                                dict(scaling=1, factor=1e-310), dict(scaling=3, factor=1e-310, trained=1.0, high=9.0)])
def test_rope_refuses_frequencies_past_the_range(L, kw):
    """Finite parameters whose frequencies are not: position 0 times them is NaN."""
    f = (ctypes.c_double * 32)()
    assert L.tt_rope_frequencies(rope(**kw), f) == -1
    assert L.tt_k_rope(rope(**kw), P, P, None, 4, 4, 2, 0, 0, 0) == -1


def test_rope_takes_a_ramp_without_an_end(L):
    """high = infinity keeps no frequency."""
    f = (ctypes.c_double * 32)()
    assert L.tt_rope_frequencies(rope(scaling=3, factor=8.0, trained=8192.0, low=1.0, high=float("inf")), f) == 0
    np.testing.assert_allclose(np.array(f), frequencies(64, 10000.0) / 8, rtol=1e-13)


@pytest.mark.parametrize("T,scale", [(1e-39, 1.0), (1e-30, 1.0), (1e-19, 1.0), (1.9e19, 1.0), (1e38, 0.0),
                                     (1e18, 1e30)])
def test_distill_refuses_temperatures_past_the_range(L, T, scale):
    """1 / T, T^2 and scale T are factors in 32 bits: infinite or without their
    bits they leave NaN or a wrong loss."""
    assert L.tt_k_distill(P, P, P, 3, T, P, 2 * P, 4, 10, scale) == -1


def test_inline_assembly_names_the_registers_it_writes():
    """m0 holds the address of a direct load to LDS: the compiler has to know
    that it changes."""
    import glob
    import os
    import re
    found = 0
    for path in glob.glob(os.path.join(tinytorch_amd.ROOT, "tinytorch_amd", "csrc", "*")):
        with open(path) as f:
            for block in re.findall(r"asm volatile\((.*?)\);", f.read(), re.S):
                if re.search(r"_mov_b32 m0\b", block):
                    found += 1
                    assert '"m0"' in block, (path, block)
    assert found
