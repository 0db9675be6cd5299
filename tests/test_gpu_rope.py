"""Rotary positions against 64 bits: both pairings, part of the head, scaled
frequencies, far positions, row distances and unaligned rows."""
import numpy as np
import pytest

import transformer_ref as ref
from tinytorch_amd import Rope
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

SCALED = [dict(), dict(scaling=1, factor=4.0), dict(scaling=2, factor=4.0),
          dict(scaling=3, factor=8.0, trained=8192.0, low=1.0, high=32.0)]
NAMES = ("plain", "linear", "ntk", "parts")


def _rope(dim, rot, interleaved, kw, magnitude=0.0):
    return Rope(dim, rot, int(interleaved), kw.get("scaling", 0), 10000.0, kw.get("factor", 1.0),
                kw.get("trained", 0.0), kw.get("low", 0.0), kw.get("high", 0.0), magnitude)


def _freq(rot, kw):
    return ref.frequencies(rot, 10000.0, NAMES[kw.get("scaling", 0)], kw.get("factor", 1.0), kw.get("trained", 0.0),
                           kw.get("low", 0.0), kw.get("high", 0.0))


@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 1, 2, 2), (3, 2, 64, 64), (65, 5, 80, 32), (33, 3, 128, 128),
                                                (7, 20, 128, 64), (100, 1, 18, 10), (5, 7, 33, 8), (300, 8, 64, 64),
                                                (2, 3, 600, 512), (9, 40, 256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(tlib, rows, heads, dim, rot, interleaved):
    rng = np.random.default_rng(rows * 100 + dim + rot)
    for kw in SCALED:
        x = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        pos = rng.integers(0, 200000, rows).astype(np.int32)
        f = _freq(rot, kw)
        d, p, y = DevBuf.from_np(x), DevBuf.from_np(pos), DevBuf(x.size)
        for transpose in (0, 1):
            y.fill(np.nan)
            check(tlib.tt_k_rope(_rope(dim, rot, interleaved, kw), d.ptr, y.ptr, p.ptr, rows, 0, heads, 0, 0,
                                 transpose), "rope")
            got = y.to_np(x.shape)
            ref.close(got, ref.rope(x, pos, f, interleaved, bool(transpose)), f"{kw} {transpose}")
            assert np.array_equal(got[..., rot:], x[..., rot:])
        y.fill(np.nan)
        check(tlib.tt_k_rope(_rope(dim, rot, interleaved, kw, 1.25), d.ptr, y.ptr, None, rows, 3, heads, 0, 0, 0),
              "rope")
        ref.close(y.to_np(x.shape), ref.rope(x, np.arange(rows) % 3, f, interleaved, magnitude=1.25), "seq")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("ldx,ldy", [(520, 384), (384, 520), (385, 386)])
def test_rope_row_distances(tlib, interleaved, ldx, ldy):
    """The first heads of a wider buffer; what lies between rows stays."""
    rng = np.random.default_rng(ldx)
    buf = rng.standard_normal((11, ldx)).astype(np.float32)
    pos = rng.integers(0, 100, 11).astype(np.int32)
    d, p, y = DevBuf.from_np(buf), DevBuf.from_np(pos), DevBuf(11 * ldy)
    y.fill(7.0)
    check(tlib.tt_k_rope(_rope(64, 64, interleaved, {}), d.ptr, y.ptr, p.ptr, 11, 0, 6, ldx, ldy, 0), "rope")
    got = y.to_np((11, ldy))
    ref.close(got[:, :384].reshape(11, 6, 64),
              ref.rope(buf[:, :384].reshape(11, 6, 64), pos, _freq(64, {}), interleaved))
    assert np.all(got[:, 384:] == 7.0)
    # in place, rows apart
    check(tlib.tt_k_rope(_rope(64, 64, interleaved, {}), d.ptr, d.ptr, p.ptr, 11, 0, 6, ldx, ldx, 0), "rope")
    inp = d.to_np((11, ldx))
    assert np.array_equal(inp[:, :384], got[:, :384]) and np.array_equal(inp[:, 384:], buf[:, 384:])


def test_rope_unaligned_pointer(tlib):
    x = np.random.default_rng(5).standard_normal((4, 2, 64)).astype(np.float32)
    d, y = DevBuf(x.size + 1), DevBuf(x.size + 1)
    check(tlib.tth_h2d(d.ptr + 4, x.ctypes.data, x.nbytes), "h2d")
    check(tlib.tt_k_rope(_rope(64, 64, False, {}), d.ptr + 4, y.ptr + 4, None, 4, 4, 2, 0, 0, 0), "rope")
    ref.close(y.to_np()[1:].reshape(x.shape), ref.rope(x, np.arange(4), _freq(64, {}), False))


@pytest.mark.parametrize("shape", [(6, 96), (2, 3, 96), (2, 3, 3, 32)])
def test_rope_node(tlib, shape):
    from tinytorch_amd.torch_py import Node
    rng = np.random.default_rng(9)
    x, dy = (rng.standard_normal((6, 3, 32)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 5000, 6)
    f = _freq(16, {})
    X = Node.leaf(x.reshape(shape))
    y = X.rope(3, 32, pos, rot_dim=16, interleaved=True)
    assert y.value().shape == shape
    ref.close(y.value().reshape(x.shape), ref.rope(x, pos, f, True))
    y.backward(dy.reshape(shape))
    ref.close(X.grad().reshape(x.shape), ref.rope(dy, pos, f, True, True))
    ref.close(X.rope(3, 32, seq_len=3, rot_dim=16).value().reshape(x.shape),
              ref.rope(x, np.arange(6) % 3, f, False))
    for bad in (lambda: X.rope(4, 32, seq_len=3), lambda: X.rope(3, 32, [1, 2]), lambda: X.rope(3, 32),
                lambda: X.rope(3, 32, seq_len=3, rot_dim=15), lambda: X.rope(0, 32, seq_len=3)):
        with pytest.raises(ValueError):
            bad()


def test_rope_gradient_by_differences(tlib):
    """The rotation is linear: its gradient's product with a direction is the
    output's product along that direction."""
    rng = np.random.default_rng(3)
    x, dy = (rng.standard_normal((5, 2, 24)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 9000, 5).astype(np.int32)
    d, g, p, y = DevBuf.from_np(x), DevBuf.from_np(dy), DevBuf.from_np(pos), DevBuf(x.size)
    r = _rope(24, 20, True, SCALED[3], 1.1)
    check(tlib.tt_k_rope(r, d.ptr, y.ptr, p.ptr, 5, 0, 2, 0, 0, 0), "rope")
    f = (y.to_np(x.shape).astype(np.float64) * dy).sum()
    check(tlib.tt_k_rope(r, g.ptr, y.ptr, p.ptr, 5, 0, 2, 0, 0, 1), "rope")
    assert abs(f - (y.to_np(x.shape).astype(np.float64) * x).sum()) <= 20 * ref.U * 1.1 * np.abs(x * dy).sum() * 2
