"""Layer norm, forward and backward, against 64 bits: every width of its row
groups, rows that are not 16-byte aligned, rows too long for registers."""
import ctypes

import numpy as np
import pytest

import transformer_ref as ref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

SIZES = [(5000, 3), (4097, 2), (3000, 1), (4099, 5), (3, 6), (3, 7), (600, 2555), (2, 16383), (2, 16385),
         (1, 1), (3, 1), (1, 7), (5, 4), (257, 64), (33, 255), (7, 256), (9, 257), (600, 512), (5, 516), (3, 1000),
         (1025, 1024), (4099, 1003), (4, 1028), (17, 2047), (3, 2048), (70, 3000), (5, 4096), (3, 4100),
         (9, 8191), (2, 8192), (300, 8200), (3, 16384), (5, 16385), (70, 20000)]


def _inputs(rows, cols):
    rng = np.random.default_rng(rows * 7919 + cols)
    x = (rng.standard_normal((rows, cols)) * 1.5 + rng.standard_normal(cols)).astype(np.float32)
    return (x, (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32), rng.standard_normal(cols).astype(np.float32),
            rng.standard_normal((rows, cols)).astype(np.float32))


def _ptr(d):
    return d.ptr if d is not None else None


def _run(L, x, w, b, dy, eps=1e-5, ws=None, want=(True, True, True)):
    rows, cols = x.shape
    dx_, dw_, db_, ddy = (DevBuf.from_np(t) if t is not None else None for t in (x, w, b, dy))
    y, mean, rstd = DevBuf(x.size), DevBuf(rows), DevBuf(rows)
    out = [DevBuf(n) if on else None for n, on in zip((x.size, cols, cols), want)]
    for d in [y, mean, rstd] + [o for o in out if o is not None]:
        d.fill(np.nan)
    check(L.tt_k_layernorm_fwd(dx_.ptr, _ptr(dw_), _ptr(db_), y.ptr, mean.ptr, rstd.ptr, rows, cols, eps), "fwd")
    check(L.tt_k_layernorm_bwd(dx_.ptr, _ptr(dw_), ddy.ptr, mean.ptr, rstd.ptr, *[_ptr(o) for o in out], rows, cols,
                               ws), "bwd")
    shapes = [x.shape, (rows,), (rows,), x.shape, (cols,), (cols,)]
    return [d.to_np(s) if d is not None else None for d, s in zip([y, mean, rstd] + out, shapes)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_layernorm(tlib, rows, cols):
    x, w, b, dy = _inputs(rows, cols)
    got = _run(tlib, x, w, b, dy)
    want = ref.layernorm(x, w, b, dy)
    for name, g, v in zip(("y", "mean", "rstd", "dx", "dw", "db"), got, want):
        ref.close(g, v, f"{name} {rows}x{cols}")
    again = _run(tlib, x, w, b, dy)  # the sums have one order
    for g, a in zip(got, again):
        assert np.array_equal(g.view(np.uint32), a.view(np.uint32))


@pytest.mark.parametrize("rows,cols", [(37, 96), (5, 1003), (3, 5000), (2, 16400)])
def test_layernorm_parts(tlib, rows, cols):
    """Without weight or bias; each gradient alone; mean and rstd not asked for."""
    x, w, b, dy = _inputs(rows, cols)
    for ww, bb in ((None, None), (w, None), (None, b)):
        got = _run(tlib, x, ww, bb, dy)
        for name, g, v in zip(("y", "mean", "rstd", "dx", "dw", "db"), got, ref.layernorm(x, ww, bb, dy)):
            ref.close(g, v, name)
    full = _run(tlib, x, w, b, dy)
    for i in range(3):
        got = _run(tlib, x, w, b, dy, want=[k == i for k in range(3)])
        ref.close(got[3 + i], ref.layernorm(x, w, b, dy)[3 + i])
    y, d = DevBuf(x.size), [DevBuf.from_np(t) for t in (x, w, b)]
    check(tlib.tt_k_layernorm_fwd(d[0].ptr, d[1].ptr, d[2].ptr, y.ptr, None, None, rows, cols, 1e-5), "fwd")
    assert np.array_equal(y.to_np(x.shape), full[0])


def test_layernorm_workspace_allocates_nothing(tlib):
    x, w, b, dy = _inputs(300, 520)
    want = _run(tlib, x, w, b, dy)
    ws = DevBuf(tlib.tt_k_layernorm_bwd_ws(300, 520) // 4)
    d = [DevBuf.from_np(t) for t in (x, w, dy)]
    mean, rstd = DevBuf.from_np(want[1]), DevBuf.from_np(want[2])
    out = [DevBuf(n) for n in (x.size, 520, 520)]
    assert tlib.tth_fail_alloc_after(0) == 0
    try:
        rc = tlib.tt_k_layernorm_bwd(d[0].ptr, d[1].ptr, d[2].ptr, mean.ptr, rstd.ptr, *[o.ptr for o in out], 300,
                                     520, ws.ptr)
        none = tlib.tt_k_layernorm_bwd(d[0].ptr, d[1].ptr, d[2].ptr, mean.ptr, rstd.ptr, *[o.ptr for o in out],
                                       300, 520, None)
    finally:
        tlib.tth_fail_alloc_after(-1)
    assert rc == 0 and none == -2
    for o, v in zip(out, want[3:]):
        assert np.array_equal(o.to_np(v.shape), v)


def test_layernorm_edge_rows(tlib):
    """A constant row; a row of large offset; a row with an infinity (NaN, its
    own row alone)."""
    x, w, b, dy = _inputs(6, 40)
    x[1] = 3.0
    x[2] = x[2] * 1e-3 + 100.0
    x[4, 7] = np.inf
    got = _run(tlib, x, w, b, dy)
    keep = [0, 1, 2, 3, 5]
    for g, v in zip(got[:4], ref.layernorm(x[keep], w, b, dy[keep])[:4]):
        ref.close(g[keep], v)
    assert np.isnan(got[0][4]).all() and np.isnan(got[3][4]).all()


@pytest.mark.parametrize("needs", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
@pytest.mark.parametrize("has", [(1, 1), (1, 0), (0, 1), (0, 0)])
def test_layernorm_node(tlib, needs, has):
    """Gradients of those that need one, twice backward adds up; the axes before
    the last are rows."""
    from tinytorch_amd.torch_py import Node
    x, w, b, dy = _inputs(12, 33)
    X = Node.leaf(x.reshape(3, 4, 33), bool(needs[0]))
    W = Node.leaf(w, bool(needs[1])) if has[0] else None
    B = Node.leaf(b, bool(needs[2])) if has[1] else None
    y = X.layernorm(W, B)
    want = ref.layernorm(x, w if has[0] else None, b if has[1] else None, dy)
    assert y.value().shape == (3, 4, 33)
    ref.close(y.value().reshape(12, 33), want[0])
    y.backward(dy)
    for n, on, v in ((X, needs[0], want[3]), (W, needs[1], want[4]), (B, needs[2], want[5])):
        if n is None:
            continue
        if not on:
            assert n.grad() is None
            continue
        ref.close(n.grad().reshape(v[0].shape), v)
    y.backward(dy)
    if needs[0]:
        g = X.grad().reshape(12, 33)
        ref.close(g, (2 * want[3][0], 2 * want[3][1] + 2 * ref.U * np.abs(want[3][0])))
    with pytest.raises(ValueError):
        X.layernorm(Node.leaf(np.ones(32, np.float32)))
    with pytest.raises(ValueError):
        X.layernorm(W, B, eps=-1.0)


def test_layernorm_gradient_by_differences(tlib):
    x, w, b, dy = _inputs(4, 19)
    got = _run(tlib, x, w, b, dy)
    rng = np.random.default_rng(1)
    for i, g in ((0, got[3]), (1, got[4]), (2, got[5])):
        p = [x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)]
        d = rng.standard_normal(p[i].shape)
        f = []
        for h in (1e-5, -1e-5):
            q = list(p)
            q[i] = p[i] + h * d
            m = q[0] - q[0].mean(1, keepdims=True)
            y = m / np.sqrt((m * m).mean(1, keepdims=True) + 1e-5) * q[1] + q[2]
            f.append((y * dy).sum())
        slope = (f[0] - f[1]) / 2e-5
        # the differences are good to about 1e-9, the gradient to its bound
        assert abs(slope - (g * d).sum()) <= 1e-5 * np.abs(g * d).sum()


def test_layernorm_gradients_of_the_longest_rows(tlib):
    """Past 2^26 columns: the sums for dw and db pass a grid axis's threads.  With
    one row, mean 0 and rstd 1 they are dy x and dy, to the bit."""
    cols = (1 << 26) + 5
    rng = np.random.default_rng(3)
    x, dy = rng.standard_normal(cols, np.float32), rng.standard_normal(cols, np.float32)
    d = [DevBuf.from_np(t) for t in (x, dy, np.zeros(1, np.float32), np.ones(1, np.float32))]
    dw, db = DevBuf(cols), DevBuf(cols)
    check(tlib.tt_k_layernorm_bwd(d[0].ptr, None, *[t.ptr for t in d[1:]], None, dw.ptr, db.ptr, 1, cols, None), "bwd")
    assert np.array_equal(dw.to_np(), dy * x) and np.array_equal(db.to_np(), dy)
    for t in d + [dw, db]:
        t.free()
    tlib.tth_release_cache()
