"""RMS norm with the residual's addition, forward and backward, against 64 bits:
every width of its row groups, rows that are not 16-byte aligned, rows too long for
registers."""
import numpy as np
import pytest

import training_ref as ref
from transformer_ref import close
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 1), (4097, 2), (5000, 3), (1, 4), (1, 7), (4099, 5), (5, 4), (257, 64), (33, 255), (7, 256),
         (9, 257), (600, 512), (5, 516), (3, 1000), (1, 1024), (1025, 1024), (4099, 1003), (4, 1028), (17, 2047),
         (3, 2048), (600, 2555), (5, 4096), (3, 4100), (9, 8191), (2, 8192), (300, 8200), (3, 16383), (3, 16384),
         (5, 16385), (70, 20000)]
NAMES = ("y", "sum", "rstd", "dx", "dw")


def _inputs(rows, cols):
    rng = np.random.default_rng(rows * 7919 + cols)

    def n(*s):
        return rng.standard_normal(s).astype(np.float32)

    return n(rows, cols), 2 * n(rows, cols), 1 + 0.2 * n(cols), n(rows, cols), n(rows, cols)


def _ptr(d):
    return d.ptr if d is not None else None


def _run(L, x, res, w, dy, dsum, eps=1e-5, ws=None, want=(True, True), in_place=False):
    rows, cols = x.shape
    X, R, W, DY, DS = (DevBuf.from_np(t) if t is not None else None for t in (x, res, w, dy, dsum))
    y, rstd, s = DevBuf(x.size), DevBuf(rows), (R if in_place else DevBuf(x.size)) if res is not None else None
    dx = (DS if in_place and dsum is not None else DevBuf(x.size)) if want[0] else None
    dw = DevBuf(cols) if want[1] else None
    for d in [y, rstd] + ([] if in_place else [t for t in (s, dx) if t is not None]) + ([dw] if dw else []):
        d.fill(np.nan)
    check(L.tt_k_rmsnorm_fwd(X.ptr, _ptr(R), _ptr(W), y.ptr, _ptr(s), rstd.ptr, rows, cols, eps), "fwd")
    check(L.tt_k_rmsnorm_bwd(_ptr(s) or X.ptr, _ptr(W), DY.ptr, _ptr(DS), rstd.ptr, _ptr(dx), _ptr(dw), rows, cols,
                             ws), "bwd")
    shapes = [x.shape, x.shape, (rows,), x.shape, (cols,)]
    return [d.to_np(k) if d is not None else None for d, k in zip([y, s, rstd, dx, dw], shapes)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_rmsnorm(tlib, rows, cols):
    x, res, w, dy, ds = _inputs(rows, cols)
    got = _run(tlib, x, res, w, dy, ds)
    for name, g, v in zip(NAMES, got, ref.rmsnorm(x, res, w, dy, ds)):
        close(g, v, f"{name} {rows}x{cols}")
    # the sums have one order; the sum over the residual, dx over the other gradient
    for g, a in zip(got, _run(tlib, x, res, w, dy, ds, in_place=True)):
        assert np.array_equal(g.view(np.uint32), a.view(np.uint32))


@pytest.mark.parametrize("rows,cols", [(37, 96), (5, 1003), (3, 5000), (2, 16400), (9, 3)])
def test_rmsnorm_parts(tlib, rows, cols):
    """Without residual, weight or the other gradient; each gradient alone; sum and
    rstd not asked for."""
    x, res, w, dy, ds = _inputs(rows, cols)
    for rr, ww, dd in ((None, None, None), (res, None, None), (None, w, ds), (res, w, None), (None, w, None)):
        got = _run(tlib, x, rr, ww, dy, dd)
        for name, g, v in zip(NAMES, got, ref.rmsnorm(x, rr, ww, dy, dd)):
            if name != "sum" or rr is not None:
                close(g, v, name)
    full = _run(tlib, x, res, w, dy, ds)
    for i in range(2):
        got = _run(tlib, x, res, w, dy, ds, want=[k == i for k in range(2)])
        assert np.array_equal(got[3 + i], full[3 + i]) or cols > 16384 or cols < 4 or i == 0
        close(got[3 + i], ref.rmsnorm(x, res, w, dy, ds)[3 + i])
    y, d = DevBuf(x.size), [DevBuf.from_np(t) for t in (x, res, w)]
    check(tlib.tt_k_rmsnorm_fwd(d[0].ptr, d[1].ptr, d[2].ptr, y.ptr, None, None, rows, cols, 1e-5), "fwd")
    assert np.array_equal(y.to_np(x.shape), full[0])


def test_rmsnorm_any_alignment(tlib):
    """Operands that begin at any float, and nothing written past their ends."""
    rows, cols = 5, 260
    x, res, w, dy, ds = _inputs(rows, cols)
    want = _run(tlib, x, res, w, dy, ds)
    for off in (1, 2, 3):
        def place(a):
            b = np.full(a.size + 8, np.nan, np.float32)
            b[off:off + a.size] = a.ravel()
            return DevBuf.from_np(b)

        X, R, W, DY, DS = (place(a) for a in (x, res, w, dy, ds))
        out = [DevBuf(n + 8) for n in (x.size, x.size, rows, x.size, cols)]
        for o in out:
            o.fill(-7.0)
        X, R, W, DY, DS = (t.ptr + 4 * off for t in (X, R, W, DY, DS))
        o = [t.ptr + 4 * off for t in out]
        check(tlib.tt_k_rmsnorm_fwd(X, R, W, o[0], o[1], o[2], rows, cols, 1e-5), "fwd")
        check(tlib.tt_k_rmsnorm_bwd(o[1], W, DY, DS, o[2], o[3], o[4], rows, cols, None), "bwd")
        for d, v in zip(out, want):
            g = d.to_np()
            assert np.array_equal(g[off:off + v.size], v.ravel())
            assert (g[:off] == -7).all() and (g[off + v.size:] == -7).all()


def test_rmsnorm_workspace_allocates_nothing(tlib):
    x, res, w, dy, ds = _inputs(300, 520)
    want = _run(tlib, x, res, w, dy, ds)
    ws = DevBuf(tlib.tt_k_rmsnorm_bwd_ws(300, 520) // 4)
    d = [DevBuf.from_np(t) for t in (want[1], w, dy, ds, want[2])]
    out = [DevBuf(n) for n in (x.size, 520)]
    args = [t.ptr for t in d] + [o.ptr for o in out] + [300, 520]
    assert tlib.tth_fail_alloc_after(0) == 0
    try:
        rc, none = tlib.tt_k_rmsnorm_bwd(*args, ws.ptr), tlib.tt_k_rmsnorm_bwd(*args, None)
    finally:
        tlib.tth_fail_alloc_after(-1)
    assert rc == 0 and none == -2
    for o, v in zip(out, want[3:]):
        assert np.array_equal(o.to_np(v.shape), v)


def test_rmsnorm_edge_rows(tlib):
    """A row of zeros; of tiny and of large values; one whose squares pass the
    range; an infinity and a NaN (in their own rows alone)."""
    x, _, w, dy, ds = _inputs(8, 40)
    x[1] = 0.0
    x[2] *= 1e-20
    x[3] *= 1e15
    x[4] *= 1e25
    x[5, 7] = np.inf
    x[6, 9] = np.nan
    got = _run(tlib, x, None, w, dy, ds)
    keep = [0, 1, 2, 3, 7]
    want = ref.rmsnorm(x[keep], None, w, dy[keep], ds[keep])
    for i in (0, 2, 3):
        close(got[i][keep], want[i])
    assert got[2][4] == 0 and (got[0][4] == 0).all() and np.array_equal(got[3][4], ds[4])
    assert np.isnan(got[0][5][7]) and (got[0][5][:7] == 0).all()
    assert np.isnan(got[0][6]).all() and np.isnan(got[3][6]).all()


def _node_run(Node, x, res, w, needs, has_res, has_w):
    X = Node.leaf(x, bool(needs[0]))
    R = Node.leaf(res, bool(needs[1])) if has_res else None
    W = Node.leaf(w, bool(needs[2])) if has_w else None
    return X, R, W, X.rmsnorm(W, R) if has_res else (X.rmsnorm(W), None)


@pytest.mark.parametrize("needs", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (0, 0, 0)])
@pytest.mark.parametrize("has", [(1, 1), (1, 0), (0, 1), (0, 0)])
@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_rmsnorm_node(tlib, bound, needs, has):
    """Gradients of those that need one, with the sum used once more behind the norm;
    backward twice adds up; the axes before the last are rows."""
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node
    x, res, w, dy, ds = _inputs(12, 33)
    X, R, W, (y, s) = _node_run(Node, x.reshape(3, 4, 33), res.reshape(3, 4, 33), w, needs, *has)
    want = ref.rmsnorm(x, res if has[0] else None, w if has[1] else None, dy, ds)
    assert y.value().shape == (3, 4, 33)
    close(y.value().reshape(12, 33), want[0])
    last = y
    if s is not None:
        close(s.value().reshape(12, 33), want[1])
        last = y + s * Node.leaf((ds / dy).reshape(3, 4, 33), False)  # its gradient: ds, to two roundings
    live = (needs[0], has[0] and needs[1], has[1] and needs[2])
    if not any(live):
        last.backward(dy)
        assert X.grad() is None
        return
    last.backward(dy)
    dx, tol = want[3] if has[0] else ref.rmsnorm(x, None, w if has[1] else None, dy)[3]
    tol = tol + 3 * ref.U * np.abs(ds)
    for n, on in ((X, live[0]), (R, live[1])):
        if n is not None:
            assert (n.grad() is None) == (not on)
            if on:
                close(n.grad().reshape(12, 33), (dx, tol))
    if live[2]:
        close(W.grad(), want[4])
    first = X.grad()
    y.backward(dy)  # once more, past the sum
    if live[0]:
        again = ref.rmsnorm(x, res if has[0] else None, w if has[1] else None, dy)[3]
        # the sum's own gradient stays from the first pass and is passed on with it
        more = 2 * dx if has[0] else dx
        close(X.grad().reshape(12, 33), (more + again[0], 3 * tol + again[1] + 8 * ref.U * (np.abs(dx) + np.abs(again[0]))))
        assert first is not None


@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_rmsnorm_node_twice(tlib, bound):
    """One node as x and as the residual: the sum is twice it, and its gradient has
    both; and one node as x and as the weight."""
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node
    x, _, w, dy, _ = _inputs(5, 21)
    X = Node.leaf(x)
    y, s = X.rmsnorm(Node.leaf(w, False), X)
    y.backward(dy)
    want = ref.rmsnorm(x, x, w, dy)
    close(y.value(), want[0])
    assert np.array_equal(s.value(), 2 * x)
    close(X.grad(), (2 * want[3][0], 2 * want[3][1]))
    W = Node.leaf(w)
    y = W.rmsnorm(W)
    y.backward(dy[0])
    want = ref.rmsnorm(w[None], None, w, dy[:1])
    close(y.value(), (want[0][0][0], want[0][1][0]))
    dx, dw = want[3], want[4]
    both = dx[0][0] + dw[0]
    close(W.grad(), (both, dx[1][0] + dw[1] + ref.U * np.abs(both)))


def test_rmsnorm_node_refuses(tlib):
    from tinytorch_amd.torch_py import Node
    x, res, w, _, _ = _inputs(4, 8)
    X = Node.leaf(x)
    for kw in (dict(w=Node.leaf(w[:7])), dict(residual=Node.leaf(res[:3])), dict(residual=Node.leaf(res.reshape(2, 16))),
               dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            X.rmsnorm(**kw)


def test_rmsnorm_gradient_by_differences(tlib):
    x, res, w, dy, ds = _inputs(4, 19)
    got = _run(tlib, x, res, w, dy, ds)
    rng = np.random.default_rng(1)
    for i, g in ((0, got[3]), (1, got[3]), (2, got[4])):
        p = [t.astype(np.float64) for t in (x, res, w)]
        d = rng.standard_normal(p[i].shape)
        f = []
        for h in (1e-5, -1e-5):
            q = list(p)
            q[i] = p[i] + h * d
            s = q[0] + q[1]
            f.append((s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5) * q[2] * dy).sum() + (s * ds).sum())
        slope = (f[0] - f[1]) / 2e-5
        # the differences are good to about 1e-9, the gradient to its bound
        assert abs(slope - (g * d).sum()) <= 1e-5 * np.abs(g * d).sum()
