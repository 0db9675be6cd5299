"""Newton-Schulz steps and Muon of matrices of up to 32 rows or columns, whose steps are
taken in 64 bits, six at a time: values that are off by their own rounding."""
import ctypes

import numpy as np
import pytest

import training_ref as ref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

NEAR = ref.A**4 * ref.PART  # of products: a rounding of their parts through four steps' slope at 0

SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (4, 31), (5, 64), (65, 6), (10, 785), (129, 10), (16, 16), (17, 16), (16, 130),
          (17, 40), (32, 32), (31, 33), (33, 31), (32, 1024), (1024, 7), (32, 1025), (1025, 3), (3, 1024), (5, 4000),
          (4097, 16), (17, 4096), (20, 5003), (32, 70001), (70001, 32), (1, 100003), (300007, 2)]


def _steps64(x, steps):
    x = x.astype(np.float64)
    y = x.T if x.shape[0] > x.shape[1] else x
    norm = np.linalg.norm(y)
    y = y / norm if norm else y
    for _ in range(steps):
        p = y @ y.T
        y = (ref.A * np.eye(len(y)) + ref.B * p + ref.C * (p @ p)) @ y
    return y.T if x.shape[0] > x.shape[1] else y


def _steps32(x, steps):
    y = x.astype(np.float64)
    y = (y.T if x.shape[0] > x.shape[1] else y) / np.linalg.norm(y)
    y = y.astype(np.float32)
    a, b, c = (np.float32(t) for t in (ref.A, ref.B, ref.C))
    for _ in range(steps):
        p = y @ y.T
        y = a * y + (b * p + c * (p @ p)) @ y
    return y.T if x.shape[0] > x.shape[1] else y


def _close(got, want):
    """A value's own rounding, and what 64 bits leave after six steps (2^-53 of the
    squares of singular values, times how the steps depend on those, 1e7 for 1e-3 of
    the largest): far under 2^-26 of its row and column."""
    rows, cols = (np.linalg.norm(want, axis=a, keepdims=True) for a in (1, 0))
    tol = ref.U * np.abs(want) + 2.0**-26 * np.minimum(rows, cols)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / np.maximum(tol, 1e-300))


def _matrix(rows, cols, kind, seed=0):
    x = np.random.default_rng(rows * 7 + cols + seed).standard_normal((rows, cols))
    if kind == "weak":
        x[::2] *= 1e-6
        x[:, ::3] *= 1e-5
    if kind == "steep":
        x = 1e-2 * x + np.outer(x[:, 0], x[0])
    return x.astype(np.float32)


def _run(L, x, steps, in_place=False, ws=None):
    X = DevBuf.from_np(x)
    y = X if in_place else DevBuf(x.size + 4)
    if not in_place:
        y.fill(-7.0)
    check(L.tt_k_newton_schulz(X.ptr, y.ptr, x.shape[0] if x.ndim == 3 else 1, *x.shape[-2:], steps, ws), "steps")
    got = y.to_np()
    assert in_place or (got[-4:] == -7).all()
    return got[:x.size].reshape(x.shape)


@pytest.mark.parametrize("kind", ["even", "weak", "steep"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_steps_of_few_rows(tlib, rows, cols, kind):
    x = _matrix(rows, cols, kind)
    for steps in (1, 5, 6):
        got = _run(tlib, x, steps)
        _close(got, _steps64(x, steps))
    assert np.array_equal(got, _run(tlib, x, 6, in_place=True))
    need = tlib.tt_k_newton_schulz_ws(1, rows, cols)
    assert (need == 0) == (max(rows, cols) <= 1024) and need < 1 << 20
    ws = DevBuf(need // 4 + 16)
    ws.fill(np.nan)
    assert np.array_equal(got, _run(tlib, x, 6, ws=ws.ptr))
    assert np.isnan(ws.to_np()[need // 4:]).all()


@pytest.mark.parametrize("rows,cols", [(6, 50), (30, 900), (9, 3000), (2500, 20)])
def test_many_steps_of_few_rows(tlib, rows, cols):
    """From six steps on X goes on from its fp32 values.  Where these are near 1 the steps
    enlarge their rounding, by 4.2 at most and 1.6 at the fixed point 0.87 (2^-24 by 1.6^24
    is 5e-3): fp32 products pass on the same and round more often, and 8 times what they
    leave is for how it happens to fall."""
    for kind in ("even", "weak"):
        x = _matrix(rows, cols, kind)
        for steps in (12, 30):
            got, want, single = _run(tlib, x, steps), _steps64(x, steps), _steps32(x, steps)
            for axis in (0, 1):
                off, near = (np.linalg.norm(t - want, axis=axis) / np.linalg.norm(want, axis=axis) for t in (got, single))
                assert off.max() <= max(2.0**-22, 8 * near.max())
    assert np.isfinite(_run(tlib, x, 64)).all()


@pytest.mark.parametrize("rows,cols,rank", [(8, 100, 3), (31, 32, 4), (16, 500, 8), (700, 32, 5), (12, 3000, 2),
                                            (5000, 32, 9)])
def test_many_steps_of_lower_rank(tlib, rows, cols, rank):
    """Singular values of 0, of small whole numbers: what the squares' rounding puts in
    their place, of either sign, grows by A^2 a step.  All stay within 1.21 and what fp32
    values leave, whose own rounding grows in these directions until it is as large as
    the rest: the measure is what fp32 products leave, as they fall within 8 times."""
    rng = np.random.default_rng(rows)
    x = (rng.integers(-3, 4, (rows, rank)) @ rng.integers(-3, 4, (rank, cols))).astype(np.float32)
    near = ref.A**4 * ref.PART
    for steps in (6, 7, 12, 18, 20, 33, 64):
        got, want = _run(tlib, x, steps).astype(np.float64), _steps64(x, steps)
        assert np.isfinite(got).all()
        assert np.linalg.norm(got, 2) <= 1.21
        off, single = (np.linalg.norm(t - want) for t in (got, _steps32(x, steps)))
        assert off <= max(near * np.linalg.norm(want), 8 * single), (steps, off, single)


@pytest.mark.parametrize("rows,cols", [(5, 40), (40, 31), (3, 2000)])
@pytest.mark.parametrize("count", [2, 63, 64, 65, 200])
def test_many_matrices_of_few_rows(tlib, count, rows, cols):
    x = np.stack([_matrix(rows, cols, "even", i) * np.float32(10.0**(i % 7 - 3)) for i in range(count)])
    x[1] = np.nan
    got = _run(tlib, x, 5)
    assert np.isnan(got[1]).all()
    for i in {0, count // 2, count - 1} - {1}:
        assert np.array_equal(got[i], _run(tlib, x[i], 5))
        _close(got[i], _steps64(x[i], 5))


@pytest.mark.parametrize("rows,cols", [(4, 30), (30, 17), (20, 3000), (1030, 2)])
def test_few_rows_of_bad_values(tlib, rows, cols):
    for bad in (np.nan, np.inf, -np.inf):
        x = _matrix(rows, cols, "even")
        x[rows // 2, cols // 2] = bad
        assert np.isnan(_run(tlib, x, 5)).all()
    assert (_run(tlib, np.zeros((rows, cols), np.float32), 5) == 0).all()
    for scale in (1e-44, 1e-30, 1e30, 1e37):
        x = (_matrix(rows, cols, "even") * np.float64(scale)).astype(np.float32)
        _close(_run(tlib, x, 5), _steps64(x, 5))
    x = np.zeros((rows, cols), np.float32)
    x[rows - 1, 0] = -3.0
    s = 1.0
    for _ in range(5):
        s = ref.A * s + ref.B * s**3 + ref.C * s**5
    got = _run(tlib, x, 5)
    assert abs(got[rows - 1, 0] + s) <= 2 * ref.U and np.count_nonzero(got) == 1


@pytest.mark.parametrize("nesterov", [0, 1])
@pytest.mark.parametrize("shapes,products", [([(5, 7), (1, 9), (31, 32)], 0),
                                             ([(10, 785), (3000, 4), (12, 2000), (32, 1024)], 0),
                                             ([(129, 10), (40, 50), (70, 60)], 0), ([(40, 50), (4, 5000), (64, 64)], 0),
                                             ([(3, 40 + i) for i in range(8)] + [(1030 + i, 5) for i in range(8)], 0),
                                             ([(129, 10), (40, 50), (4, 5000), (150, 160)], 1),
                                             ([(20000, 3), (150, 160), (1, 70000), (16, 16384)], 1),
                                             ([(1300, 1200), (16, 1200), (700, 30), (2, 16385)], 1)])
def test_muon_of_few_rows(tlib, shapes, products, nesterov):
    """By themselves, beside others in LDS, and (products) beside matrices whose launches
    they share, as near as those are, but for the longest."""
    rng = np.random.default_rng(4)
    w, g, v = ([rng.standard_normal(s).astype(np.float32) for s in shapes] for _ in range(3))
    W, G, V = ([DevBuf.from_np(t) for t in ts] for ts in (w, g, v))
    rows, cols = ((ctypes.c_long * len(shapes))(*[s[i] for s in shapes]) for i in (0, 1))
    lr, mu, decay = (np.float32(t) for t in (0.02, 0.95, 0.1))
    need = tlib.tt_k_muon_multi_ws(rows, cols, len(shapes))
    ws = DevBuf(need // 4 + 16)
    ws.fill(np.nan)

    def p(ds):
        return (ctypes.c_void_p * len(ds))(*[d.ptr for d in ds])

    for k in range(2):
        check(tlib.tt_k_muon_multi(p(W), p(G), p(V), rows, cols, len(shapes), lr, mu, nesterov, decay,
                                   None if k else ws.ptr), "muon")
        assert np.isnan(ws.to_np()[need // 4:]).all()
        for i, s in enumerate(shapes):
            vel = mu * v[i] + g[i]  # each operation rounded, as fp32 does it
            u = mu * vel + g[i] if nesterov else vel
            assert np.array_equal(V[i].to_np(s), vel)
            got = W[i].to_np(s)
            x = _steps64(u, 5)
            if min(s) > 32 or products and max(s) <= 16384:
                size = float(lr) * 0.2 * np.sqrt(max(s)) * np.linalg.norm(x)
                kept = (1 - float(lr) * float(decay)) * w[i].astype(np.float64)
                off = np.linalg.norm(got - (kept - float(lr) * 0.2 * np.sqrt(max(s)) * x))
                assert off <= NEAR * size + 4 * ref.U * (np.linalg.norm(kept) + size)
            else:
                rate = float(lr) * 0.2 * np.sqrt(max(s))
                kept = (1 - float(lr) * float(decay)) * w[i].astype(np.float64)
                size = np.abs(kept) + rate * np.abs(x)
                edge = np.minimum(*(np.linalg.norm(x, axis=a, keepdims=True) for a in (1, 0)))
                assert (np.abs(got - (kept - rate * x)) <= 4 * ref.U * size + rate * 2.0**-26 * edge).all()
            assert not np.array_equal(got, w[i])
            w[i], v[i] = got, vel
