"""Newton-Schulz steps and Muon of matrices with weak rows and columns.  The steps
multiply each row and column from the left or right by a matrix whose eigenvalues lie
within [0.64, 3.45] a step, so a weak one stays weak, and what fp32 products leave is
small against that row or column itself, not only against the matrix."""
import ctypes

import numpy as np
import pytest

import training_ref as ref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

# An operand's rounding, 2^-22 of its row's norm, in a direction that is weak in this
# row and strong nowhere, times the steps' slope at 0 of 3.4445 four times.
NEAR = ref.A**4 * ref.PART


def _steps(x, steps, dtype=np.float64):
    y = x.astype(np.float64)
    turned = y.shape[0] > y.shape[1]
    y = y.T if turned else y
    norm = np.linalg.norm(y)
    y = (y / norm if norm else y).astype(dtype)
    a, b, c = (dtype(t) for t in (ref.A, ref.B, ref.C))
    for _ in range(steps):
        p = y @ y.T
        y = a * y + (b * p + c * (p @ p)) @ y
    return y.T if turned else y


def _worst(got, want):
    """Of the rows and of the columns, relative to each."""
    out = []
    for axis in (1, 0):
        off, size = np.linalg.norm(got - want, axis=axis), np.linalg.norm(want, axis=axis)
        assert (off[size == 0] == 0).all()
        out.append(np.max(off[size > 0] / size[size > 0]))
    return out


def _weak(rows, cols, factor, kind, seed=0):
    x = np.random.default_rng(rows + cols + seed).standard_normal((rows, cols))
    if kind == "graded":
        x = x * np.geomspace(1, factor, rows)[:, None] * np.geomspace(factor, 1, cols)
    if kind in ("rows", "both"):
        x[::2] *= factor
    if kind in ("columns", "both"):
        x[:, 1::3] *= factor
    if kind == "one":
        x[rows // 2] *= factor
        x[0] = 0  # zeros stay zeros
        x[:, cols - 1] = 0
    return x.astype(np.float32)


def _close(got, x, steps):
    """Once values are near 1 a step's slope there, 4.2 at 1.21 and -1.6 at the fixed
    point 0.87, passes errors on enlarged, so after many steps what fp32 products leave
    is the measure: an operand's rounding, 2^-22, is 4 times fp32's, the steps pass both
    on alike, and twice that for how it happens to fall."""
    want, near = _steps(x, steps), [NEAR, NEAR]
    if steps > 6:
        near = [max(NEAR, 8 * t) for t in _worst(_steps(x, steps, np.float32), want)]
    worst = _worst(got, want)
    assert worst[0] <= near[0] and worst[1] <= near[1], (worst, near)


def _run(L, x, steps, in_place=False):
    X = DevBuf.from_np(np.ascontiguousarray(x))
    y = X if in_place else DevBuf(x.size)
    check(L.tt_k_newton_schulz(X.ptr, y.ptr, x.shape[0] if x.ndim == 3 else 1, *x.shape[-2:], steps, None), "steps")
    return y.to_np(x.shape)


# in LDS; by tiles of 32, with shared lengths too; of 128; of 256
SMALL = [(20, 45), (45, 20), (64, 64), (96, 100), (128, 128), (200, 300), (300, 200), (40, 4000), (4000, 40), (2, 3000)]


@pytest.mark.parametrize("factor", [1e-3, 1e-5, 1e-7, 1e-10])
@pytest.mark.parametrize("kind", ["rows", "columns", "both", "graded", "one"])
@pytest.mark.parametrize("rows,cols", SMALL)
def test_weak_rows_and_columns(tlib, rows, cols, kind, factor):
    x = _weak(rows, cols, factor, kind)
    for steps in (1, 5, 6):
        got = _run(tlib, x, steps)
        _close(got, x, steps)
    assert np.array_equal(got, _run(tlib, x, 6, in_place=True))


@pytest.mark.parametrize("kind", ["rows", "columns", "both", "one"])
@pytest.mark.parametrize("rows,cols", [(45, 20), (96, 100), (200, 300), (300, 200), (40, 4000)])
@pytest.mark.parametrize("steps", [7, 12, 16])
def test_many_steps(tlib, rows, cols, kind, steps):
    """What was weak is as large as the rest in the end."""
    for factor in (1.0, 1e-3, 1e-7):
        x = _weak(rows, cols, factor, kind)
        got = _run(tlib, x, steps)
        _close(got, x, steps)
        assert np.array_equal(got, _run(tlib, x, steps, in_place=True))
    several = np.stack([x, x[::-1], x])
    for got, want in zip(_run(tlib, several, steps), (x, x[::-1], x)):
        _close(got, want, steps)


@pytest.mark.parametrize("kind", ["rows", "columns", "both"])
@pytest.mark.parametrize("rows,cols,steps", [(1400, 1460, 5), (1290, 1700, 7), (1700, 1290, 8), (2100, 7010, 5),
                                             (7003, 2101, 7)])
def test_weak_in_large_matrices(tlib, rows, cols, steps, kind):
    x = _weak(rows, cols, 1e-7, kind)
    _close(_run(tlib, x, steps), x, steps)


@pytest.mark.parametrize("shapes", [[(30, 50), (96, 60)], [(785, 256), (129, 10), (300, 500)],
                                    [(1500, 1300), (40, 50), (900, 1400)]])
def test_muon_of_weak_rows(tlib, shapes):
    """From no weights, so that what a step adds is all there is."""
    x = [_weak(*s, 1e-6, "both", i) for i, s in enumerate(shapes)]
    W, V, G = [DevBuf.from_np(0 * t) for t in x], [DevBuf.from_np(0 * t) for t in x], [DevBuf.from_np(t) for t in x]

    def p(ds):
        return (ctypes.c_void_p * len(ds))(*[d.ptr for d in ds])

    r, c = ((ctypes.c_long * len(shapes))(*[s[i] for s in shapes]) for i in (0, 1))
    check(tlib.tt_k_muon_multi(p(W), p(G), p(V), r, c, len(shapes), 0.5, 0.9, 0, 0.0, None), "muon")
    for w, t, s in zip(W, x, shapes):
        _close(w.to_np(s) / (-0.5 * 0.2 * np.sqrt(max(s))), t, 5)


@pytest.mark.parametrize("rows,cols", [(45, 20), (200, 300), (1400, 1460)])
def test_bad_values_among_weak(tlib, rows, cols):
    for bad in (np.nan, np.inf):
        x = _weak(rows, cols, 1e-7, "both")
        x[4, 1] = bad
        for steps in (1, 5, 8):
            assert np.isnan(_run(tlib, x, steps)).all()
    x = np.zeros((rows, cols), np.float32)
    for steps in (5, 9):
        assert (_run(tlib, x, steps) == 0).all()


@pytest.mark.parametrize("count,rows,cols", [(6, 33, 1 << 20), (7, 1 << 20, 34)])
def test_flat_matrices_in_groups(tlib, count, rows, cols):
    """Their images pass 4 GiB together: a part of them at a time."""
    alone, all_ws = (tlib.tt_k_newton_schulz_ws(n, rows, cols) for n in (1, count))
    assert all_ws < 5 << 30 and all_ws < count * alone
    x = np.random.default_rng(5).standard_normal((1, rows, cols), np.float32)
    x = np.concatenate([x * np.float32(2.0**i) for i in range(count)])
    x[count - 2] = 0
    got, want = _run(tlib, x, 2), _steps(x[0], 2)
    # (a part's products go by tiles of their own, so the sums' order is not that of one alone)
    for g in (got[0], got[count // 2], got[count - 1], _run(tlib, x[0], 2)):
        worst = _worst(g, want)
        assert max(worst) <= NEAR, worst
    assert (got[count - 2] == 0).all()


@pytest.mark.parametrize("rows,cols,rank", [(40, 60, 5), (96, 100, 30), (200, 300, 7), (300, 200, 100), (40, 4000, 8)])
def test_many_steps_of_lower_rank(tlib, rows, cols, rank):
    """Singular values of 0, of small whole numbers: what rounding puts in their place
    grows until it is as large as the rest, and no larger."""
    rng = np.random.default_rng(rows)
    x = (rng.integers(-3, 4, (rows, rank)) @ rng.integers(-3, 4, (rank, cols))).astype(np.float32)
    for steps in (6, 7, 18, 33, 64):
        got, want = _run(tlib, x, steps).astype(np.float64), _steps(x, steps)
        assert np.linalg.norm(got, 2) <= 1.21
        off, single = (np.linalg.norm(t - want) for t in (got, _steps(x, steps, np.float32)))
        assert off <= max(NEAR * np.linalg.norm(want), 8 * single)
