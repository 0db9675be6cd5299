"""Newton-Schulz steps of matrices that a workgroup has in LDS: every number of blocks
of rows, rows up to where LDS ends, even matrices and uneven ones side by side; and
steps of matrices of any size of value."""
import numpy as np
import pytest

import training_ref as ref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

# A rounding of the fp16 parts, 2^-22, in a weak direction, times the steps' slope at 0
# of 3.4445 four times: of a matrix, and of each row and column, whose size no step
# multiplies by less than 0.64.
NEAR = ref.A**4 * ref.PART


def _steps64(x, steps):
    x = x.astype(np.float64)
    y = x.T if x.shape[0] > x.shape[1] else x
    norm = np.linalg.norm(y)
    y = y / norm if norm else y
    for _ in range(steps):
        p = y @ y.T
        y = ref.A * y + (ref.B * p + ref.C * (p @ p)) @ y
    return y.T if x.shape[0] > x.shape[1] else y


def _close(got, want, near=NEAR):
    for axis in (None, 1, 0):
        off, size = np.linalg.norm(got - want, axis=axis), np.linalg.norm(want, axis=axis)
        assert np.all(off <= near * size), (axis, np.max(off / np.maximum(size, 1e-300)))


def _matrix(rng, rows, cols, kind):
    x = rng.standard_normal((rows, cols))
    if kind == 1:
        x[rows // 3:] *= 1e-6
    if kind == 2:
        x[:, ::2] *= 1e-5
        x[::2] *= 1e-5
    if kind == 3:
        x[rows // 2] = 0
        x[:, cols // 2:] = 0
    return x.astype(np.float32)


def _run(L, x, steps, in_place=False):
    X = DevBuf.from_np(x)
    y = X if in_place else DevBuf(x.size + 4)
    if not in_place:
        y.fill(-7.0)
    check(L.tt_k_newton_schulz(X.ptr, y.ptr, x.shape[0], *x.shape[1:], steps, None), "steps")
    got = y.to_np()
    assert in_place or (got[-4:] == -7).all()
    return got[:x.size].reshape(x.shape)


@pytest.mark.parametrize("rows,cols", [(128, 128), (97, 128), (127, 100), (128, 160), (160, 128), (100, 150), (101, 129),
                                       (64, 480), (480, 64), (33, 449), (40, 470), (32, 992), (992, 32), (1, 990),
                                       (31, 830), (96, 300), (300, 65), (95, 97), (96, 96), (64, 64), (64, 65), (33, 33)])
def test_many_matrices_in_lds(tlib, rows, cols):
    """32 of them and more have a workgroup each, and what it does goes by its matrix."""
    count = 33
    assert tlib.tt_k_newton_schulz_ws(count, rows, cols) == 0
    rng = np.random.default_rng(rows * 1000 + cols)
    x = np.stack([_matrix(rng, rows, cols, i % 4) for i in range(count)])
    x[17] = 0
    for steps in (1, 5, 6):
        got = _run(tlib, x, steps)
        for i in (0, 1, 2, 3, 17, 30, 31, 32):
            _close(got[i], _steps64(x[i], steps))
    assert np.array_equal(got, _run(tlib, x, 6, in_place=True))


@pytest.mark.parametrize("rows,cols", [(32, 992), (992, 32), (32, 513), (64, 384), (384, 64), (96, 160), (160, 96), (65, 129),
                                       (97, 97), (128, 128), (100, 127), (128, 160)])
def test_one_matrix_in_lds_or_not(tlib, rows, cols):
    """A single one has a workgroup while its products are short; either way it is as one of
    many, but for the order of the sums."""
    rng = np.random.default_rng(rows + 1000 * cols)
    for kind in range(4):
        x = _matrix(rng, rows, cols, kind)[None]
        for steps in (1, 5):
            _close(_run(tlib, x, steps)[0], _steps64(x[0], steps))
        assert np.array_equal(_run(tlib, x, 5), _run(tlib, x, 5, in_place=True))


@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-30, 1e-10, 1e10, 1e30, 3e37])
@pytest.mark.parametrize("rows,cols", [(20, 45), (150, 160), (1300, 1400)])
def test_steps_near_at_any_scale(tlib, rows, cols, scale):
    """By norm, as near as any."""
    x = np.random.default_rng(3).standard_normal((1, rows, cols)) * np.float64(scale)
    x = x.astype(np.float32)
    assert np.abs(x).max() > 0
    got, want = _run(tlib, x, 5)[0], _steps64(x[0], 5)
    assert np.linalg.norm(got - want) <= NEAR * np.linalg.norm(want)
