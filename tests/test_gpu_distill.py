"""Distillation against 64 bits: row widths, entries left out or of one
column, empty rows, infinite logits, temperatures."""
import numpy as np
import pytest

import transformer_ref as ref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu


def _inputs(rows, cols, top, spread=2.0):
    rng = np.random.default_rng(rows * 31 + cols * 7 + top)
    z = (rng.standard_normal((rows, cols)) * spread).astype(np.float32)
    ids = np.stack([rng.permutation(cols)[:top] if top <= cols else rng.integers(0, cols, top)
                    for _ in range(rows)]).astype(np.int32)
    return z, ids, (5 + rng.standard_normal((rows, top)) * 2).astype(np.float32)


def _run(L, z, ids, t, T, scale, grad=True):
    rows, cols = z.shape
    d = [DevBuf.from_np(a) for a in (z, ids, t)]
    loss, dz = DevBuf(rows), DevBuf(z.size) if grad else None
    loss.fill(np.nan)
    if grad:
        dz.fill(np.nan)
    check(L.tt_k_distill(d[0].ptr, d[1].ptr, d[2].ptr, ids.shape[1], T, loss.ptr, dz.ptr if grad else None, rows,
                         cols, scale), "distill")
    return loss.to_np(), dz.to_np(z.shape) if grad else None


@pytest.mark.parametrize("rows,cols,top", [(1, 1, 1), (3, 2, 2), (700, 3, 3), (9, 5, 2), (9, 6, 6), (9, 7, 1),
                                           (3, 131071, 40), (600, 66001, 5), (5, 10, 3), (130, 63, 8), (4, 64, 64), (3, 100, 65),
                                           (7, 1003, 8), (2, 1024, 1), (2, 1025, 17), (5, 4096, 128), (3, 4097, 5),
                                           (2, 16384, 64), (3, 16387, 3), (2, 32000, 64), (2, 32769, 33),
                                           (2, 65536, 16), (3, 65537, 9), (2, 131072, 50), (2, 2000, 1024),
                                           (3, 7, 1024)])
def test_distill(tlib, rows, cols, top):
    z, ids, t = _inputs(rows, cols, top)
    for T in (1.0, 3.0):
        loss, dz = _run(tlib, z, ids, t, T, 1.0 / rows)
        want = ref.distill(z, ids, t, T, 1.0 / rows)
        ref.close(loss, want[0], "loss")
        ref.close(dz, want[1], "dlogits")
        only, _ = _run(tlib, z, ids, t, T, 1.0 / rows, grad=False)
        assert np.array_equal(only, loss)


@pytest.mark.parametrize("cols", [50, 5000, 70000])
def test_distill_entries(tlib, cols):
    """Ids outside the columns, one column several times, rows that hold
    nothing, teacher logits of -inf, student logits of -inf."""
    z, ids, t = _inputs(12, cols, 6)
    ids[0, 2], ids[0, 4] = -1, cols
    ids[1] = -1
    ids[2, :] = [3, 9, 3, 3, 9, 1]
    t[3] = -np.inf
    t[4, 1:] = -np.inf
    z[5, ids[5, 0]] = -np.inf             # a column that the teacher wants
    z[6, (ids[6, 0] + 1) % cols] = -np.inf  # perhaps one that it does not
    z[7] = -np.inf
    ids[8] = ids[8, 0]
    z[9] = np.float32(-3.4028235e38)
    t[10] = np.float32(-3.4028235e38)
    ids[11, 0], t[11, 0] = np.int32(-2147483648), np.nan  # left out: its logit is not looked at
    loss, dz = _run(tlib, z, ids, t, 2.0, 0.25)
    want = ref.distill(z, ids, t, 2.0, 0.25)
    ref.close(loss, want[0], "loss")
    ref.close(dz, want[1], "dlogits")
    assert loss[1] == 0 and loss[3] == 0 and not dz[1].any() and not dz[3].any()
    assert np.isposinf(loss[5])


def test_distill_nan_stays_in_its_row(tlib):
    z, ids, t = _inputs(4, 300, 5)
    z[1, 7] = np.nan
    t[2, 3] = np.nan
    loss, dz = _run(tlib, z, ids, t, 1.0, 1.0)
    want = ref.distill(z[[0, 3]], ids[[0, 3]], t[[0, 3]], 1.0, 1.0)
    assert np.isnan(loss[1]) and np.isnan(loss[2])
    ref.close(loss[[0, 3]], want[0])
    ref.close(dz[[0, 3]], want[1])


def test_distill_node(tlib):
    from tinytorch_amd.torch_py import Node
    z, ids, t = _inputs(9, 40, 4)
    (rl, e_rl), (dz, e_dz) = ref.distill(z, ids, t, 2.0, 1.0 / 9)
    Z = Node.leaf(z)
    loss = Z.distill(ids, t, 2.0)
    mean = (np.array([rl.mean()]), np.array([e_rl.mean() + 12 * ref.U * np.abs(rl).mean()]))
    ref.close(loss.value(), mean)
    loss.backward(None)
    ref.close(Z.grad(), (dz, e_dz))
    loss.backward(None)  # the kept seed, added
    ref.close(Z.grad(), (2 * dz, 2 * e_dz + 2 * ref.U * np.abs(dz)))
    # with the labels' loss, as a student is trained
    Z2 = Node.leaf(z)
    y = np.arange(9, dtype=np.int32)
    total = Z2.distill(ids, t, 2.0) * 0.5 + Z2.softmax_ce(y) * 0.5
    total.backward(None)
    p = np.exp(z.astype(np.float64) - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    p[np.arange(9), y] -= 1
    np.testing.assert_allclose(Z2.grad(), 0.5 * dz + 0.5 * p / 9, rtol=1e-5, atol=2e-7)
    const = Node.leaf(z, False).distill(ids, t, 2.0)
    ref.close(const.value(), mean)
    const.backward(None)
    for bad in (lambda: Z.distill(ids[:8], t[:8]), lambda: Z.distill(ids, t[:, :3]),
                lambda: Z.distill(ids, t, 0.0), lambda: Z.distill(ids[:, :0], t[:, :0]),
                lambda: Node.leaf(z.reshape(3, 3, 40)).distill(ids, t)):
        with pytest.raises(ValueError):
            bad()


def test_distill_gradient_by_differences(tlib):
    z, ids, t = _inputs(3, 30, 4)
    _, dz = _run(tlib, z, ids, t, 2.0, 1.0)
    d = np.random.default_rng(2).standard_normal(z.shape)
    f = [ref.distill(z.astype(np.float64) + h * d, ids, t, 2.0, 1.0)[0][0].sum() for h in (1e-5, -1e-5)]
    assert abs((f[0] - f[1]) / 2e-5 - (dz * d).sum()) <= 1e-5 * np.abs(dz * d).sum()


WIDTHS = [2, 50, 1003, 4096, 5000, 16384, 32001, 65536, 70001]  # each kernel, with and without a tail


@pytest.mark.parametrize("cols", WIDTHS)
def test_distill_rows_of_nan(tlib, cols):
    """Rows of NaN, and of NaN and -inf, have no finite loss and no finite
    gradient, whatever their width; a row of -inf and the others do."""
    z, ids, t = _inputs(6, cols, 2)
    z[1] = np.nan
    z[2] = -np.inf
    z[2, cols - 1] = np.nan
    z[3] = np.nan
    z[3, 0] = -np.inf
    z[4] = -np.inf
    want = ref.distill(z[[0, 4, 5]], ids[[0, 4, 5]], t[[0, 4, 5]], 2.0, 0.5)
    loss, dz = _run(tlib, z, ids, t, 2.0, 0.5)
    assert np.isnan(loss[1:4]).all() and np.isnan(dz[1:4]).all()
    ref.close(loss[[0, 4, 5]], want[0], "loss")
    ref.close(dz[[0, 4, 5]], want[1], "dlogits")
    only, _ = _run(tlib, z, ids, t, 2.0, 0.5, grad=False)
    assert np.array_equal(only, loss, equal_nan=True)


@pytest.mark.parametrize("cols", WIDTHS)
def test_distill_rows_left_out(tlib, cols):
    """Rows without entries, or with -inf for all of them, have loss and gradient
    0 whatever their logits hold."""
    z, ids, t = _inputs(7, cols, 2)
    z[0] = np.nan
    z[1, 0] = np.nan
    z[2, cols - 1] = np.inf
    z[3] = np.inf
    z[4, cols // 2] = np.nan
    z[5] = -np.inf
    ids[:3], ids[3] = -1, cols
    t[4:6] = -np.inf
    ids[4] = cols // 2
    loss, dz = _run(tlib, z, ids, t, 2.0, 0.5)
    assert not loss[:6].any() and not dz[:6].any()
    want = ref.distill(z[6:], ids[6:], t[6:], 2.0, 0.5)
    ref.close(loss[6:], want[0], "loss")
    ref.close(dz[6:], want[1], "dlogits")
    only, _ = _run(tlib, z, ids, t, 2.0, 0.5, grad=False)
    assert np.array_equal(only, loss)
