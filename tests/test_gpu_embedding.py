"""Token embeddings and the table's gradient, against 64 bits: batches that sort
in one block, by one merge and by two; rows of every width; tokens that are one, all
different, outside the table, and as often as words are."""
import numpy as np
import pytest

import training_ref as ref
from transformer_ref import close
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu


def _tokens(rng, rows, vocab, kind):
    if kind == "one":
        return np.full(rows, vocab // 2, np.int32)
    if kind == "none":
        return np.full(rows, -1, np.int32)
    if kind == "even":
        return rng.integers(0, vocab, rows).astype(np.int32)
    if kind == "falling":
        return (vocab - 1 - np.arange(rows) % vocab).astype(np.int32)
    ids = np.minimum(np.exp(rng.random(rows) * np.log(vocab + 1.0)).astype(np.int64) - 1, vocab - 1)  # words
    ids = rng.permutation(vocab)[ids].astype(np.int32)
    if kind == "padded":
        ids[rng.random(rows) < 0.3] = rng.choice([-1, vocab, -2**31, 2**31 - 1])
    return ids


def _grad(L, ids, dy, vocab, scale=1.0, old=None, ws=None):
    d, g = DevBuf.from_np(ids), DevBuf.from_np(dy)
    dw = DevBuf(vocab * dy.shape[1]) if old is None else DevBuf.from_np(old)
    if old is None:
        dw.fill(np.nan)
    check(L.tt_k_embedding_bwd(d.ptr, g.ptr, dw.ptr, len(ids), vocab, dy.shape[1], scale, int(old is not None), ws),
          "bwd")
    return dw.to_np((vocab, dy.shape[1]))


@pytest.mark.parametrize("rows,vocab,cols", [(1, 1, 1), (1, 5, 4), (7, 3, 2), (33, 9, 3), (5, 300, 5), (64, 50, 8),
                                             (100, 11, 23), (257, 70, 64), (1000, 500, 65), (3, 40, 256),
                                             (333, 90, 259), (50, 60, 1024), (9, 7, 1027), (4, 5, 4099)])
@pytest.mark.parametrize("kind", ["words", "padded"])
def test_embedding(tlib, rows, vocab, cols, kind):
    rng = np.random.default_rng(rows + 31 * cols)
    w, ids = rng.standard_normal((vocab, cols)).astype(np.float32), _tokens(rng, rows, vocab, kind)
    w[0, 0] = np.inf  # reaches its own token's rows alone
    W, I, y = DevBuf.from_np(w), DevBuf.from_np(ids), DevBuf(rows * cols + 4)
    y.fill(-7.0)
    check(tlib.tt_k_embedding_fwd(W.ptr, I.ptr, y.ptr, rows, vocab, cols, 1.7), "fwd")
    got = y.to_np()
    assert np.array_equal(got[:-4].reshape(rows, cols), ref.embedding(w, ids, 1.7))
    assert (got[-4:] == -7).all()


@pytest.mark.parametrize("kind", ["words", "padded", "one", "even", "falling", "none"])
@pytest.mark.parametrize("rows,vocab,cols", [(1, 3, 4), (31, 7, 5), (32, 9, 4), (33, 40, 8), (65, 5, 1), (511, 600, 2), (512, 40, 300), (513, 50, 7), (700, 31, 3),
                                             (2048, 100, 12), (2049, 1000, 23), (4100, 1003, 259), (5000, 77, 130),
                                             (8192, 300, 20), (8193, 300, 20), (9000, 40000, 36), (70000, 5000, 8), (17000, 900, 1100), (66000, 300, 2)])
def test_embedding_gradient(tlib, rows, vocab, cols, kind):
    rng = np.random.default_rng(rows + 17 * cols)
    ids, dy = _tokens(rng, rows, vocab, kind), rng.standard_normal((rows, cols)).astype(np.float32)
    got = _grad(tlib, ids, dy, vocab, 0.37)
    close(got, ref.embedding_grad(ids, dy, vocab, 0.37), f"{rows} {vocab} {cols} {kind}")
    assert np.array_equal(got, _grad(tlib, ids, dy, vocab, 0.37))  # the sums have one order
    old = rng.standard_normal((vocab, cols)).astype(np.float32)
    got = _grad(tlib, ids, dy, vocab, 0.37, old)
    close(got, ref.embedding_grad(ids, dy, vocab, 0.37, old.astype(np.float64)))
    idle = np.setdiff1d(np.arange(vocab), ids)  # rows of no token are left as they are
    old[idle] = np.nan
    assert np.isnan(_grad(tlib, ids, dy, vocab, 0.37, old)[idle]).all()


def test_embedding_gradient_hides_padding(tlib):
    """What a padded row holds reaches nothing; an infinity reaches its token alone."""
    rng = np.random.default_rng(5)
    ids, dy = _tokens(rng, 3000, 50, "padded"), rng.standard_normal((3000, 20)).astype(np.float32)
    pad = (ids < 0) | (ids >= 50)
    clean = _grad(tlib, ids, np.where(pad[:, None], 0, dy).astype(np.float32), 50)
    dy[pad] = np.nan
    assert pad.any() and np.array_equal(_grad(tlib, ids, dy, 50), clean)
    at = int(np.flatnonzero(~pad)[0])
    dy[at, 3] = np.inf
    got = _grad(tlib, ids, dy, 50)
    assert got[ids[at], 3] == np.inf and np.isfinite(got).sum() == got.size - 1


def test_embedding_gradient_any_alignment(tlib):
    rng = np.random.default_rng(6)
    rows, vocab, cols = 300, 21, 36
    ids, dy = _tokens(rng, rows, vocab, "words"), rng.standard_normal((rows, cols)).astype(np.float32)
    want = _grad(tlib, ids, dy, vocab)
    for off in (1, 2, 3):
        g, dw = DevBuf(dy.size + 8), DevBuf(vocab * cols + 8)
        dw.fill(-7.0)
        check(tlib.tth_h2d(g.ptr + 4 * off, dy.ctypes.data, dy.nbytes), "h2d")
        i = DevBuf(rows + 4, np.int32)
        check(tlib.tth_h2d(i.ptr + 4 * off, ids.ctypes.data, ids.nbytes), "h2d")
        check(tlib.tt_k_embedding_bwd(i.ptr + 4 * off, g.ptr + 4 * off, dw.ptr + 4 * off, rows, vocab, cols, 1.0, 0,
                                      None), "bwd")
        got = dw.to_np()
        assert np.array_equal(got[off:off + want.size].reshape(want.shape), want)
        assert (got[:off] == -7).all() and (got[off + want.size:] == -7).all()


@pytest.mark.parametrize("rows", [512, 5000, 9000])
def test_embedding_workspace_allocates_nothing(tlib, rows):
    """A few rows need none."""
    rng = np.random.default_rng(7)
    vocab, cols = 300, 40
    ids, dy = _tokens(rng, rows, vocab, "words"), rng.standard_normal((rows, cols)).astype(np.float32)
    want = _grad(tlib, ids, dy, vocab)
    need = tlib.tt_k_embedding_bwd_ws(rows, vocab, cols)
    ws = DevBuf(need // 4 + 16)
    ws.fill(-7.0)
    d, g, dw = DevBuf.from_np(ids), DevBuf.from_np(dy), DevBuf(vocab * cols)
    args = [d.ptr, g.ptr, dw.ptr, rows, vocab, cols, 1.0, 0]
    assert tlib.tth_fail_alloc_after(0) == 0
    try:
        rc, none = tlib.tt_k_embedding_bwd(*args, ws.ptr), tlib.tt_k_embedding_bwd(*args, None)
    finally:
        tlib.tth_fail_alloc_after(-1)
    assert rc == 0 and none == (-2 if need else 0) and (need == 0) == (rows == 512)
    assert np.array_equal(dw.to_np(want.shape), want)
    assert (ws.to_np()[need // 4:] == -7).all()


@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_embedding_node(tlib, bound):
    """Two lookups of one table: the second one's gradient is added to the first's."""
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node
    rng = np.random.default_rng(8)
    w = rng.standard_normal((13, 6)).astype(np.float32)
    a, b = np.array([[3, 12, 3], [-1, 0, 7]], np.int32), np.array([3, 5, 13, 0, 0, 9], np.int32)
    da, db = (rng.standard_normal((6, 6)).astype(np.float32) for _ in range(2))
    W = Node.leaf(w)
    ya, yb = W.embedding(a, 2.0), W.embedding(b)
    assert np.array_equal(ya.value(), ref.embedding(w, a.ravel(), 2.0))
    assert np.array_equal(yb.value(), ref.embedding(w, b, 1.0))
    (ya * Node.leaf(da, False) + yb * Node.leaf(db, False)).backward(np.ones((6, 6), np.float32))
    one, two = ref.embedding_grad(a.ravel(), da, 13, 2.0), ref.embedding_grad(b, db, 13, 1.0)
    close(W.grad(), (one[0] + two[0], one[1] + two[1] + 2 * ref.U * (np.abs(one[0]) + np.abs(two[0]))))
    frozen = Node.leaf(w, False).embedding(b)
    frozen.backward(db)
    with pytest.raises(ValueError):
        W.embedding(np.empty(0, np.int32))
    with pytest.raises(ValueError):
        Node.leaf(w.reshape(13, 3, 2)).embedding(b)


@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_embedding_node_wide_ids(tlib, bound):
    """Ids past 32 bits are outside the table, whatever their low bits are."""
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node
    rng = np.random.default_rng(10)
    w, dy = rng.standard_normal((9, 5)).astype(np.float32), rng.standard_normal((6, 5)).astype(np.float32)
    ids = np.array([[4, 2**32 + 4, -2**32 + 1], [2**31, -1, 8]])
    W = Node.leaf(w)
    y = W.embedding(ids)
    y.backward(dy)
    want = np.zeros((6, 5), np.float32)
    want[0], want[5] = w[4], w[8]
    grad = np.zeros((9, 5), np.float32)
    grad[4], grad[8] = dy[0], dy[5]
    assert np.array_equal(y.value(), want) and np.array_equal(W.grad(), grad)
    assert np.array_equal(W.embedding([4, 8]).value(), w[[4, 8]])


def test_embedding_gradient_by_differences(tlib):
    rng = np.random.default_rng(9)
    ids, dy = _tokens(rng, 60, 17, "padded"), rng.standard_normal((60, 7)).astype(np.float32)
    w, d = rng.standard_normal((17, 7)), rng.standard_normal((17, 7))
    has = (ids >= 0) & (ids < 17)

    def f(t):
        return ((w + t * d)[ids[has]] * 1.5 * dy[has]).sum()

    g = _grad(tlib, ids, dy, 17, 1.5)
    assert abs((f(1e-3) - f(-1e-3)) / 2e-3 - (g * d).sum()) <= 1e-5 * np.abs(g * d).sum()


@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_embedding_node_ids_of_other_types(tlib, bound):
    """Ids are whole numbers by type: 1.7 is not taken for 1."""
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node
    w = np.random.default_rng(11).standard_normal((9, 5)).astype(np.float32)
    W = Node.leaf(w)
    for ids in ([1.7, 2.0], np.array([1.0, 2.0]), np.array([1, 2], np.float32), np.array([np.nan]), [1 + 0j], 2.0, ["1"],
                [], [None]):
        with pytest.raises(ValueError):
            W.embedding(ids)
    for kind in (np.int8, np.uint8, np.int16, np.uint16, np.int32, np.uint32, np.int64, np.uint64):
        ids = np.array([[3, 0, 8], [1, 1, 2]], kind)
        assert np.array_equal(W.embedding(ids).value(), w[ids.ravel().astype(int)])
        assert np.array_equal(W.embedding(ids[:, ::2]).value(), w[ids[:, ::2].ravel().astype(int)])
    assert np.array_equal(W.embedding(4).value(), w[[4]])
    top = np.array([2**64 - 1, 2**63 + 4, 5], np.uint64)  # outside, not -1 + 2^64's low bits
    assert np.array_equal(W.embedding(top).value(), np.stack([0 * w[0], 0 * w[0], w[5]]))
