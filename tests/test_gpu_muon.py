"""Newton-Schulz steps and the optimizer around them, against 64 bits: matrices of
every kind of shape, several at once, and what the steps are for (singular values)."""
import ctypes

import numpy as np
import pytest

import training_ref as ref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

# How near the steps come where roundings do not all add up: one of the fp16 parts',
# 2^-22, in a weak direction, which four steps multiply by their slope at 0 each
# while the strong ones stay near 1.
NEAR = ref.A**4 * ref.PART

SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (4, 31), (32, 32), (33, 32), (31, 65), (10, 785), (129, 10), (64, 64),
          (65, 127), (100, 333), (257, 128), (128, 129), (150, 2100), (1030, 70), (31, 1100), (60, 500), (90, 260),
          (120, 160), (160, 128), (129, 129), (300, 300)]


def _matrix(rows, cols, kind="full", seed=0):
    rng = np.random.default_rng(rows * 1000 + cols + seed)
    x = rng.standard_normal((rows, cols))
    if kind == "steep":  # a few strong directions
        few = max(1, min(rows, cols) // 16)
        x = 0.1 * x + rng.standard_normal((rows, few)) @ rng.standard_normal((few, cols))
    return x.astype(np.float32)


def _steps(L, x, steps, ws=None, in_place=False):
    x = np.ascontiguousarray(x)
    count = x.shape[0] if x.ndim == 3 else 1
    X = DevBuf.from_np(x)
    y = X if in_place else DevBuf(x.size + 4)
    if not in_place:
        y.fill(-7.0)
    check(L.tt_k_newton_schulz(X.ptr, y.ptr, count, *x.shape[-2:], steps, ws), "newton_schulz")
    got = y.to_np()
    assert in_place or (got[-4:] == -7).all()
    return got[:x.size].reshape(x.shape)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_one_step(tlib, rows, cols):
    """A single step, value by value."""
    x = _matrix(rows, cols)
    want, tol = ref.one_step(*ref.normed(x))
    if rows > cols:
        want, tol = want.T, tol.T
    got = _steps(tlib, x, 1)
    assert (np.abs(got - want) <= tol + ref.U * np.abs(want)).all(), np.max(np.abs(got - want) / tol)
    assert np.array_equal(got, _steps(tlib, x, 1, in_place=True))


@pytest.mark.parametrize("kind", ["full", "steep"])
@pytest.mark.parametrize("rows,cols", SHAPES + [(300, 1000), (520, 515)])
def test_steps(tlib, rows, cols, kind):
    x = _matrix(rows, cols, kind)
    for steps in (2, 5):
        want, tol = ref.newton_schulz(x, steps)
        got = _steps(tlib, x, steps)
        off = np.linalg.norm(got - want)
        assert off <= tol, (steps, off, tol)
        assert off <= NEAR * np.linalg.norm(want), (steps, off / np.linalg.norm(want))


@pytest.mark.parametrize("rows,cols", [(5, 4000), (3101, 60), (100, 8000), (40, 70001), (220, 3500)])
def test_one_step_long(tlib, rows, cols):
    """Few rows of a long product: its length is shared."""
    x = _matrix(rows, cols)
    want, tol = ref.one_step(*ref.normed(x))
    if rows > cols:
        want, tol = want.T, tol.T
    got = _steps(tlib, x, 1)
    assert (np.abs(got - want) <= tol + ref.U * np.abs(want)).all(), np.max(np.abs(got - want) / tol)
    ws = DevBuf(tlib.tt_k_newton_schulz_ws(1, rows, cols) // 4 + 16)
    ws.fill(np.nan)
    assert np.array_equal(got, _steps(tlib, x, 1, ws.ptr))
    assert np.isnan(ws.to_np()[-16:]).all()
    want, tol = ref.newton_schulz(x, 5)
    got = _steps(tlib, np.stack([x, x[::-1], x]), 5)
    for g, w in zip(got, (want, want[::-1], want)):
        assert np.linalg.norm(g - w) <= min(tol, NEAR * np.linalg.norm(want))


@pytest.mark.parametrize("rows,cols", [(1430, 1400), (1060, 2600)])
def test_one_step_large(tlib, rows, cols):
    """By tiles of 128: value by value."""
    x = _matrix(rows, cols)
    want, tol = ref.one_step(*ref.normed(x))
    if rows > cols:
        want, tol = want.T, tol.T
    got = _steps(tlib, x, 1)
    assert (np.abs(got - want) <= tol + ref.U * np.abs(want)).all(), np.max(np.abs(got - want) / tol)


def _steps64(x, steps):
    x = x.astype(np.float64)
    y = x.T if x.shape[0] > x.shape[1] else x
    y = y / np.linalg.norm(y)
    for _ in range(steps):
        p = y @ y.T
        y = ref.A * y + (ref.B * p + ref.C * (p @ p)) @ y
    return y.T if x.shape[0] > x.shape[1] else y


@pytest.mark.parametrize("shape,steps", [((1390, 1470), 5), ((1700, 1290), 5), ((2100, 7010), 4), ((7003, 2101), 3),
                                         ((3, 1020, 1010), 5), ((130, 150, 155), 5)])
def test_steps_large(tlib, shape, steps):
    """By tiles of 128 and 256, upright and turned, one matrix and several."""
    x = np.random.default_rng(7).standard_normal(shape).astype(np.float32)
    got = _steps(tlib, x, steps)
    for i in ((0, shape[0] - 1) if len(shape) == 3 else (slice(None),)):
        want = _steps64(x[i], steps)
        off = np.linalg.norm(got[i] - want) / np.linalg.norm(want)
        assert off <= NEAR, off
        big = np.abs(got[i] - want).max() / np.sqrt((want**2).mean())
        assert big <= 40 * NEAR, big  # of some millions of values none is off by many times the rest
    assert np.array_equal(got, _steps(tlib, x, steps, in_place=True))
    more = 1 << 10
    need = tlib.tt_k_newton_schulz_ws(x.size // (shape[-1] * shape[-2]), *shape[-2:])
    ws = DevBuf(need // 4 + more)
    ws.fill(np.nan)
    assert np.array_equal(got, _steps(tlib, x, steps, ws.ptr))  # what a workspace holds before does not count
    assert np.isnan(ws.to_np()[-more:]).all()


@pytest.mark.parametrize("m,n,count", [(3300, 3400, 1), (4430, 4450, 2)])
def test_one_step_larger(tlib, m, n, count):
    """The symmetric products by tiles of 128 where the last one is by 256, and by 256."""
    x = np.random.default_rng(8).standard_normal((m, n)).astype(np.float32)
    got = _steps(tlib, np.stack([x] * count), 1)
    want = _steps64(x, 1)
    for g in got:
        assert np.linalg.norm(g - want) <= NEAR * np.linalg.norm(want)
        assert np.abs(g - want).max() <= 40 * NEAR * np.sqrt((want**2).mean())


def test_steps_take_singular_values(tlib):
    """From known singular vectors: a s + b s^3 + c s^5, five times."""
    rng = np.random.default_rng(3)
    u, v = np.linalg.qr(rng.standard_normal((60, 60)))[0], np.linalg.qr(rng.standard_normal((200, 60)))[0]
    s = np.geomspace(1.0, 3e-3, 60)
    x = ((u * s) @ v.T).astype(np.float32)
    s = s / np.linalg.norm(s)
    for _ in range(5):
        s = ref.A * s + ref.B * s**3 + ref.C * s**5
    got = _steps(tlib, x, 5).astype(np.float64)
    # x's own rounding, U of its norm, grows by the steps' slopes too
    tol = NEAR + ref.A**5 * ref.U
    assert np.abs(u.T @ got @ v - np.diag(s)).max() <= tol


@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-30, 1e-10, 1e10, 1e30, 3e37])
def test_steps_at_any_scale(tlib, scale):
    """The squares of tiny and huge values are within the norm's range."""
    x = _matrix(20, 45)
    small = (x * np.float64(scale)).astype(np.float32)
    want, tol = ref.newton_schulz(small.astype(np.float64), 5)
    assert np.linalg.norm(_steps(tlib, small, 5) - want) <= tol


def test_steps_of_zeros_and_bad_values(tlib):
    assert (_steps(tlib, np.zeros((40, 70), np.float32), 5) == 0).all()
    for bad in (np.nan, np.inf):
        x = _matrix(40, 70)
        x[3, 5] = bad
        assert np.isnan(_steps(tlib, x, 5)).all()
    x = np.zeros((50, 33), np.float32)
    x[7, 9] = -2.0  # one direction: its value is that of 1
    s = 1.0
    for _ in range(5):
        s = ref.A * s + ref.B * s**3 + ref.C * s**5
    want = np.zeros_like(x)
    want[7, 9] = -s
    assert np.abs(_steps(tlib, x, 5) - want).max() <= 1e-5


@pytest.mark.parametrize("rows,cols", [(37, 50), (150, 140)])
@pytest.mark.parametrize("count", [1, 2, 17, 64, 65, 140])
def test_steps_of_many(tlib, count, rows, cols):
    """Each as alone, whatever the others hold."""
    x = np.stack([_matrix(rows, cols, seed=i) for i in range(count)])
    if count > 2:
        x[1] = np.nan
    got = _steps(tlib, x, 5)
    for i in {0, min(1, count - 1), count // 2, count - 1}:
        one = _steps(tlib, x[i], 5)
        assert np.array_equal(got[i], one, equal_nan=True)
    ws = DevBuf(tlib.tt_k_newton_schulz_ws(count, rows, cols) // 4 + 16)
    ws.fill(-7.0)
    assert np.array_equal(_steps(tlib, x, 5, ws.ptr), got, equal_nan=True)
    assert (ws.to_np()[-16:] == -7).all()


@pytest.mark.parametrize("count", [3, 31, 32, 40])
def test_steps_of_many_with_blocks(tlib, count):
    """Matrices of many blocks that fit LDS: together they have a workgroup each from 32
    on, and fewer of them go product by product."""
    rows, cols = 95, 300
    assert (tlib.tt_k_newton_schulz_ws(count, rows, cols) == 0) == (count >= 32)
    x = np.stack([_matrix(rows, cols, seed=i) for i in range(count)])
    got = _steps(tlib, x, 5)
    for i in {0, 1, count // 2, count - 1}:
        want, off = ref.newton_schulz(x[i], 5)
        assert np.linalg.norm(got[i] - want) <= off
        assert np.linalg.norm(got[i] - want) <= NEAR * np.linalg.norm(want)


def _ptrs(ds):
    return (ctypes.c_void_p * len(ds))(*[d.ptr for d in ds])


def _long(xs):
    return (ctypes.c_long * len(xs))(*xs)


def _muon64(w, g, v, lr, mu, nesterov, decay):
    """The step, and a bound of its weights' error's 2-norm; v's is exact to two
    roundings."""
    w, g, v = (t.astype(np.float64) for t in (w, g, v))
    v = mu * v + g
    u = mu * v + g if nesterov else v
    x, off = ref.newton_schulz(u, 5)
    # the momenta's and u's own roundings: 5 of them, through slopes of 4 at most
    off = off + 4.3**5 * 5 * ref.U * np.linalg.norm(np.abs(u) + np.abs(mu * v) + np.abs(g)) / max(np.linalg.norm(u), 1e-300)
    rate = lr * 0.2 * np.sqrt(max(w.shape))
    new = (1 - lr * decay) * w - rate * x
    return new, v, rate * off + 4 * ref.U * (np.linalg.norm(w) + rate * np.linalg.norm(x))


@pytest.mark.parametrize("nesterov", [0, 1])
@pytest.mark.parametrize("shapes", [[(30, 50)], [(785, 256), (257, 128), (129, 10)],
                                    [(5, 7), (64, 64), (33, 400), (200, 20), (1, 9)],
                                    [(3 + i, 40 - 2 * i) for i in range(16)],
                                    [(1100, 1300), (33, 50), (1200, 1000), (700, 2000)]])
def test_muon_step(tlib, shapes, nesterov):
    rng = np.random.default_rng(4)
    w, g, v = ([rng.standard_normal(s).astype(np.float32) for s in shapes] for _ in range(3))
    W, G, V = ([DevBuf.from_np(t) for t in ts] for ts in (w, g, v))
    rows, cols = _long([s[0] for s in shapes]), _long([s[1] for s in shapes])
    lr, mu, decay = np.float32(0.02), np.float32(0.95), np.float32(0.1)
    ws = DevBuf(tlib.tt_k_muon_multi_ws(rows, cols, len(shapes)) // 4)
    for k in range(2):
        check(tlib.tt_k_muon_multi(_ptrs(W), _ptrs(G), _ptrs(V), rows, cols, len(shapes), lr, mu, nesterov, decay,
                                   ws.ptr if k else None), "muon")
        for i, s in enumerate(shapes):
            want, vel, tol = _muon64(w[i], g[i], v[i], float(lr), float(mu), nesterov, float(decay))
            got, v_got = W[i].to_np(s), V[i].to_np(s)
            bound = 2 * ref.U * (np.abs(float(mu) * v[i].astype(np.float64)) + np.abs(g[i]) + np.abs(vel))
            assert (np.abs(v_got - vel) <= bound).all()
            assert np.linalg.norm(got - want) <= tol
            assert np.linalg.norm(got - want) <= 2 * NEAR * np.linalg.norm(want - w[i]) + 4 * ref.U * np.linalg.norm(w[i])
            w[i], v[i] = got, v_got
            assert np.array_equal(G[i].to_np(s), g[i])


@pytest.mark.parametrize("shapes", [[(1500, 1600), (1400, 5), (2000, 900), (60, 1900), (900, 900), (40, 3000)],
                                    [(64, 4000), (30, 50), (129, 3300), (5000, 9)],
                                    [(2200, 6300), (6000, 9), (33, 2100), (500, 400)], [(3250, 3260), (40, 50)]])
def test_muon_step_large_and_small(tlib, shapes):
    """Tiles of many lengths of product, dealt to workgroups together."""
    rng = np.random.default_rng(5)
    w, g, v = ([rng.standard_normal(s).astype(np.float32) for s in shapes] for _ in range(3))
    W, G, V = ([DevBuf.from_np(t) for t in ts] for ts in (w, g, v))
    rows, cols = _long([s[0] for s in shapes]), _long([s[1] for s in shapes])
    need = tlib.tt_k_muon_multi_ws(rows, cols, len(shapes)) // 4
    ws = DevBuf(need + 16)
    ws.fill(np.nan)
    lr, mu, decay = np.float32(0.02), np.float32(0.95), np.float32(0.1)
    check(tlib.tt_k_muon_multi(_ptrs(W), _ptrs(G), _ptrs(V), rows, cols, len(shapes), lr, mu, 1, decay, ws.ptr), "muon")
    assert np.isnan(ws.to_np()[need:]).all()
    for i, s in enumerate(shapes):
        want, _, tol = _muon64(w[i], g[i], v[i], float(lr), float(mu), 1, float(decay))
        got = W[i].to_np(s)
        assert np.linalg.norm(got - want) <= tol
        assert np.linalg.norm(got - want) <= 2 * NEAR * np.linalg.norm(want - w[i]) + 4 * ref.U * np.linalg.norm(w[i])


@pytest.mark.parametrize("rows,cols", [(70, 90), (270, 390)])
def test_muon_workspace_allocates_nothing(tlib, rows, cols):
    """The smaller needs none."""
    x = _matrix(rows, cols)
    want = _steps(tlib, x, 5)
    need = tlib.tt_k_newton_schulz_ws(1, rows, cols)
    X, y, ws = DevBuf.from_np(x), DevBuf(x.size), DevBuf(need // 4 + 1)
    w, g, v = (DevBuf.from_np(_matrix(rows, cols, seed=s)) for s in (1, 2, 3))
    wss = DevBuf(tlib.tt_k_muon_multi_ws(_long([rows]), _long([cols]), 1) // 4 + 1)
    assert (need == 0) == (rows == 70)
    assert tlib.tth_fail_alloc_after(0) == 0
    try:
        rc = [tlib.tt_k_newton_schulz(X.ptr, y.ptr, 1, rows, cols, 5, ws.ptr),
              tlib.tt_k_newton_schulz(X.ptr, y.ptr, 1, rows, cols, 5, None)]
        for p in (wss.ptr, None):
            rc.append(tlib.tt_k_muon_multi(_ptrs([w]), _ptrs([g]), _ptrs([v]), _long([rows]), _long([cols]), 1, 0.1,
                                           0.9, 1, 0.0, p))
    finally:
        tlib.tth_fail_alloc_after(-1)
    assert rc == ([0, -2, 0, -2] if need else [0] * 4)
    assert np.array_equal(y.to_np(x.shape), want)


@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_optim_muon(tlib, bound):
    """18 parameters (two runs of launches), of which one has no gradient and some
    have more than two axes; a new rate between the steps."""
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node, Optim
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node, Optim
    rng = np.random.default_rng(11)
    shapes = [(6, 3, 2, 2), (5, 2, 3)] + [(4 + i, 9) for i in range(16)]
    w = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    g = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    v = [np.zeros_like(t) for t in w]
    P = [Node.leaf(t) for t in w]
    opt = Optim.muon(lr=0.05, momentum=0.9, nesterov=True, weight_decay=0.2)
    for lr in (0.05, 0.01):
        opt.lr = lr
        for i, p in enumerate(P):
            if i != 3 and lr == 0.05:
                (p * Node.leaf(g[i], False)).backward(np.ones(shapes[i], np.float32))
        opt.step(P)
        for i, p in enumerate(P):
            if i == 3:
                assert np.array_equal(p.value(), w[i])
                continue
            flat = (shapes[i][0], -1)
            args = [t.reshape(flat) for t in (w[i], g[i], v[i])]
            want, vel, tol = _muon64(*args, float(np.float32(lr)), float(np.float32(0.9)), 1, float(np.float32(0.2)))
            got = p.value()
            # the momenta are the 64-bit ones here, off by their own two roundings
            assert np.linalg.norm(got.reshape(flat) - want) <= 2 * tol
            w[i], v[i] = got, vel.astype(np.float32).reshape(shapes[i])


def test_optim_muon_refuses(tlib):
    from tinytorch_amd.torch_py import Node, Optim
    rng = np.random.default_rng(12)
    a, b = Node.leaf(rng.standard_normal((4, 5))), Node.leaf(rng.standard_normal(5))
    for n in (a, b):
        n.backward(np.ones(n.value().shape, np.float32))
    before = a.value()
    for params in ([a, b], [a, a.detach()], [b]):
        opt = Optim.muon()
        with pytest.raises(ValueError):
            opt.step(params)
        assert np.array_equal(a.value(), before)
    opt = Optim.muon()
    opt.step([a])
    with pytest.raises(ValueError):
        opt.step([b])
    assert not np.array_equal(a.value(), before)
    with pytest.raises(ValueError):
        Optim.muon(lr=float("nan"))
