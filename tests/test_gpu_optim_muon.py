"""Muon as an optimizer: steps of many parameters, their momenta from step to step,
and steps that cannot be made."""
import sys

import numpy as np
import pytest

import tinytorch_amd
import training_ref as ref

pytestmark = pytest.mark.gpu


def _classes(bound):
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node, Optim
    else:
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node, Optim
    return Node, Optim


def _give(Node, p, g):
    """Adds g to p's gradient."""
    (p * Node.leaf(g, False)).backward(np.ones(g.shape, np.float32))


@pytest.mark.parametrize("allocations", [0, 1, 2])
def test_no_memory_for_a_step(tlib, allocations):
    """18 matrices, two runs of launches with a workspace: a step is made or it is not,
    and after one that was not the next is as if it had not been tried."""
    Node, Optim = _classes("ctypes")
    rng = np.random.default_rng(1)
    shapes = [(150, 140 + i) for i in range(16)] + [(170, 200), (300, 310)]
    w = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    grads = [[rng.standard_normal(s).astype(np.float32) for s in shapes] for _ in range(2)]
    sets = [[Node.leaf(t) for t in w] for _ in range(2)]
    opts = [Optim.muon(lr=0.05, momentum=0.9) for _ in range(2)]
    for k, g in enumerate(grads):
        for P in sets:
            for p, t in zip(P, g):
                _give(Node, p, t)
        opts[0].step(sets[0])
        if k:
            before = [p.value() for p in sets[1]]
            assert tlib.tth_fail_alloc_after(allocations) == 0
            try:
                opts[1].step(sets[1])
                made = True
            except ValueError:
                made = False
            finally:
                tlib.tth_fail_alloc_after(-1)
            assert made == (allocations > 0)
            if not made:
                for p, t in zip(sets[1], before):
                    assert np.array_equal(p.value(), t)
        if not k or not made:
            opts[1].step(sets[1])
    for a, b in zip(*sets):
        assert np.array_equal(a.value(), b.value())


# of the orthogonal factor: a rounding of the fp16 parts in a weak direction, which
# four steps multiply by their slope at 0 each
NEAR = ref.A**4 * ref.PART


def _orthogonal64(u):
    x = u if u.shape[0] <= u.shape[1] else u.T
    x = x / np.linalg.norm(x)
    for _ in range(5):
        p = x @ x.T
        x = ref.A * x + (ref.B * p + ref.C * (p @ p)) @ x
    return x if u.shape[0] <= u.shape[1] else x.T


def _step64(w, v, g, lr, mu, nesterov, decay):
    v = mu * v + g
    u = mu * v + g if nesterov else v
    rate = lr * 0.2 * np.sqrt(max(w.shape))
    return (1 - lr * decay) * w - rate * _orthogonal64(u), v, rate


@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_momenta_from_step_to_step(tlib, bound, nesterov):
    """Another gradient every step, so that u is no multiple of one: the momenta of
    each parameter count, with the optimizer's own factor and form.  One parameter has
    a gradient from the second step on, one none in the third; 18 make two runs."""
    Node, Optim = _classes(bound)
    rng = np.random.default_rng(21)
    shapes = [(6, 3, 2, 2), (40, 50), (130, 140), (5, 30)] + [(7 + i, 19) for i in range(14)]
    flat = [(s[0], int(np.prod(s[1:]))) for s in shapes]
    w = [rng.standard_normal(s).astype(np.float32).astype(np.float64) for s in shapes]
    v = [np.zeros(f) for f in flat]
    P = [Node.leaf(t.astype(np.float32)) for t in w]
    lr, mu, decay = (float(np.float32(t)) for t in (0.05, 0.9, 0.1))
    opt = Optim.muon(lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay)
    for step in range(4):
        P = [p.detach() for p in P]  # without the last step's gradients
        skipped = 1 if step == 0 else 2 if step == 2 else None
        g = [rng.standard_normal(s).astype(np.float32) for s in shapes]
        for i, p in enumerate(P):
            if i != skipped:
                _give(Node, p, g[i])
        opt.step(P)
        for i, (p, s, f) in enumerate(zip(P, shapes, flat)):
            got = p.value().astype(np.float64)
            if i == skipped:
                assert np.array_equal(got, w[i])
                continue
            args = w[i].reshape(f), v[i], g[i].astype(np.float64).reshape(f)
            want, new, rate = _step64(*args, lr, mu, nesterov, decay)
            size = np.linalg.norm(want - (1 - lr * decay) * args[0])
            tol = NEAR * size + 4 * ref.U * (np.linalg.norm(args[0]) + size)
            assert np.linalg.norm(got.reshape(f) - want) <= tol, (step, i)
            if np.abs(v[i]).max() > 0:  # from its second gradient on
                for wrong in ((0.0, nesterov), (mu, not nesterov)):
                    other = _step64(*args, lr, *wrong, decay)[0]
                    assert np.linalg.norm(other - want) > 100 * tol, (step, i, wrong)
            w[i], v[i] = got, new  # (the momenta in 64 bits: off by their own roundings, far under NEAR)
