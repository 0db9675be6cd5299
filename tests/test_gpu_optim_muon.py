"""Muon as an optimizer: steps of many parameters, their momenta from step to step,
and steps that cannot be made."""
import sys

import numpy as np
import pytest

import tinytorch_amd

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
