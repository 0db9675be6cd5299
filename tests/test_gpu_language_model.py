"""The operators of a language model's training step together: tokens through a
block to the loss, its gradients against differences of the same model in 64 bits,
a step of Muon on the matrices and of Adam on the rest; a token at a time against the
whole text; and the calls captured into a graph."""
import ctypes

import numpy as np
import pytest

import training_ref as ref
import transformer_ref as tref
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

B, L, C, HEADS, D, F, V = 2, 9, 24, 3, 8, 40, 31
NAMES = ("table", "n1", "wq", "wk", "wv", "wo", "n2", "w1", "w2", "n3", "out")
MATRICES = ("wq", "wk", "wv", "wo", "w1", "w2")


def _params(seed=0):
    rng = np.random.default_rng(seed)

    def w(*s):
        return (rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)

    def norm():
        return (1 + 0.1 * rng.standard_normal(C)).astype(np.float32)

    return dict(table=0.3 * rng.standard_normal((V, C)).astype(np.float32), n1=norm(), wq=w(C, HEADS * D),
                wk=w(C, HEADS * D), wv=w(C, HEADS * D), wo=w(HEADS * D, C), n2=norm(), w1=w(C, F), w2=w(F, C), n3=norm(),
                out=w(C, V))


def _tokens(seed=1):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, V, B * L).astype(np.int32)
    ids[:3] = ids[4]  # a word that comes often
    ids[-2:] = -1  # a padded text
    return ids, rng.integers(0, V, B * L).astype(np.int32)


SCALE = 1.7


def _loss64(p, ids, labels):
    def norm(h, w):
        return h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-5) * w

    x = np.where(ids[:, None] >= 0, p["table"][ids] * SCALE, 0.0)
    h = norm(x, p["n1"])
    q, k, v = ((h @ p[n]).reshape(B, L, HEADS, D) for n in ("wq", "wk", "wv"))
    mask = tref.seen(B, L, L, causal=True)
    a = tref.attention(q, k, v, mask)["o"][0].reshape(B * L, HEADS * D) @ p["wo"]
    x = x + a
    x = x + np.maximum(norm(x, p["n2"]) @ p["w1"], 0) @ p["w2"]
    z = norm(x, p["n3"]) @ p["out"]
    z = z - z.max(1, keepdims=True)
    return -(z - np.log(np.exp(z).sum(1, keepdims=True)))[np.arange(B * L), labels].mean()


def _loss(Node, P, ids, labels):
    x = P["table"].embedding(ids, SCALE)
    h = x.rmsnorm(P["n1"])
    q, k, v = (h.matmul(P[n]) for n in ("wq", "wk", "wv"))
    a = q.attention(k, v, B, HEADS, HEADS, D, causal=True).matmul(P["wo"])
    h, x = a.rmsnorm(P["n2"], residual=x)
    a = h.matmul(P["w1"]).relu().matmul(P["w2"])
    h, x = a.rmsnorm(P["n3"], residual=x)
    return h.matmul(P["out"]).softmax_ce(labels)


@pytest.mark.parametrize("bound", ["ctypes", "pybind"])
def test_training_step(tlib, bound):
    if bound == "ctypes":
        from tinytorch_amd.torch_py import Node, Optim
    else:
        import sys
        import tinytorch_amd
        if tinytorch_amd.BUILD not in sys.path:
            sys.path.insert(0, tinytorch_amd.BUILD)
        from tinytorch_pybind import Node, Optim
    p = _params()
    ids, labels = _tokens()
    P = {n: Node.leaf(p[n]) for n in NAMES}
    loss = _loss(Node, P, ids, labels)
    p64 = {n: t.astype(np.float64) for n, t in p.items()}
    base = _loss64(p64, ids, labels)
    # a few hundred fp32 operations deep, each off by U of values near 1
    assert abs(float(loss.value().ravel()[0]) - base) <= 1e-5
    loss.backward(None)
    rng = np.random.default_rng(2)
    grads = {n: P[n].grad().astype(np.float64) for n in NAMES}
    for n in NAMES:
        for _ in range(2):
            d = rng.standard_normal(p[n].shape)
            f = [_loss64({**p64, n: p64[n] + t * d}, ids, labels) for t in (1e-5, -1e-5)]
            slope, got = (f[0] - f[1]) / 2e-5, (grads[n] * d).sum()
            # differences are good to 1e-9, the gradients to fp32 sums of some hundred terms
            assert abs(slope - got) <= 1e-7 + 1e-4 * np.abs(grads[n] * d).sum(), n
    assert (grads["table"][np.setdiff1d(np.arange(V), ids)] == 0).all()
    rest = [n for n in NAMES if n not in MATRICES]
    muon, adam = Optim.muon(lr=0.02, momentum=0.9, weight_decay=0.01), Optim.adam(lr=0.003)
    muon.step([P[n] for n in MATRICES])
    adam.step([P[n] for n in rest])
    lr, decay = float(np.float32(0.02)), float(np.float32(0.01))
    for n in MATRICES:
        u = (1 + float(np.float32(0.9))) * grads[n]  # the first step's momentum is the gradient
        x, off = ref.newton_schulz(u, 5)
        rate = lr * 0.2 * np.sqrt(max(u.shape))
        want = (1 - lr * decay) * p64[n] - rate * x
        tol = rate * (off + 4.3**5 * 6 * ref.U * 3) + 4 * ref.U * (np.linalg.norm(p64[n]) + rate * np.linalg.norm(x))
        assert np.linalg.norm(P[n].value() - want) <= tol, n
    for n in rest:
        assert np.isfinite(P[n].value()).all()
    assert float(_loss(Node, P, ids, labels).value().ravel()[0]) == pytest.approx(
        _loss64({n: P[n].value().astype(np.float64) for n in NAMES}, ids, labels), abs=1e-5)


def test_tokens_one_at_a_time(tlib):
    """Rows do not know of each other: a text's rows as they come, one by one, are
    those of the whole text, to the bit."""
    rng = np.random.default_rng(3)
    T, cols, vocab = 19, 1000, 50
    table, w = rng.standard_normal((vocab, cols)).astype(np.float32), rng.standard_normal(cols).astype(np.float32)
    ids, res = rng.integers(0, vocab, T).astype(np.int32), rng.standard_normal((T, cols)).astype(np.float32)
    dt, dw, di = DevBuf.from_np(table), DevBuf.from_np(w), DevBuf.from_np(ids)
    out = []
    for step in (T, 1):
        x, y, s = DevBuf(T * cols), DevBuf(T * cols), DevBuf.from_np(res)
        for t in range(0, T, step):
            at = 4 * t * cols
            check(tlib.tt_k_embedding_fwd(dt.ptr, di.ptr + 4 * t, x.ptr + at, step, vocab, cols, 2.0), "embedding")
            check(tlib.tt_k_rmsnorm_fwd(x.ptr + at, s.ptr + at, dw.ptr, y.ptr + at, s.ptr + at, None, step, cols, 1e-5),
                  "norm")
        out.append((y.to_np(), s.to_np()))
    for a, b in zip(*out):
        assert np.array_equal(a, b)
    x = ref.embedding(table, ids, 2.0)
    tref.close(out[0][0].reshape(T, cols), ref.rmsnorm(x, res, w)[0])


def test_calls_captured_into_a_graph(tlib):
    """With workspaces of the caller's the operators are captured and replayed over
    new inputs, with eager work in between: the eager bits each time."""
    hip = {n: getattr(tlib, n) for n in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate",
                                         "hipGraphLaunch", "hipGraphExecDestroy", "hipGraphDestroy")}
    hip["hipStreamBeginCapture"].argtypes = [ctypes.c_void_p, ctypes.c_int]
    hip["hipStreamEndCapture"].argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    hip["hipGraphInstantiate"].argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_size_t]
    for n in ("hipGraphExecDestroy", "hipGraphDestroy"):
        hip[n].argtypes = [ctypes.c_void_p]
    hip["hipGraphLaunch"].argtypes = [ctypes.c_void_p] * 2
    stream = ctypes.c_void_p(tlib.tth_stream())
    rng = np.random.default_rng(4)
    rows, vocab, cols = 9000, 700, 60  # tokens that take a merge
    shapes = [(40, 50), (300, 500), (1500, 1300), (1200, 1400)]  # by tiles of 128, all in one run
    single = [(3, 64, 64), (1, 260, 300), (2, 20, 4000)]  # a workgroup each; by tiles of 32; with shared ones
    given = dict(table=(vocab, cols), dy=(rows, cols), n=(cols,), res=(rows, cols))
    given.update({f"g{i}": s for i, s in enumerate(shapes)})
    given.update({f"s{i}": s for i, s in enumerate(single)})
    given.update({f"few{i}": (100, cols) for i in range(1)})
    ids = DevBuf(rows, np.int32)
    ins = {k: DevBuf(int(np.prod(s))) for k, s in given.items()}
    state = {f"{k}{i}": s for k in "wv" for i, s in enumerate(shapes)}

    def outputs():
        o = dict(x=rows * cols, y=rows * cols, sum=rows * cols, rstd=rows, dx=rows * cols, dn=cols, dt=vocab * cols,
                 df=vocab * cols)
        o.update({f"o{i}": int(np.prod(s)) for i, s in enumerate(single)})
        o.update({k: int(np.prod(s)) for k, s in state.items()})
        return {k: DevBuf(n) for k, n in o.items()}

    long = [(ctypes.c_long * len(shapes))(*[s[i] for s in shapes]) for i in (0, 1)]
    need = dict(emb=tlib.tt_k_embedding_bwd_ws(rows, vocab, cols), rms=tlib.tt_k_rmsnorm_bwd_ws(rows, cols),
                muon=tlib.tt_k_muon_multi_ws(*long, len(shapes)), ns=max(tlib.tt_k_newton_schulz_ws(*s) for s in single))
    assert all(need.values()) and tlib.tt_k_newton_schulz_ws(*single[0]) == 0 == tlib.tt_k_embedding_bwd_ws(100, vocab, cols)
    ws = {k: DevBuf(n // 4 + 1) for k, n in need.items()}

    def run(out):
        i, o = {n: d.ptr for n, d in ins.items()}, {n: d.ptr for n, d in out.items()}
        T = tlib
        check(T.tt_k_embedding_fwd(i["table"], ids.ptr, o["x"], rows, vocab, cols, 2.0), "embedding")
        check(T.tt_k_rmsnorm_fwd(o["x"], i["res"], i["n"], o["y"], o["sum"], o["rstd"], rows, cols, 1e-5), "norm")
        check(T.tt_k_rmsnorm_bwd(o["sum"], i["n"], i["dy"], o["y"], o["rstd"], o["dx"], o["dn"], rows, cols,
                                 ws["rms"].ptr), "norm")
        check(T.tt_k_embedding_bwd(ids.ptr, o["dx"], o["dt"], rows, vocab, cols, 2.0, 0, ws["emb"].ptr), "gradient")
        check(T.tt_k_embedding_bwd(ids.ptr, i["few0"], o["df"], 100, vocab, cols, 2.0, 0, None), "gradient")
        for k, s in enumerate(single):
            check(T.tt_k_newton_schulz(i[f"s{k}"], o[f"o{k}"], *s, 5, ws["ns"].ptr if k else None), "steps")

        def p(name, of):
            return (ctypes.c_void_p * len(shapes))(*[of[f"{name}{k}"] for k in range(len(shapes))])

        check(T.tt_k_muon_multi(p("w", o), p("g", i), p("v", o), *long, len(shapes), 0.02, 0.95, 1, 0.01,
                                ws["muon"].ptr), "muon")

    begin = {}

    def renew():
        for n, d in ins.items():
            x = rng.standard_normal(given[n]).astype(np.float32)
            check(tlib.tth_h2d(d.ptr, x.ctypes.data, x.nbytes), "h2d")
        t = rng.integers(-1, vocab, rows).astype(np.int32)
        check(tlib.tth_h2d(ids.ptr, t.ctypes.data, t.nbytes), "h2d")
        begin.update({n: rng.standard_normal(s).astype(np.float32) for n, s in state.items()})

    def reset(out):
        for n, d in out.items():
            if n in begin:
                check(tlib.tth_h2d(d.ptr, begin[n].ctypes.data, begin[n].nbytes), "h2d")
            else:
                d.fill(np.nan)

    renew()
    got, want = outputs(), outputs()
    reset(want)
    run(want)
    check(tlib.tth_sync(), "sync")
    graph, ready = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip["hipStreamBeginCapture"](stream, 1) == 0
    try:
        run(got)
    finally:
        rc = hip["hipStreamEndCapture"](stream, ctypes.byref(graph))
    assert rc == 0
    assert hip["hipGraphInstantiate"](ctypes.byref(ready), graph, None, None, 0) == 0
    try:
        for replay in range(4):
            renew()
            reset(got)
            reset(want)
            for d in ws.values():
                d.fill(np.nan)
            if replay % 2:
                run(want)
                check(tlib.tth_sync(), "sync")
            assert hip["hipGraphLaunch"](ready, stream) == 0
            check(tlib.tth_sync(), "sync")
            if replay % 2 == 0:
                run(want)
            for n in got:
                a, b = got[n].to_np(), want[n].to_np()
                assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), (replay, n)
                assert np.isfinite(a).all(), n
    finally:
        check(tlib.tth_sync(), "sync")
        assert hip["hipGraphExecDestroy"](ready) == 0
        assert hip["hipGraphDestroy"](graph) == 0


def test_updates_of_a_training_step_by_norm(tlib):
    """What Muon makes of a model's own gradients, some of low rank: as near as of any
    matrix, two steps on."""
    from tinytorch_amd.torch_py import Node, Optim
    p = _params(5)
    P = {n: Node.leaf(p[n]) for n in NAMES}
    lr, mu, decay = (float(np.float32(t)) for t in (0.02, 0.9, 0.01))
    muon, v = Optim.muon(lr=lr, momentum=mu, weight_decay=decay), {n: 0.0 for n in MATRICES}
    near = ref.A**4 * ref.PART  # a rounding of the products' parts through four steps' slope at 0
    for step in range(2):
        P = {n: t.detach() for n, t in P.items()}
        _loss(Node, P, *_tokens(step)).backward(None)
        before = {n: P[n].value().astype(np.float64) for n in MATRICES}
        grads = {n: P[n].grad().astype(np.float64) for n in MATRICES}
        muon.step([P[n] for n in MATRICES])
        for n in MATRICES:
            v[n] = mu * v[n] + grads[n]
            x, _ = ref.newton_schulz(mu * v[n] + grads[n], 5)
            new = -lr * 0.2 * np.sqrt(max(x.shape)) * x
            off = np.linalg.norm(P[n].value() - (1 - lr * decay) * before[n] - new)
            size = np.linalg.norm(new)
            assert off <= near * size + 4 * ref.U * (np.linalg.norm(before[n]) + size), (step, n, off / size)
