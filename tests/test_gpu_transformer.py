"""The transformer operators together: a block trained by distillation, its
gradients against differences of the same block in 64 bits; and tokens
answered one at a time from a cache, against the whole text at once."""
import ctypes

import numpy as np
import pytest

import transformer_ref as ref
from tinytorch_amd import Attention, Rope, Strides
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu

B, L, C, HQ, HKV, D, F, V, TOP = 2, 11, 24, 4, 2, 8, 40, 30, 4
LENGTHS = np.array([11, 7], np.int32)
ZERO = np.zeros(B, np.int32)


def _params(seed=0):
    rng = np.random.default_rng(seed)

    def w(*s):
        return (rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)

    return dict(n1w=1 + 0.1 * rng.standard_normal(C).astype(np.float32), n1b=w(C), wq=w(C, HQ * D), wk=w(C, HKV * D),
                wv=w(C, HKV * D), wo=w(HQ * D, C), n2w=1 + 0.1 * rng.standard_normal(C).astype(np.float32), n2b=w(C),
                w1=w(C, F), w2=w(F, C), out=w(C, V))


def _data(seed=1):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((B * L, C)).astype(np.float32)
    ids = np.stack([rng.permutation(V)[:TOP] for _ in range(B * L)]).astype(np.int32)
    ids[L + 7:] = -1  # rows behind the second text teach nothing
    return x, ids, (3 + rng.standard_normal((B * L, TOP))).astype(np.float32)


def _block64(x, p, ids, teacher):
    f = ref.frequencies(D, 10000.0)
    pos = np.arange(B * L) % L

    def norm(h, w, b):
        d = h - h.mean(1, keepdims=True)
        return d / np.sqrt((d * d).mean(1, keepdims=True) + 1e-5) * w + b

    def heads(h, w, n):
        return (h @ w).reshape(B * L, n, D)

    h = norm(x, p["n1w"], p["n1b"])
    q = ref.rope(heads(h, p["wq"], HQ), pos, f, False)[0].reshape(B, L, HQ, D)
    k = ref.rope(heads(h, p["wk"], HKV), pos, f, False)[0].reshape(B, L, HKV, D)
    v = heads(h, p["wv"], HKV).reshape(B, L, HKV, D)
    mask = ref.seen(B, L, L, causal=True, q_start=ZERO, q_len=LENGTHS, k_len=LENGTHS)
    x = x + ref.attention(q, k, v, mask)["o"][0].reshape(B * L, HQ * D) @ p["wo"]
    x = x + np.maximum(norm(x, p["n2w"], p["n2b"]) @ p["w1"], 0) @ p["w2"]
    z = norm(x, 1.0, 0.0) @ p["out"]
    return ref.distill(z, ids, teacher, 2.0, 1.0)[0][0].mean()


def _block(x, p, ids, teacher, backend):
    """The block's nodes on the framework: parameters and loss."""
    N = backend
    n = {k: N.leaf(v, True) for k, v in p.items()}
    X = N.leaf(x, True)
    h = X.layernorm(n["n1w"], n["n1b"])
    q = h.matmul(n["wq"]).rope(HQ, D, seq_len=L)
    k = h.matmul(n["wk"]).rope(HKV, D, seq_len=L)
    a = q.attention(k, h.matmul(n["wv"]), batch=B, q_heads=HQ, kv_heads=HKV, head_dim=D, causal=True, q_start=ZERO,
                    q_len=LENGTHS, k_len=LENGTHS)
    y = X + a.matmul(n["wo"])
    y = y + y.layernorm(n["n2w"], n["n2b"]).matmul(n["w1"]).relu().matmul(n["w2"])
    loss = y.layernorm().matmul(n["out"]).distill(ids, teacher, 2.0)
    n["x"] = X
    return n, loss


def _backends():
    import importlib
    import os
    import sys
    import tinytorch_amd
    from tinytorch_amd.torch_py import Node
    sys.path.insert(0, os.path.join(tinytorch_amd.ROOT, "build"))
    try:
        m = importlib.import_module("tinytorch_pybind")
    finally:
        sys.path.pop(0)
    return [Node, m.Node]


def test_block_gradients(tlib):
    p = _params()
    x, ids, teacher = _data()
    p64 = {k: v.astype(np.float64) for k, v in p.items()}
    want = _block64(x.astype(np.float64), p64, ids, teacher)
    grads = []
    for N in _backends():
        n, loss = _block(x, p, ids, teacher, N)
        assert abs(loss.value()[0] - want) <= 1e-5 * want
        loss.backward(None)
        grads.append({k: v.grad() for k, v in n.items()})
    for k in grads[0]:  # the same calls through either binding
        assert np.array_equal(grads[0][k], grads[1][k]), k
    # each gradient along a direction of its own: the differences are good to
    # about 1e-8 of the loss over the step, the gradients to sums of fp32
    rng = np.random.default_rng(4)
    for k, g in grads[0].items():
        d = rng.standard_normal(g.shape)
        f = []
        for s in (1e-6, -1e-6):
            q = dict(p64)
            xx = x.astype(np.float64)
            if k == "x":
                xx = xx + s * d
            else:
                q[k] = q[k] + s * d
            f.append(_block64(xx, q, ids, teacher))
        slope = (f[0] - f[1]) / 2e-6
        assert abs(slope - (g * d).sum()) <= 2e-5 * np.abs(g * d).sum() + 1e-8, k
    assert not grads[0]["x"].reshape(B, L, C)[1, 7:].any()


def test_block_steps(tlib):
    """Steps of an optimizer over the block's parameters run and move every one."""
    from tinytorch_amd.torch_py import Node, Optim
    p = _params()
    x, ids, teacher = _data()
    n, loss = _block(x, p, ids, teacher, Node)
    names = [k for k in n if k != "x"]
    opt = Optim.adam(0.01)
    before = {k: n[k].value() for k in names}
    loss.backward(None)
    opt.step([n[k] for k in names])
    for k in names:
        assert np.isfinite(n[k].value()).all() and not np.array_equal(n[k].value(), before[k]), k


@pytest.mark.parametrize("interleaved", [False, True])
def test_tokens_from_a_cache(tlib, interleaved):
    """Each token's key goes turned into its cache row, and its query reads
    what is there: the rows of the whole text at once."""
    T, cap = 37, 64
    rng = np.random.default_rng(8)
    qkv = rng.standard_normal((T, (HQ + 2 * HKV) * 16)).astype(np.float32)
    r = Rope(16, 16, int(interleaved), 3, 10000.0, 8.0, 8192.0, 1.0, 32.0, 0.0)
    row, kw = qkv.shape[1], HKV * 16
    buf, pos = DevBuf.from_np(qkv), DevBuf.from_np(np.arange(T, dtype=np.int32))
    held = DevBuf.from_np(np.arange(1, T + 1, dtype=np.int32))
    ck, cv, turned, o = DevBuf(cap * kw), DevBuf(cap * kw), DevBuf(HQ * 16), DevBuf(T * HQ * 16)
    ck.fill(np.nan)
    cv.fill(np.nan)
    for t in range(T):
        at = buf.ptr + 4 * t * row
        check(tlib.tt_k_rope(r, at, turned.ptr, pos.ptr + 4 * t, 1, 0, HQ, 0, 0, 0), "rope q")
        check(tlib.tt_k_rope(r, at + 4 * HQ * 16, ck.ptr + 4 * t * kw, pos.ptr + 4 * t, 1, 0, HKV, 0, 0, 0), "rope k")
        check(tlib.tt_k_copy(cv.ptr + 4 * t * kw, at + 4 * (HQ + HKV) * 16, kw), "v")
        a = Attention(batch=1, q_rows=1, k_rows=cap, q_heads=HQ, kv_heads=HKV, head_dim=16, causal=1,
                      q_start=pos.ptr + 4 * t, k_len=held.ptr + 4 * t)
        check(tlib.tt_k_attention_fwd(a, turned.ptr, ck.ptr, cv.ptr, o.ptr + 4 * t * HQ * 16, None, None), "attn")
    got = o.to_np((1, T, HQ, 16))
    # at once, q and k turned in the joint buffer
    both = DevBuf(T * row)
    check(tlib.tt_k_copy(both.ptr, buf.ptr, T * row), "copy")
    check(tlib.tt_k_rope(r, both.ptr, both.ptr, None, T, T, HQ + HKV, row, row, 0), "rope")
    s = Strides(0, row, 0)
    a = Attention(batch=1, q_rows=T, k_rows=T, q_heads=HQ, kv_heads=HKV, head_dim=16, causal=1, q=s, k=s, v=s)
    check(tlib.tt_k_attention_fwd(a, both.ptr, both.ptr + 4 * HQ * 16, both.ptr + 4 * (HQ + HKV) * 16, o.ptr, None,
                                  None), "attn")
    whole = o.to_np((1, T, HQ, 16))
    x = both.to_np((1, T, HQ + 2 * HKV, 16))
    want = ref.attention(x[:, :, :HQ], x[:, :, HQ:HQ + HKV], x[:, :, HQ + HKV:], ref.seen(1, T, T, causal=True))["o"]
    ref.close(whole, want)
    ref.close(got, want)


def test_calls_captured_into_a_graph(tlib):
    """With workspaces of the caller's the operators are captured, forward and
    backward, and replayed over new inputs with eager work in between: the
    eager bits each time."""
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
    nb, rows, hq, hkv, dim, cols, top = 2, 300, 8, 2, 32, 500, 6
    rope = Rope(head_dim=dim, rot_dim=dim, base=10000.0)
    shapes = dict(x=(nb * rows, hq * dim), w=(hq * dim,), k=(nb * rows, hkv * dim), v=(nb * rows, hkv * dim),
                  do=(nb * rows, hq * dim), z=(nb * rows, cols), teacher=(nb * rows, top))
    given = {n: DevBuf(int(np.prod(s))) for n, s in shapes.items()}
    ids = DevBuf.from_np(rng.integers(0, cols, (nb * rows, top)).astype(np.int32))
    wide, narrow, per_row = nb * rows * hq * dim, nb * rows * hkv * dim, nb * rows

    def outputs():
        return dict(y=DevBuf(wide), mean=DevBuf(per_row), rstd=DevBuf(per_row), q=DevBuf(wide), o=DevBuf(wide),
                    one=DevBuf(nb * hq * dim), lse=DevBuf(nb * hq * rows), dq=DevBuf(wide), dk=DevBuf(narrow),
                    dv=DevBuf(narrow), dy=DevBuf(wide), dx=DevBuf(wide), dw=DevBuf(hq * dim), db=DevBuf(hq * dim),
                    loss=DevBuf(per_row), dz=DevBuf(per_row * cols))

    a = Attention(batch=nb, q_rows=rows, k_rows=rows, q_heads=hq, kv_heads=hkv, head_dim=dim, causal=1)
    few = Attention(batch=nb, q_rows=1, k_rows=rows, q_heads=hq, kv_heads=hkv, head_dim=dim)
    need = (tlib.tt_k_attention_fwd_ws(a), tlib.tt_k_attention_fwd_ws(few), tlib.tt_k_attention_bwd_ws(a),
            tlib.tt_k_layernorm_bwd_ws(per_row, hq * dim))
    assert need[0] and need[1] and need[2] and need[3]
    ws = [DevBuf(n // 4 + 1) for n in need]

    def run(out):
        o = {n: d.ptr for n, d in out.items()}
        i = {n: d.ptr for n, d in given.items()}
        L = tlib
        check(L.tt_k_layernorm_fwd(i["x"], i["w"], None, o["y"], o["mean"], o["rstd"], per_row, hq * dim, 1e-5), "ln")
        check(L.tt_k_rope(rope, o["y"], o["q"], None, per_row, rows, hq, 0, 0, 0), "rope")
        check(L.tt_k_attention_fwd(a, o["q"], i["k"], i["v"], o["o"], o["lse"], ws[0].ptr), "attention")
        check(L.tt_k_attention_fwd(few, o["q"], i["k"], i["v"], o["one"], None, ws[1].ptr), "attention")
        check(L.tt_k_attention_bwd(a, o["q"], i["k"], i["v"], o["o"], i["do"], o["lse"], o["dq"], o["dk"], o["dv"],
                                   ws[2].ptr), "attention")
        check(L.tt_k_rope(rope, o["dq"], o["dy"], None, per_row, rows, hq, 0, 0, 1), "rope")
        check(L.tt_k_layernorm_bwd(i["x"], i["w"], o["dy"], o["mean"], o["rstd"], o["dx"], o["dw"], o["db"], per_row,
                                   hq * dim, ws[3].ptr), "ln")
        check(L.tt_k_distill(i["z"], ids.ptr, i["teacher"], top, 2.0, o["loss"], o["dz"], per_row, cols, 1.0), "distill")

    def renew():
        for n, d in given.items():
            x = rng.standard_normal(shapes[n]).astype(np.float32)
            check(tlib.tth_h2d(d.ptr, x.ctypes.data, x.nbytes), "h2d")

    renew()
    got, want = outputs(), outputs()
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
            for d in got.values():
                d.fill(np.nan)
            for d in ws:
                d.fill(np.nan)
            if replay % 2:
                run(want)
                check(tlib.tth_sync(), "sync")
            assert hip["hipGraphLaunch"](ready, stream) == 0
            check(tlib.tth_sync(), "sync")
            if replay % 2 == 0:
                run(want)
            for n in got:
                assert np.array_equal(got[n].to_np().view(np.uint32), want[n].to_np().view(np.uint32)), (replay, n)
                assert np.isfinite(got[n].to_np()).all(), n
    finally:
        check(tlib.tth_sync(), "sync")
        assert hip["hipGraphExecDestroy"](ready) == 0
        assert hip["hipGraphDestroy"](graph) == 0
