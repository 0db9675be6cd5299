"""Attention, forward and backward, against 64 bits: head sizes, heads that
share keys, lengths from one row, masks that leave rows empty, layouts, and
what may lie where a mask hides it."""
import ctypes

import numpy as np
import pytest

import transformer_ref as ref
from tinytorch_amd import Attention, Strides
from tinytorch_amd.hip import DevBuf, check

pytestmark = pytest.mark.gpu


def _inputs(B, Lq, Lk, Hq, Hkv, D, seed=0):
    rng = np.random.default_rng([B, Lq, Lk, Hq, Hkv, D, seed])
    return tuple(rng.standard_normal(s).astype(np.float32)
                 for s in ((B, Lq, Hq, D), (B, Lk, Hkv, D), (B, Lk, Hkv, D), (B, Lq, Hq, D)))


def _ints(x):
    return None if x is None else DevBuf.from_np(np.asarray(x, np.int32))


def _plan(q, k, masks, held, scale=0.0, /, **layout):
    B, Lq, Hq, D = q.shape
    a = Attention(batch=B, q_rows=Lq, k_rows=k.shape[1], q_heads=Hq, kv_heads=k.shape[2], head_dim=D,
                  causal=int(masks.get("causal", False)), window=masks.get("window", 0), scale=scale, **layout)
    for n in ("q_start", "q_len", "k_len"):
        d = _ints(masks.get(n))
        if d is not None:
            held.append(d)
            setattr(a, n, d.ptr)
    return a


def _run(L, q, k, v, do, masks, scale=0.0, ws=None):
    held = []
    a = _plan(q, k, masks, held, scale)
    dq_, dk_, dv_, do_ = (DevBuf.from_np(t) for t in (q, k, v, do))
    B, Lq, Hq, D = q.shape
    o, lse = DevBuf(q.size), DevBuf(B * Hq * Lq)
    out = [DevBuf(t.size) for t in (q, k, v)]
    for d in [o, lse] + out:
        d.fill(np.nan)
    check(L.tt_k_attention_fwd(a, dq_.ptr, dk_.ptr, dv_.ptr, o.ptr, lse.ptr, ws), "fwd")
    check(L.tt_k_attention_bwd(a, dq_.ptr, dk_.ptr, dv_.ptr, o.ptr, do_.ptr, lse.ptr, *[x.ptr for x in out], ws),
          "bwd")
    return dict(o=o.to_np(q.shape), lse=lse.to_np((B, Hq, Lq)), dq=out[0].to_np(q.shape),
                dk=out[1].to_np(k.shape), dv=out[2].to_np(v.shape))


def _check(L, q, k, v, do, masks, scale=0.0):
    print("attention", q.shape, k.shape, masks, flush=True)
    got = _run(L, q, k, v, do, masks, scale)
    want = ref.attention(q, k, v, ref.seen(q.shape[0], q.shape[1], k.shape[1], **masks), scale or None, do)
    for n in want:
        ref.close(got[n], want[n], n)
    again = _run(L, q, k, v, do, masks, scale)  # every sum has one order
    for n in got:
        assert np.array_equal(got[n].view(np.uint32), again[n].view(np.uint32)), n
    return got


@pytest.mark.parametrize("D", [1, 3, 16, 20, 33, 48, 64, 65, 80, 96, 100, 112, 127, 128])
def test_head_sizes(tlib, D):
    _check(tlib, *_inputs(2, 37, 70, 4, 2, D), dict(causal=True))


@pytest.mark.parametrize("D", [16, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("Lq", [16, 17, 24, 32, 33, 48, 64, 65])
def test_rows_about_a_tile(tlib, D, Lq):
    """Where one kernel takes over from another, in a workspace of the size asked for."""
    q, k, v, do = _inputs(1, Lq, 700, 2, 2, D)
    masks = dict(causal=True)
    _check(tlib, q, k, v, do, masks)
    held = []
    a = _plan(q, k, masks, held)
    need = tlib.tt_k_attention_fwd_ws(a) // 4
    ws, o, d = DevBuf(need + 64), DevBuf(q.size), [DevBuf.from_np(t) for t in (q, k, v)]
    ws.fill(7.0)
    check(tlib.tt_k_attention_fwd(a, *[x.ptr for x in d], o.ptr, None, ws.ptr), "fwd")
    ref.close(o.to_np(q.shape), ref.attention(q, k, v, ref.seen(1, Lq, 700, **masks))["o"])
    assert (ws.to_np()[need:] == 7.0).all()


@pytest.mark.parametrize("D", [8, 31, 40, 64, 80, 95, 100, 128])
@pytest.mark.parametrize("masks", [
    dict(causal=True), dict(), dict(window=50),
    dict(causal=True, window=77, k_len=[330, 0, 100], q_len=[300, 7, 33], q_start=[30, 0, 67]),
    dict(causal=True, q_start=[2147483647, -2147483648, -7]), dict(window=3, q_start=[2147483647, -200, 300])])
def test_many_rows(tlib, D, masks):
    """From 1024 packed rows on the tiles are split into parts beforehand."""
    _check(tlib, *_inputs(3, 300, 330, 4, 1, D), masks)
    if D == 64:
        _check(tlib, *_inputs(1, 1025, 257, 2, 2, D), {n: m for n, m in masks.items() if not isinstance(m, list)})
        _check(tlib, *_inputs(2, 1024, 256, 1, 1, D), {n: m for n, m in masks.items() if not isinstance(m, list)})


@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 2), (2, 1), (1, 15), (1, 17), (1, 64), (1, 65), (1, 1000), (3, 3),
                                   (15, 16), (16, 16), (17, 31), (32, 32), (33, 33), (63, 64), (64, 65), (65, 64),
                                   (100, 300), (129, 127), (257, 257), (40, 3000)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(tlib, Lq, Lk, causal):
    _check(tlib, *_inputs(1, Lq, Lk, 2, 2, 32), dict(causal=causal))


@pytest.mark.parametrize("Hq,Hkv,Lq", [(1, 1, 50), (6, 2, 50), (5, 1, 13), (8, 1, 1), (8, 2, 2), (16, 1, 1),
                                       (17, 1, 1), (40, 1, 1), (3, 3, 129), (12, 4, 33)])
def test_shared_heads(tlib, Hq, Hkv, Lq):
    _check(tlib, *_inputs(2, Lq, 90, Hq, Hkv, 48), dict(causal=True))
    _check(tlib, *_inputs(1, Lq, 77, Hq, Hkv, 64), dict())


@pytest.mark.parametrize("masks", [
    dict(k_len=[0, 1, 33, 100]),
    dict(k_len=[5, 64, 65, 99], causal=True),
    dict(k_len=[0, 1, 33, 100], q_len=[0, 1, 33, 70], q_start=[0, 0, 0, 0], causal=True),
    dict(q_start=[-3, 0, 40, 300], causal=True),           # rows before the first key, and behind the last
    dict(q_start=[-80, 0, 40, 300], causal=True, window=7),
    dict(window=1, causal=True), dict(window=40, causal=True), dict(window=1), dict(window=9),
    dict(window=1 << 40), dict(window=64, k_len=[3, 50, 64, 100], q_start=[0, 5, 60, -70]),
    dict(k_len=[-5, 1000, 2147483647, -2147483648]),        # clamped
    dict(q_len=[-5, 1000, 2147483647, -2147483648], causal=True),
    dict(q_start=[2147483647, -2147483648, 0, 1], causal=True),
    dict(q_start=[2147483647, -2147483648, 0, 1], window=3),
    dict(q_len=[7, 70, 64, 65]), dict(q_len=[0, 0, 0, 0]),
])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (6, 2)])
def test_masks(tlib, masks, Hq, Hkv):
    t = _inputs(4, 70, 100, Hq, Hkv, 32)
    if "k_len" in masks or "q_len" in masks:
        clamped = dict(masks)
        for n, top in (("k_len", 100), ("q_len", 70)):
            if n in masks:
                clamped[n] = np.clip(np.asarray(masks[n], np.int64), 0, top)
        got = _run(tlib, *t, masks)
        want = ref.attention(*t[:3], ref.seen(4, 70, 100, **clamped), None, t[3])
        for n in want:
            ref.close(got[n], want[n], n)
    else:
        _check(tlib, *t, masks)


@pytest.mark.parametrize("Lq,Lk,Hq", [(1, 300, 4), (3, 300, 4), (70, 100, 2), (130, 130, 2), (300, 330, 8)])
def test_padding_is_not_read(tlib, Lq, Lk, Hq):
    """NaN behind k_len and q_len reaches nothing."""
    q, k, v, do = _inputs(3, Lq, Lk, Hq, 2, 64)
    masks = dict(k_len=[Lk // 3, Lk, 1], q_len=[Lq, max(1, Lq // 2), Lq], causal=True,
                 q_start=[max(0, Lk // 3 - Lq), Lk - Lq, 0])
    clean = _run(tlib, q, k, v, do, masks)
    for b in range(3):
        for t, n in ((k, masks["k_len"][b]), (v, masks["k_len"][b]), (q, masks["q_len"][b]), (do, masks["q_len"][b])):
            t[b, n:] = np.nan
    dirty = _run(tlib, q, k, v, do, masks)
    for n in clean:
        assert np.array_equal(clean[n], dirty[n]), n
    assert not dirty["dk"][0, Lk // 3:].any() and not dirty["o"][1, masks["q_len"][1]:].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("Lq,Lk,Hq,Hkv", [(70, 70, 2, 2), (4, 90, 4, 2), (200, 300, 3, 1), (300, 300, 4, 1),
                                           (40, 2000, 2, 1), (1100, 600, 1, 1), (24, 90, 1, 1)])
def test_what_a_mask_hides_stays_hidden(tlib, bad, Lq, Lk, Hq, Hkv):
    """A causal mask over infinities and NaN in one key's and one query's rows:
    what does not see them stays within its bounds, results and gradients."""
    masks = dict(causal=True)

    def part(want, name, *at):
        return want[name][0][at], want[name][1][at]

    q, k, v, do = _inputs(1, Lq, Lk, Hq, Hkv, 40)
    want = ref.attention(q, k, v, ref.seen(1, Lq, Lk, **masks), None, do)
    j = Lk - 2                       # seen by the last two queries
    v[0, j, :, 3] = bad
    k[0, j, :, 5] = bad
    got = _run(tlib, q, k, v, do, masks)
    see = np.arange(Lq) + Lk - Lq >= j
    for n in ("o", "dq"):
        ref.close(got[n][0, ~see], part(want, n, 0, ~see), n)
    ref.close(got["lse"][0][:, ~see], tuple(x[0][:, ~see] for x in want["lse"]), "lse")
    assert np.isnan(got["o"][0, see]).any(axis=(1, 2)).all()
    q, k, v, do = _inputs(1, Lq, Lk, Hq, Hkv, 40)
    i = 1                            # sees the keys up to i + Lk - Lq only
    do[0, i, :, 3] = bad
    q[0, i, :, 5] = bad
    got = _run(tlib, q, k, v, do, masks)
    blind = np.arange(Lk) > i + Lk - Lq
    for n in ("dk", "dv"):
        ref.close(got[n][0, blind], part(want, n, 0, blind), n)
    rest = np.arange(Lq) != i
    for n in ("o", "dq"):
        ref.close(got[n][0, rest], part(want, n, 0, rest), n)


def test_large_scores(tlib):
    """Scores of thousands: the running maximum carries them; all weight on one
    key, or (equal rows) on all."""
    q, k, v, do = _inputs(1, 40, 200, 2, 2, 64)
    _check(tlib, q * 40, k * 40, v, do, dict(causal=True))
    _check(tlib, q, np.broadcast_to(k[:, :1], k.shape).copy(), v, do, dict())
    _check(tlib, q, k, v, do, dict(), scale=-0.3)
    _check(tlib, q * 0, k, v, do, dict(causal=True))


def _layout(x, kind, rng):
    """x (B, L, H, D) in a buffer of another layout: the buffer, where x starts
    in it, and its strides."""
    B, Ln, H, D = x.shape
    if kind == "heads":       # (B, H, L, D)
        return np.ascontiguousarray(x.transpose(0, 2, 1, 3)), 0, Strides(H * Ln * D, D, Ln * D)
    pad = 12 if kind == "wide" else 7
    first = 4 if kind == "wide" else 3
    buf = rng.standard_normal((B, Ln + 1, H * D + pad)).astype(np.float32)
    buf[:, :Ln, first:first + H * D] = x.reshape(B, Ln, H * D)
    return buf, first, Strides((Ln + 1) * (H * D + pad), H * D + pad, D)


def _unlayout(buf, kind, first, shape):
    B, Ln, H, D = shape
    if kind == "heads":
        return buf.reshape(B, H, Ln, D).transpose(0, 2, 1, 3)
    return buf.reshape(B, Ln + 1, -1)[:, :Ln, first:first + H * D].reshape(shape)


@pytest.mark.parametrize("kind", ["heads", "wide", "odd"])
@pytest.mark.parametrize("Lq,Hq", [(1, 4), (50, 4), (300, 2), (300, 8)])
def test_layouts(tlib, kind, Lq, Hq):
    """Head-major, and rows of a wider buffer (16-byte aligned or not): the same
    results; what lies between rows stays."""
    rng = np.random.default_rng(Lq)
    q, k, v, do = _inputs(2, Lq, 310, Hq, 2, 64)
    masks = dict(causal=True)
    want = ref.attention(q, k, v, ref.seen(2, Lq, 310, causal=True), None, do)
    L = tlib
    parts = [_layout(x, kind, rng) for x in (q, k, v, do)]
    dev = [DevBuf.from_np(p[0]) for p in parts]
    at = [d.ptr + 4 * p[1] for d, p in zip(dev, parts)]
    held = []
    a = _plan(q, k, masks, held, q=parts[0][2], k=parts[1][2], v=parts[2][2], o=parts[3][2])
    outs = [DevBuf(p[0].size) for p in (parts[3], parts[0], parts[1], parts[2])]
    for o in outs:
        o.fill(9.0)
    lse = DevBuf(2 * Hq * Lq)
    po = [o.ptr + 4 * p[1] for o, p in zip(outs, (parts[3], parts[0], parts[1], parts[2]))]
    check(L.tt_k_attention_fwd(a, *at[:3], po[0], lse.ptr, None), "fwd")
    check(L.tt_k_attention_bwd(a, *at[:3], po[0], at[3], lse.ptr, *po[1:], None), "bwd")
    for n, o, p, x in zip(("o", "dq", "dk", "dv"), outs, (parts[3], parts[0], parts[1], parts[2]), (q, q, k, v)):
        got = o.to_np()
        ref.close(_unlayout(got, kind, p[1], x.shape), want[n], n)
        assert (got == 9.0).sum() >= got.size - x.size, n
    # each gradient alone
    for keep in ((1, 0, 0), (0, 1, 1)):
        alone = [DevBuf(p[0].size) for p in parts[:3]]
        check(L.tt_k_attention_bwd(a, *at[:3], po[0], at[3], lse.ptr,
                                   *[d.ptr + 4 * p[1] if on else None for d, p, on in zip(alone, parts, keep)], None),
              "bwd")
        for d, p, on, n, x in zip(alone, parts, keep, ("dq", "dk", "dv"), (q, k, v)):
            if on:
                ref.close(_unlayout(d.to_np(), kind, p[1], x.shape), want[n], n)


@pytest.mark.parametrize("Lq,Lk,Hq,Hkv", [(1, 5000, 4, 2), (2, 1300, 4, 1), (1, 130, 16, 16), (24, 3000, 1, 1), (20, 5000, 4, 2),
                                          (130, 2000, 1, 1), (600, 2000, 2, 1)])
def test_keys_split_over_workgroups(tlib, Lq, Lk, Hq, Hkv):
    """Long caches with ragged lengths, some within the first part; the parts
    join to the same bits with a workspace of the caller's, and nothing is
    allocated then."""
    q, k, v, do = _inputs(3, Lq, Lk, Hq, Hkv, 64)
    masks = dict(k_len=[Lk, 40, Lk // 2 + 1], q_start=[Lk - Lq, 40 - Lq, Lk // 2 + 1 - Lq], causal=True)
    got = _check(tlib, q, k, v, do, masks)
    held = []
    a = _plan(q, k, masks, held)
    need = tlib.tt_k_attention_fwd_ws(a)
    assert need > 0
    ws, o = DevBuf(need // 4), DevBuf(q.size)
    d = [DevBuf.from_np(t) for t in (q, k, v)]
    ws.fill(np.nan)
    assert tlib.tth_fail_alloc_after(0) == 0
    try:
        rc = tlib.tt_k_attention_fwd(a, d[0].ptr, d[1].ptr, d[2].ptr, o.ptr, None, ws.ptr)
        none = tlib.tt_k_attention_fwd(a, d[0].ptr, d[1].ptr, d[2].ptr, o.ptr, None, None)
    finally:
        tlib.tth_fail_alloc_after(-1)
    assert rc == 0 and none == -2
    assert np.array_equal(o.to_np(q.shape), got["o"])


@pytest.mark.parametrize("B,Lq,Lk,H", [(100, 40, 50, 1), (64, 70, 33, 3), (2, 33, 17000, 1), (2, 17000, 40, 1),
                                       (3, 1100, 1500, 2)])
def test_ragged_batches_over_many_workgroups(tlib, B, Lq, Lk, H):
    """Batches of up to 64 sequences, and up to 256 tiles of a sequence, are taken
    tile by tile from the fullest on; others in their own order.  Every row and
    key is written once, whatever the lengths."""
    t = _inputs(B, Lq, Lk, H, H, 16)
    rng = np.random.default_rng(B)
    q_len, k_len = rng.integers(0, Lq + 1, B), rng.integers(0, Lk + 1, B)
    k_len[-1], q_len[0] = Lk, Lq
    _check(tlib, *t, dict(k_len=k_len, q_len=q_len, q_start=np.zeros(B, np.int64), causal=Lq > Lk))


@pytest.mark.parametrize("Lq,Lk", [(40, 60), (700, 300)])
def test_backward_in_a_workspace_of_the_caller(tlib, Lq, Lk):
    """Whatever it holds before: the same bits, with nothing allocated."""
    q, k, v, do = _inputs(2, Lq, Lk, 4, 2, 96)
    masks = dict(causal=True, k_len=[Lk, Lk // 3], q_start=[0, Lk // 3 - Lq])
    want = _run(tlib, q, k, v, do, masks)
    held = []
    a = _plan(q, k, masks, held)
    need = tlib.tt_k_attention_bwd_ws(a)
    ws, d = DevBuf(need // 4 + 8), [DevBuf.from_np(t) for t in (q, k, v, want["o"], do, want["lse"])]
    out = [DevBuf(t.size) for t in (q, k, v)]
    for fill in (np.nan, 1e30):
        ws.fill(fill)
        assert tlib.tth_fail_alloc_after(0) == 0
        try:
            rc = tlib.tt_k_attention_bwd(a, *[x.ptr for x in d], *[x.ptr for x in out], ws.ptr)
            none = tlib.tt_k_attention_bwd(a, *[x.ptr for x in d], *[x.ptr for x in out], None)
        finally:
            tlib.tth_fail_alloc_after(-1)
        assert rc == 0 and none == -2
        for n, x, t in zip(("dq", "dk", "dv"), out, (q, k, v)):
            assert np.array_equal(x.to_np(t.shape), want[n]), n
        assert (ws.to_np()[need // 4:] == np.float32(fill)).all() or np.isnan(fill)


def test_offsets_past_32_bits(tlib):
    """Rows 2^23 floats apart: the last ones lie past 2^31 elements."""
    n, apart = 300, 1 << 23
    q, k, v, _ = _inputs(1, 1, n, 2, 1, 64)
    big = DevBuf((n - 1) * apart + 128)
    for j in range(n):
        for t, off in ((k, 0), (v, 64)):
            row = np.ascontiguousarray(t[0, j, 0])
            check(tlib.tth_h2d(big.ptr + 4 * (j * apart + off), row.ctypes.data, row.nbytes), "h2d")
    s = Strides(0, apart, 0)
    for Lq in (1, 30, 1100):
        q = _inputs(1, Lq, n, 2, 1, 64)[0]
        held, o, d = [], DevBuf(q.size), DevBuf.from_np(q)
        a = _plan(q, k, {}, held, k=s, v=s)
        check(tlib.tt_k_attention_fwd(a, d.ptr, big.ptr, big.ptr + 256, o.ptr, None, None), "fwd")
        ref.close(o.to_np(q.shape), ref.attention(q, k, v, ref.seen(1, Lq, n))["o"])
    big.free()
    tlib.tth_release_cache()


@pytest.mark.parametrize("rank", [2, 4])
def test_attention_node(tlib, rank):
    from tinytorch_amd.torch_py import Node
    q, k, v, do = _inputs(2, 19, 23, 4, 2, 32)
    masks = dict(causal=True, window=11, k_len=[23, 9], q_len=[19, 12], q_start=[4, 0])
    want = ref.attention(q, k, v, ref.seen(2, 19, 23, **masks), 0.2, do)

    def shaped(x):
        return x if rank == 4 else x.reshape(x.shape[0] * x.shape[1], -1)

    Q, K, V = (Node.leaf(shaped(x)) for x in (q, k, v))
    y = Q.attention(K, V, 2, 4, 2, 32, scale=0.2, **masks)
    ref.close(y.value().reshape(q.shape), want["o"])
    y.backward(shaped(do))
    for n, name, x in ((Q, "dq", q), (K, "dk", k), (V, "dv", v)):
        ref.close(n.grad().reshape(x.shape), want[name], name)
    # gradients of some inputs only
    for needs in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        n3 = [Node.leaf(shaped(x), bool(on)) for x, on in zip((q, k, v), needs)]
        n3[0].attention(n3[1], n3[2], 2, 4, 2, 32, scale=0.2, **masks).backward(shaped(do))
        for n, on, name, x in zip(n3, needs, ("dq", "dk", "dv"), (q, k, v)):
            if on:
                ref.close(n.grad().reshape(x.shape), want[name], name)
            else:
                assert n.grad() is None
    for bad in (lambda: Q.attention(K, V, 3, 4, 2, 32), lambda: Q.attention(K, V, 2, 4, 3, 32),
                lambda: Q.attention(K, Q, 2, 4, 2, 32), lambda: Q.attention(K, V, 2, 4, 2, 32, window=-1),
                lambda: Q.attention(K, V, 2, 4, 2, 32, k_len=[1]), lambda: Q.attention(K, V, 0, 4, 2, 32)):
        with pytest.raises(ValueError):
            bad()


def test_one_node_as_query_key_and_value(tlib):
    from tinytorch_amd.torch_py import Node
    x, _, _, do = _inputs(1, 21, 21, 2, 2, 16)
    want = ref.attention(x, x, x, ref.seen(1, 21, 21, causal=True), None, do)
    X = Node.leaf(x)
    y = X.attention(X, X, 1, 2, 2, 16, causal=True)
    y.backward(do)
    val = sum(want[n][0] for n in ("dq", "dk", "dv"))
    tol = sum(want[n][1] + 2 * ref.U * np.abs(want[n][0]) for n in ("dq", "dk", "dv"))
    ref.close(X.grad(), (val, tol))


def test_gradients_by_differences(tlib):
    q, k, v, do = _inputs(1, 9, 12, 4, 2, 8)
    masks = dict(causal=True, k_len=[11])
    got = _run(tlib, q, k, v, do, masks)
    m = ref.seen(1, 9, 12, **masks)
    rng = np.random.default_rng(0)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rng.standard_normal((q, k, v)[i].shape)
        f = []
        for h in (1e-5, -1e-5):
            p = [t.astype(np.float64) for t in (q, k, v)]
            p[i] = p[i] + h * d
            f.append((ref.attention(*p, m)["o"][0] * do).sum())
        assert abs((f[0] - f[1]) / 2e-5 - (got[name] * d).sum()) <= 1e-5 * np.abs(got[name] * d).sum()


@pytest.mark.parametrize("Lq,Lk,Hq,Hkv", [(1, 300, 4, 2), (1, 5000, 4, 2), (20, 3000, 1, 1), (70, 70, 2, 2),
                                          (130, 2000, 1, 1), (300, 330, 4, 1), (1100, 900, 1, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_nan_that_has_no_weight_is_seen(tlib, Lq, Lk, Hq, Hkv, causal):
    """0 * NaN is NaN, also where a key's weight is 0 next to the others' and it
    lies in a part of keys that have none."""
    q, k, v, do = _inputs(1, Lq, Lk, Hq, Hkv, 64)
    q, k = np.abs(q) + 1, np.abs(k) + 1
    see = ref.seen(1, Lq, Lk, causal=causal)
    for none, j in ((slice(0, Lk // 2), 0), (slice(Lk // 2, Lk), Lk // 2 + 1)):
        k2, v2 = k.copy(), v.copy()
        k2[0, none] = -60   # hundreds below the others: exp is 0 in 32 bits
        want = ref.attention(q, k2, v, see, None, do)["o"]
        v2[0, j, :, 3] = np.nan
        got = _run(tlib, q, k2, v2, do, dict(causal=causal))["o"]
        meet = see[0, :, j]
        assert np.isnan(got[0, meet, :, 3]).all()
        rest = np.ones(got.shape, bool)
        rest[0, meet, :, 3] = False
        ref.close(got[rest], tuple(x[rest] for x in want), "o")


@pytest.mark.parametrize("Lq,Lk,Hq,Hkv,causal", [(1, 300, 4, 2, False), (20, 700, 1, 1, True), (70, 100, 2, 2, True),
                                                 (130, 2000, 1, 1, False), (300, 330, 8, 2, True),
                                                 (1100, 900, 1, 1, True)])
@pytest.mark.parametrize("bad", [0.0, np.nan])
def test_operands_that_end_with_the_last_sequence(tlib, Lq, Lk, Hq, Hkv, causal, bad):
    """q, k, v and dout lie at the end of an allocation, their last sequence cut
    off behind its q_len and k_len; a NaN in the last key brings the slow paths."""
    q, k, v, do = _inputs(2, Lq, Lk, Hq, Hkv, 48)
    masks = dict(q_len=[Lq, Lq // 2], k_len=[Lk, Lk // 3], q_start=[Lk - Lq, Lk // 3 - Lq // 2], causal=causal)
    see = ref.seen(2, Lq, Lk, **masks)
    want = ref.attention(q, k, v, see, None, do)
    j = masks["k_len"][1] - 1
    k[1, j, :, 5] += bad
    v[1, j, :, 3] += bad
    held, at = [], []
    size = 66 << 20
    for t, n in ((q, masks["q_len"][1]), (k, j + 1), (v, j + 1), (do, masks["q_len"][1])):
        x = np.ascontiguousarray(t.reshape(-1)[:t[0].size + t[1, :n].size])
        held.append(DevBuf(size // 4))
        at.append(held[-1].ptr + size - x.nbytes)
        check(tlib.tth_h2d(at[-1], x.ctypes.data, x.nbytes), "h2d")
    a = _plan(q, k, masks, held)
    o, lse, out = DevBuf(q.size), DevBuf(2 * Hq * Lq), [DevBuf(t.size) for t in (q, k, v)]
    check(tlib.tt_k_attention_fwd(a, *at[:3], o.ptr, lse.ptr, None), "fwd")
    check(tlib.tt_k_attention_bwd(a, *at[:3], o.ptr, at[3], lse.ptr, *[x.ptr for x in out], None), "bwd")
    rest = ~see[:, :, j] if bad else np.ones((2, Lq), bool)
    rest[0] = True
    for n, x in (("o", o), ("dq", out[0])):
        ref.close(x.to_np(q.shape)[rest], tuple(w[rest] for w in want[n]), n)
    if not bad:
        ref.close(out[1].to_np(k.shape), want["dk"], "dk")
        ref.close(out[2].to_np(v.shape), want["dv"], "dv")


INFINITE = [(1, 300, 4, 2), (1, 5000, 4, 2), (16, 90, 1, 1), (32, 700, 1, 1), (33, 700, 1, 1), (70, 70, 2, 2),
            (300, 330, 4, 1), (1100, 600, 1, 1)]


def _infinite(tlib, shape, masks, which, bad):
    """Results with an infinity at column 5 (at 3 in v and dout) of one key's or
    query's first head, what to expect without it, and who sees it."""
    Lq, Lk, Hq, Hkv = shape
    q, k, v, do = _inputs(1, Lq, Lk, Hq, Hkv, 40)
    see = ref.seen(1, Lq, Lk, **masks)
    want = ref.attention(q, k, v, see, None, do)
    # the last key that some but not all queries see, or the last
    n = see[0].sum(0)
    j = int(np.flatnonzero((n > 0) & (n < Lq) if ((n > 0) & (n < Lq)).any() else n > 0)[-1])
    i = Lq // 2
    dict(q=q, k=k, v=v, do=do)[which][0, j if which in "kv" else i, 0, 5 if which in "qk" else 3] = bad
    return _run(tlib, q, k, v, do, masks), want, see[0], i, j


@pytest.mark.parametrize("bad", [np.inf, -np.inf])
@pytest.mark.parametrize("masks", [dict(), dict(causal=True)])
@pytest.mark.parametrize("shape", INFINITE)
def test_infinite_keys(tlib, shape, masks, bad):
    """One infinity in k, of either sign of the product: NaN for the queries that
    see it and what comes of them, whichever kernel takes them."""
    got, want, see, _, j = _infinite(tlib, shape, masks, "k", bad)
    G, meet = shape[2] // shape[3], see[:, j]
    assert meet.any()
    heads = np.arange(shape[2]) < G
    for n in ("o", "dq"):
        assert np.isnan(got[n][0][meet][:, heads]).all(), n
        for rows, hs in ((~meet, slice(None)), (slice(None), ~heads)):
            ref.close(got[n][0][rows][:, hs], tuple(x[0][rows][:, hs] for x in want[n]), n)
    assert np.isnan(got["lse"][0][heads][:, meet]).all()
    ref.close(got["lse"][0][heads][:, ~meet], tuple(x[0][heads][:, ~meet] for x in want["lse"]), "lse")
    touched = see[meet].any(0)
    for n in ("dk", "dv"):
        assert np.isnan(got[n][0, touched, 0]).all(), n
        ref.close(got[n][0, ~touched, 0], tuple(x[0, ~touched, 0] for x in want[n]), n)


@pytest.mark.parametrize("bad", [np.inf, -np.inf])
@pytest.mark.parametrize("masks", [dict(), dict(causal=True)])
@pytest.mark.parametrize("shape", INFINITE)
def test_infinite_values(tlib, shape, masks, bad):
    """One infinity in v: NaN in its column of the results that see it, and in
    what their rows' gradients reach; dv and lse do not depend on it."""
    got, want, see, _, j = _infinite(tlib, shape, masks, "v", bad)
    G, meet = shape[2] // shape[3], see[:, j]
    heads = np.arange(shape[2]) < G
    o = got["o"][0]
    assert np.isnan(o[meet][:, heads, 3]).all()
    rest = np.ones(o.shape, bool)
    rest[np.ix_(meet, heads, [3])] = False
    ref.close(o[rest], tuple(x[0][rest] for x in want["o"]), "o")
    ref.close(got["lse"], want["lse"], "lse")
    ref.close(got["dv"], want["dv"], "dv")
    assert np.isnan(got["dq"][0][meet][:, heads]).all()
    ref.close(got["dq"][0][~meet], tuple(x[0][~meet] for x in want["dq"]), "dq")
    assert np.isnan(got["dk"][0, see[meet].any(0), 0]).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf])
@pytest.mark.parametrize("masks", [dict(), dict(causal=True)])
@pytest.mark.parametrize("shape", INFINITE)
def test_infinite_queries_and_gradients(tlib, shape, masks, bad):
    """One infinity in q: NaN for its row and the keys that it sees; in dout: NaN
    in dq of its row, in dk of these keys and in its column of their dv."""
    for which in ("q", "do"):
        got, want, see, i, _ = _infinite(tlib, shape, masks, which, bad)
        rest, keys = np.arange(shape[0]) != i, see[i]
        for n in ("o", "dq"):
            if which == "q" or n == "dq":
                assert np.isnan(got[n][0, i, 0]).all(), (which, n)
            else:
                ref.close(got[n], want[n], n)
            ref.close(got[n][0, rest], tuple(x[0, rest] for x in want[n]), n)
        assert np.isnan(got["lse"][0, 0, i]) == (which == "q")
        assert np.isnan(got["dk"][0, keys, 0]).all(), which
        at = slice(None) if which == "q" else 3
        assert np.isnan(got["dv"][0, keys, 0][:, at]).all(), which
        for n in ("dk", "dv"):
            ref.close(got[n][0, ~keys], tuple(x[0, ~keys] for x in want[n]), n)


def test_infinite_queries_that_see_no_key(tlib):
    """No key: 0 and -inf, whatever the query holds."""
    for Lq in (1, 20, 70, 1100):
        q, k, v, do = _inputs(1, Lq, 90, 1, 1, 40)
        q[0, Lq // 2] = np.inf
        got = _run(tlib, q, k, v, do, dict(k_len=[0]))
        assert np.isneginf(got["lse"]).all()
        assert not any(got[n].any() for n in ("o", "dq", "dk", "dv")), Lq
