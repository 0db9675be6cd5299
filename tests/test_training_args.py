"""What RMS norm, token embeddings and Muon refuse: on the CPU, nothing is
launched."""
import ctypes

import pytest

import tinytorch_amd

P = 0x1000  # a pointer that no refused call reads
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def L():
    return tinytorch_amd.lib()


@pytest.mark.parametrize("args", [(None, P, 4, 8, 1e-5), (P, None, 4, 8, 1e-5), (P, P, 0, 8, 1e-5),
                                  (P, P, 4, 0, 1e-5), (P, P, -1, 8, 1e-5), (P, P, 4, 8, -1e-5), (P, P, 4, 8, NAN),
                                  (P, P, 4, 8, INF), (P, P, 1 << 40, 1 << 20, 1e-5), (P, P, 4, 1 << 31, 1e-5)])
def test_rmsnorm_refuses(L, args):
    x, y, rows, cols, eps = args
    assert L.tt_k_rmsnorm_fwd(x, None, None, y, None, None, rows, cols, eps) == -1


def test_rmsnorm_backward_refuses(L):
    for i in range(3):
        args = [P] * 3  # s, dy, rstd
        args[i] = None
        assert L.tt_k_rmsnorm_bwd(args[0], P, args[1], P, args[2], P, P, 4, 8, None) == -1
    for rows, cols in ((0, 8), (8, 0), (1 << 40, 1 << 20)):
        assert L.tt_k_rmsnorm_bwd(P, P, P, P, P, P, P, rows, cols, None) == -1
        assert L.tt_k_rmsnorm_bwd_ws(rows, cols) == 0
    assert L.tt_k_rmsnorm_bwd(P, P, P, P, P, None, None, 4, 8, None) == 0  # nothing asked for


SIZES = [(0, 5, 4), (3, 0, 4), (3, 5, 0), (-1, 5, 4), ((1 << 28) + 1, 5, 4), (3, (1 << 30) + 1, 4),
         (3, 5, (1 << 22) + 1)]


@pytest.mark.parametrize("sizes", SIZES)
def test_embedding_refuses_sizes(L, sizes):
    assert L.tt_k_embedding_fwd(P, P, P, *sizes, 1.0) == -1
    assert L.tt_k_embedding_bwd(P, P, P, *sizes, 1.0, 0, P) == -1
    assert L.tt_k_embedding_bwd_ws(*sizes) == 0


def test_embedding_refuses_missing_operands(L):
    for i in range(3):
        args = [P] * 3
        args[i] = None
        assert L.tt_k_embedding_fwd(*args, 3, 5, 4, 1.0) == -1
        assert L.tt_k_embedding_bwd(*args, 3, 5, 4, 1.0, 0, P) == -1


@pytest.mark.parametrize("count,rows,cols,steps", [(0, 4, 4, 5), (-1, 4, 4, 5), (1, 0, 4, 5), (1, 4, 0, 5),
                                                   (1, (1 << 20) + 1, 4, 5), (1, 4, (1 << 20) + 1, 5),
                                                   (1, 1 << 17, 1 << 17, 5), (1, 4, 4, 0), (1, 4, 4, 65),
                                                   (1 << 39, 4, 4, 5)])
def test_newton_schulz_refuses(L, count, rows, cols, steps):
    assert L.tt_k_newton_schulz(P, P, count, rows, cols, steps, P) == -1
    if 1 <= steps <= 64 and count < 1 << 39:
        assert L.tt_k_newton_schulz_ws(count, rows, cols) == 0


def _muon(L, rows, cols, count=None, w=None, g=None, v=None, lr=0.1, mu=0.9, decay=0.0):
    n = len(rows)

    def p(x):
        return (ctypes.c_void_p * n)(*(x if x is not None else [P * (i + 1) for i in range(n)]))

    r, c = (ctypes.c_long * n)(*rows), (ctypes.c_long * n)(*cols)
    return L.tt_k_muon_multi(p(w), p(g), p(v), r, c, n if count is None else count, lr, mu, 1, decay, P)


@pytest.mark.parametrize("kw", [dict(rows=[4, 0], cols=[4, 4]), dict(rows=[4, 4], cols=[4, (1 << 20) + 1]),
                                dict(rows=[4], cols=[4], w=[None]), dict(rows=[4], cols=[4], g=[None]),
                                dict(rows=[4], cols=[4], v=[None]), dict(rows=[4], cols=[4], count=-1),
                                dict(rows=[4] * 17, cols=[4] * 17), dict(rows=[4], cols=[4], lr=NAN),
                                dict(rows=[4], cols=[4], mu=INF), dict(rows=[4], cols=[4], decay=NAN),
                                dict(rows=[4, 4], cols=[4, 4], w=[P, P]), dict(rows=[4, 4], cols=[4, 4], v=[P, P])])
def test_muon_refuses(L, kw):
    assert _muon(L, **kw) == -1


def test_muon_without_matrices(L):
    assert L.tt_k_muon_multi((ctypes.c_void_p * 1)(P), (ctypes.c_void_p * 1)(P), (ctypes.c_void_p * 1)(P),
                             (ctypes.c_long * 1)(4), (ctypes.c_long * 1)(4), 0, 0.1, 0.9, 1, 0.0, None) == 0
    assert L.tt_k_muon_multi(None, None, None, None, None, 1, 0.1, 0.9, 1, 0.0, None) == -1
    assert L.tt_k_muon_multi_ws(None, None, 1) == 0


def test_workspace_sizes(L):
    """About 14 bytes a value, 20 of a square matrix's, for 64 matrices of a shape at
    most, and up to 128 MiB; nothing for small matrices."""
    more = 128 << 20
    for m, n, least, most in ((1024, 4096, 12, 14.1), (512, 512, 20, 20.2), (300, 400, 16, 20)):
        one = L.tt_k_newton_schulz_ws(1, m, n)
        assert least * m * n <= one <= most * m * n + more
        many = L.tt_k_newton_schulz_ws(64, m, n)
        assert 64 * least * m * n <= many <= 64 * most * m * n + more
        assert many == L.tt_k_newton_schulz_ws(1000, m, n) == L.tt_k_newton_schulz_ws(64, n, m)
    assert L.tt_k_newton_schulz_ws(1000, 128, 128) == 0 == L.tt_k_newton_schulz_ws(1, 10, 785)
    r, c = (ctypes.c_long * 2)(1024, 512), (ctypes.c_long * 2)(4096, 512)
    both = L.tt_k_muon_multi_ws(r, c, 2)
    assert 12 * 1024 * 4096 + 20 * 512 * 512 <= both <= 14.1 * 1024 * 4096 + 20.2 * 512 * 512 + more
    # 16 bytes a token, and two parts of 4 bytes a column for every 8 tokens or more
    for rows in (513, 8192, 100000):
        assert 16 * rows <= L.tt_k_embedding_bwd_ws(rows, 32000, 1024) <= 16 * (rows + 3) + 8 * 1024 * ((rows + 7) // 8)
    assert L.tt_k_embedding_bwd_ws(512, 32000, 1024) == 0


@pytest.mark.parametrize("args", [(NAN, 0.9, 1, 0.0), (0.1, INF, 1, 0.0), (0.1, 0.9, 1, NAN)])
def test_optim_muon_refuses(L, args):
    assert not L.ag_optim_muon(*args)


def test_nodes_refuse_missing_operands(L):
    assert not L.ag_rmsnorm(None, None, None, 1e-5, None)
    assert not L.ag_embedding(None, P, 3, 1.0)


def _images(m, n):
    """What a matrix may take in the workspace, of sides rounded up to 32."""
    m, n = (32 * ((s + 31) // 32) for s in (min(m, n), max(m, n)))
    return (12 * m * n + 8 * m * m) * 1.002 + (16 << 10)


FLAT = [(1, 1 << 20), (1 << 20, 1), (4, 4096), (9, 5000), (3, 100000), (33, 2000), (257, 300), (1000, 31), (1, 40000)]


@pytest.mark.parametrize("m,n", FLAT)
def test_workspace_of_flat_matrices(L, m, n):
    more, groups = 128 << 20, 4 << 30
    for count in (1, 2, 20, 64, 1000):
        ws = L.tt_k_newton_schulz_ws(count, m, n)
        assert ws <= max(_images(m, n), min(groups, min(count, 64) * _images(m, n))) + more
        assert ws == L.tt_k_newton_schulz_ws(count, n, m)
    r, c = (ctypes.c_long * 2)(m, 300), (ctypes.c_long * 2)(n, 400)
    assert L.tt_k_muon_multi_ws(r, c, 2) <= _images(m, n) + _images(300, 400) + more


@pytest.mark.parametrize("rows,cols", [(513, 1), (514, 3), (520, 1), (8191, 1), (66000, 1), (70001, 5), (100001, 300),
                                       (8193, 1 << 20)])
def test_workspace_of_the_tables_gradient(L, rows, cols):
    full = (rows + 7) // 8 * 8
    assert 16 * rows <= L.tt_k_embedding_bwd_ws(rows, 1000, cols) <= 16 * full + full * cols


@pytest.mark.parametrize("m,n", [(1, 1 << 20), (32, 1 << 20), (4, 4096), (3, 1025), (16, 70001)])
def test_workspace_of_few_rows(L, m, n):
    for count in (1, 5, 64, 1000):
        assert 0 < L.tt_k_newton_schulz_ws(count, m, n) <= min(count, 64) * 600000
        assert L.tt_k_newton_schulz_ws(count, m, min(n, 1024)) == 0
    many = (ctypes.c_long * 16)(*[m] * 16), (ctypes.c_long * 16)(*[n] * 16)
    assert L.tt_k_muon_multi_ws(*many, 16) <= 16 * 600000
