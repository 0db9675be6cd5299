"""RMS norm, token embeddings and Newton-Schulz steps in 64 bits, with a bound for
each output of what fp32 arithmetic may leave: a sum of n terms is off by at most
n U times the sum of their absolute values, any other operation by U times its
value, and errors of inputs pass on by the derivative's absolute value."""
import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative to the value
A, B, C = 3.4445, -4.7750, 2.0315


def rmsnorm(x, res, w, dy=None, dsum=None, eps=1e-5):
    """y, sum, rstd[, dx, dw], each with its bound."""
    x = x.astype(np.float64)
    s = x if res is None else x + res.astype(np.float64)
    n, cols = x.shape
    e_s = 0 * s if res is None else U * np.abs(s)
    w = np.ones(cols) if w is None else w.astype(np.float64)
    q = (s * s).mean(1, keepdims=True)
    e_q = (cols + 3) * U * q + 2 * (np.abs(s) * e_s).mean(1, keepdims=True)
    r = 1 / np.sqrt(q + eps)
    e_r = r * (0.5 * e_q / (q + eps) + 4 * U)
    h = s * r
    e_h = e_s * r + np.abs(s) * e_r + U * np.abs(h)
    y = h * w
    out = [(y, e_h * np.abs(w) + U * np.abs(y)), (s, e_s), (r[:, 0], e_r[:, 0])]
    if dy is None:
        return out
    dy = dy.astype(np.float64)
    g = dy * w
    p = (g * h).mean(1, keepdims=True)
    e_p = (cols + 4) * U * np.abs(g * h).mean(1, keepdims=True) + (np.abs(g) * e_h).mean(1, keepdims=True)
    t = g - h * p
    e_t = U * np.abs(g) + np.abs(h) * e_p + e_h * np.abs(p) + 3 * U * (np.abs(g) + np.abs(h * p))
    dx = t * r
    e_x = e_t * r + np.abs(t) * e_r + U * np.abs(dx)
    if dsum is not None:
        dx = dx + dsum.astype(np.float64)
        e_x = e_x + U * np.abs(dx)
    out.append((dx, e_x))
    out.append(((dy * h).sum(0), (np.abs(dy) * e_h).sum(0) + (n + 1) * U * np.abs(dy * h).sum(0)))
    return out


def embedding(w, ids, scale):
    """The rows, which are one product each: as fp32 rounds it."""
    has = (ids >= 0) & (ids < len(w))
    return np.where(has[:, None], w[np.where(has, ids, 0)] * np.float32(scale), np.float32(0))


def embedding_grad(ids, dy, vocab, scale, old=None):
    dw, total, count = np.zeros((vocab, dy.shape[1])), np.zeros((vocab, dy.shape[1])), np.zeros(vocab)
    has = (ids >= 0) & (ids < vocab)
    d = dy[has].astype(np.float64)
    np.add.at(dw, ids[has], d)
    np.add.at(total, ids[has], np.abs(d))
    np.add.at(count, ids[has], 1)
    scale = float(np.float32(scale))
    val, tol = dw * scale, (count[:, None] + 1) * U * total * abs(scale)
    if old is not None:
        val = val + old
        tol = np.where(count[:, None] > 0, tol + U * np.abs(val), 0)
    return val, tol


# A product of the fp16 parts: each operand's value is off by 2^-22 of it (two halves
# of a step, 2^-11 each) and 2^-39 (half the least step of fp16, 2^-25, over 2^14);
# the parts' last product is left out, 2^-22 of the values' again; and the 3 K terms
# are added in fp32, whose order and rounding the hardware has: 2 U each.
PART, LEAST = 2.0 ** -22, 2.0 ** -39


def _product(x, y, ex, ey):
    """x @ y and its bound, for operands that are off by ex and ey already."""
    ex, ey = ex + PART * np.abs(x) + LEAST, ey + PART * np.abs(y) + LEAST
    ax, ay = np.abs(x), np.abs(y)
    k = x.shape[1]
    return x @ y, ex @ (ay + ey) + ax @ ey + (6 * k * U + PART) * (ax @ ay)


def normed(u):
    """U / |U|_F along the shorter side, and its bound."""
    x = u.astype(np.float64)
    x = x.T if x.shape[0] > x.shape[1] else x
    norm = np.sqrt((x * x).sum())
    x = x / norm if norm > 0 else x
    return x, U * np.abs(x)


def one_step(x, ex):
    """A step from x, known to ex, value by value."""
    p, ep = _product(x, x.T, ex, ex.T)
    ep = ep + U * np.abs(p)
    pp, epp = _product(p, p.T, ep, ep.T)
    q = B * p + C * pp
    eq = abs(B) * (ep + PART * np.abs(p) + LEAST) + C * epp + 4 * U * (abs(B) * np.abs(p) + C * np.abs(pp))
    qx, eqx = _product(q, x, eq, ex)
    y = A * x + qx
    return y, A * (ex + PART * np.abs(x) + LEAST) + eqx + 4 * U * (A * np.abs(x) + np.abs(qx))


def newton_schulz(u, steps):
    """The result and a bound of its error's 2-norm.  One step's is that of its
    values; what a step leaves, the next ones multiply by 4 at most (the largest slope
    of a s + b s^3 + c s^5 over [0, 1.21]; a function of singular values that is odd
    changes in the 2-norm no faster than in one number)."""
    x, ex = normed(u)
    off = np.linalg.norm(ex)
    for _ in range(steps):
        y, local = one_step(x, 0 * x)
        off = 4.3 * off + np.linalg.norm(local)
        x = y
    return (x.T if u.shape[0] > u.shape[1] else x), off
