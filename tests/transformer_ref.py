"""The transformer operators in 64 bits, with a bound for each output of what
fp32 arithmetic may leave: every sum of n terms is off by at most n U times the
sum of their absolute values, every other operation by U times its value, and
errors of inputs pass on by the derivative's absolute value."""
import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative to the value


def layernorm(x, w, b, dy=None, eps=1e-5):
    """y, mean, rstd[, dx, dw, db], each with its bound."""
    x = x.astype(np.float64)
    n, C = x.shape
    w = np.ones(C) if w is None else w.astype(np.float64)
    b = np.zeros(C) if b is None else b.astype(np.float64)
    mean = x.mean(1, keepdims=True)
    d = x - mean
    e_mean = (C + 1) * U * np.abs(x).mean(1, keepdims=True)
    e_d = e_mean + U * np.abs(d)
    var = (d * d).mean(1, keepdims=True)
    e_var = (C + 3) * U * var + 2 * (np.abs(d) * e_d).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    e_r = rstd * (0.5 * e_var / (var + eps) + 4 * U)
    h = d * rstd
    e_h = e_d * rstd + np.abs(d) * e_r + 2 * U * np.abs(h)
    y = h * w + b
    e_y = e_h * np.abs(w) + 2 * U * (np.abs(h * w) + np.abs(b))
    out = [(y, e_y), (mean[:, 0], e_mean[:, 0]), (rstd[:, 0], e_r[:, 0])]
    if dy is None:
        return out
    dy = dy.astype(np.float64)
    g = dy * w
    e_g = U * np.abs(g)
    s, q = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    e_s = (C + 2) * U * np.abs(g).mean(1, keepdims=True)
    e_q = (C + 3) * U * np.abs(g * h).mean(1, keepdims=True) + (np.abs(g) * e_h).mean(1, keepdims=True)
    t = g - s - h * q
    e_t = e_g + e_s + np.abs(h) * e_q + e_h * np.abs(q) + 4 * U * (np.abs(g) + np.abs(s) + np.abs(h * q))
    out.append((t * rstd, e_t * rstd + np.abs(t) * e_r + U * np.abs(t * rstd)))
    out.append(((dy * h).sum(0), (np.abs(dy) * e_h).sum(0) + (n + 1) * U * np.abs(dy * h).sum(0)))
    out.append((dy.sum(0), n * U * np.abs(dy).sum(0)))
    return out


def frequencies(rot, base, scaling="plain", factor=1.0, trained=0.0, low=0.0, high=0.0):
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        r = np.clip((trained * f / (2 * np.pi) - low) / (high - low), 0, 1)
        f = (1 - r) * f / factor + r * f
    return f


def rope(x, pos, f, interleaved, transpose=False, magnitude=1.0):
    """x (rows, heads, dim); the bound counts an angle off by 4 U of a turn's
    half (its fraction rounded to fp32, sine and cosine to two steps), two
    products and a sum."""
    x = x.astype(np.float64)
    R = 2 * len(f)
    t = pos.astype(np.float64)[:, None] * f[None, :] * (-1 if transpose else 1)
    c, s = np.cos(t)[:, None] * magnitude, np.sin(t)[:, None] * magnitude
    y = x.copy()
    tol = np.zeros_like(x)
    even, odd = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., even], x[..., odd]
    y[..., even], y[..., odd] = a * c - b * s, a * s + b * c
    e = (np.abs(a) + np.abs(b)) * magnitude * (np.pi + 4 + 3) * U
    tol[..., even] = tol[..., odd] = e
    return y, tol


def seen(batch, q_rows, k_rows, causal=False, window=0, q_start=None, q_len=None, k_len=None):
    i, j = np.arange(q_rows)[None, :, None], np.arange(k_rows)[None, None, :]
    at = (np.full(batch, k_rows - q_rows) if q_start is None else np.asarray(q_start, np.int64))[:, None, None] + i
    m = np.ones((batch, q_rows, k_rows), bool)
    if k_len is not None:
        m &= j < np.asarray(k_len)[:, None, None]
    if q_len is not None:
        m &= i < np.asarray(q_len)[:, None, None]
    if causal:
        m &= j <= at
    if window:
        m &= (at - j if causal else np.abs(at - j)) < window
    return m


def attention(q, k, v, mask, scale=None, do=None):
    """q (B, Lq, Hq, D), k and v (B, Lk, Hkv, D), mask (B, Lq, Lk).  What the
    mask hides may hold anything."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    G = Hq // Hkv
    scale = 1 / np.sqrt(D) if scale is None else scale
    names = ("o", "lse") + (("dq", "dk", "dv") if do is not None else ())
    out = {n: (np.zeros(s), np.zeros(s)) for n, s in
           zip(names, (q.shape, (B, Hq, Lq), q.shape, k.shape, v.shape))}
    for b in range(B):
        rows, cols = mask[b].any(1), mask[b].any(0)
        for h in range(Hq):
            m = mask[b]
            Q = np.where(rows[:, None], q[b, :, h].astype(np.float64), 0)
            K = np.where(cols[:, None], k[b, :, h // G].astype(np.float64), 0)
            V = np.where(cols[:, None], v[b, :, h // G].astype(np.float64), 0)
            S = scale * Q @ K.T
            e_s = (D + 6) * U * abs(scale) * (np.abs(Q) @ np.abs(K).T)
            top = np.where(m, S, -np.inf).max(1, keepdims=True)
            top = np.where(np.isfinite(top), top, 0)
            P = np.where(m, np.exp(np.where(m, S - top, 0)), 0)
            n = Lk
            total = P.sum(1, keepdims=True)
            lse = np.where(total > 0, top + np.log(np.where(total > 0, total, 1)), -np.inf)
            P = P / np.where(total > 0, total, 1)
            worst = np.where(m, e_s + 2 * U * np.abs(S - top), 0)
            e_lse = worst.max(1, keepdims=True) + (n + 8) * U + 4 * U * np.abs(np.where(total > 0, lse, 0))
            e_p = worst + worst.max(1, keepdims=True) + (n + 8) * U  # relative
            o = P @ V
            e_o = (P * e_p) @ np.abs(V) + (n + 4) * U * (P @ np.abs(V))
            out["o"][0][b, :, h], out["o"][1][b, :, h] = o, e_o
            out["lse"][0][b, h], out["lse"][1][b, h] = lse[:, 0], np.where(total > 0, e_lse, 0)[:, 0]
            if do is None:
                continue
            dO = np.where(rows[:, None], do[b, :, h].astype(np.float64), 0)
            n2 = Lq * G
            dP = dO @ V.T
            e_dp = (D + 1) * U * (np.abs(dO) @ np.abs(V).T)
            dl = (dO * o).sum(1, keepdims=True)
            e_dl = (D + 4) * U * (np.abs(dO) * np.abs(o)).sum(1, keepdims=True) + (np.abs(dO) * e_o).sum(1, keepdims=True)
            e_p2 = worst + e_lse + 4 * U * np.abs(np.where(m, S, 0))
            dS = P * (dP - dl)
            e_ds = P * (e_p2 * np.abs(dP - dl) + e_dp + e_dl + 4 * U * (np.abs(dP) + np.abs(dl)))
            for name, val, tol, at in (
                    ("dq", scale * dS @ K, abs(scale) * ((e_ds + (n + 2) * U * np.abs(dS)) @ np.abs(K)), h),
                    ("dk", scale * dS.T @ Q, abs(scale) * ((e_ds + (n2 + 2) * U * np.abs(dS)).T @ np.abs(Q)), h // G),
                    ("dv", P.T @ dO, (P * (e_p2 + (n2 + 2) * U)).T @ np.abs(dO), h // G)):
                out[name][0][b, :, at] += val
                out[name][1][b, :, at] += tol
    return out


def distill(z, ids, teacher, T, scale):
    """Row losses and the gradient, with their bounds."""
    z, t = z.astype(np.float64), teacher.astype(np.float64) / T
    rows, cols = z.shape
    loss, dz = np.zeros(rows), np.zeros_like(z)
    e_loss, e_dz = np.zeros(rows), np.zeros_like(z)
    for r in range(rows):
        ok = (ids[r] >= 0) & (ids[r] < cols)
        tt = np.where(ok, t[r], -np.inf)
        if not ok.any() or tt.max() == -np.inf:
            continue
        x = np.zeros(cols) if np.all(z[r] == -np.inf) else z[r] / T
        # differences first: next to the lowest values a logarithm would be lost
        m, mt = x.max(), tt.max()
        log_z, log_t = np.log(np.exp(x - m).sum()), np.log(np.exp(tt - mt).sum())
        with np.errstate(invalid="ignore"):
            far, far_t = np.abs(np.where(np.isfinite(x), x - m, 0)), np.abs(np.where(np.isfinite(tt), tt - mt, 0))
            q, p = np.exp(x - m - log_z), np.where(ok, np.exp(tt - mt - log_t), 0)
            lq = np.where(ok, (x - m)[np.where(ok, ids[r], 0)] - log_z, 0)
            use = p > 0
            lp = np.where(use, tt - mt - log_t, 0)
            loss[r] = T * T * np.where(use, p * (lp - lq), 0).sum()
            e_q = (cols + 8) * U + 4 * U * far
            e_p = (len(p) + 8) * U + 4 * U * far_t
            e_lq = (cols + 8) * U + 6 * U * (np.abs(np.where(use, lq, 0)) + log_z)
            e_loss[r] = T * T * (p * (e_p * (np.abs(lp - lq) + 1) + e_lq + 4 * U * np.abs(lp - lq)) +
                                 len(p) * U * np.abs(p * (lp - lq)))[use].sum()
        dz[r], e_dz[r] = q, e_q * q
        np.add.at(dz[r], ids[r][ok], -p[ok])
        np.add.at(e_dz[r], ids[r][ok], p[ok] * (e_p[ok] + 4 * U))
        dz[r] *= scale * T
        e_dz[r] = abs(scale) * T * (e_dz[r] + 4 * U * np.abs(q)) + 4 * U * np.abs(dz[r])
    return (loss, e_loss), (dz, e_dz)


def close(got, want, what=""):
    val, tol = want
    fin = np.isfinite(val)
    tol = np.where(fin, tol, 0)
    assert np.array_equal(got[~fin], val[~fin]), f"{what}: values without a finite one differ"
    # what is smaller than fp32's least normal value may be 0
    off = np.abs(np.where(fin, got, 0).astype(np.float64) - np.where(fin, val, 0)) - (tol + 1e-37)
    bad = fin & ~(off <= 0)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside their bounds, first at "
                           f"{np.argwhere(bad)[0]}: {got[tuple(np.argwhere(bad)[0])]} for "
                           f"{val[tuple(np.argwhere(bad)[0])]} +- {tol[tuple(np.argwhere(bad)[0])]}")
