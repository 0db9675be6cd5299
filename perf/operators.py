"""What a transformer's operators are timed on: layer norm, rotary positions,
attention and distillation from a teacher's top logits, through the
device-level entry points of tt_hip.h, over the sizes they are used with.

Kinds of case:

  norm       a layer norm over the last axis; `train`: forward, then the
             gradients of input, weight and bias.
  rope       rotary positions on the first `heads` heads of the rows of a
             buffer that holds `more` heads behind them; `train`: the rotation,
             then its gradient.
  attention  q, k, v laid out sequence by sequence, row by row, head by head;
             `train`: forward, then the gradients of q, k and v.
  distill    the loss and the gradient of a student's logits, or with `train`
             false the losses alone.

Everything is fp32, the one type the framework computes in.
"""
import ctypes
import math

import numpy as np
import torch

own = False  # False: the operators in elementary torch operations


# ---------------------------------------------------------------- the cases

def _norm(name, rows, cols, train):
    return dict(name=name, kind="norm", rows=rows, cols=cols, train=train)


def _rope(name, batch, seq, heads, more, dim, rot, interleaved, scaling, far, train):
    return dict(name=name, kind="rope", batch=batch, seq=seq, heads=heads, more=more, dim=dim, rot=rot,
                interleaved=interleaved, scaling=scaling, far=far, train=train)


def _attention(name, batch, q_rows, k_rows, q_heads, kv_heads, dim, causal, window, shortest, train):
    return dict(name=name, kind="attention", batch=batch, q_rows=q_rows, k_rows=k_rows, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, causal=causal, window=window, shortest=shortest, train=train)


def _distill(name, rows, cols, top, temperature, train):
    return dict(name=name, kind="distill", rows=rows, cols=cols, top=top, temperature=temperature,
                train=train)


def listed():
    return [
        # one token's activations on the way through a trained model: latency
        _norm("norm_token", 1, 1024, False),
        # the activations of a training batch of 8 x 1024 tokens
        _norm("norm_train", 8192, 1024, True),
        # odd rows and columns: no row but the first is aligned
        _norm("norm_odd", 4099, 1003, True),
        # the next token of eight long conversations: q and k heads of a joint
        # projection, positions past the trained length
        _rope("rope_token", 8, 1, 20, 4, 128, 128, False, "parts", 131072, False),
        # a training batch, interleaved pairs on half of each head
        _rope("rope_train", 4, 2048, 32, 16, 64, 32, True, "none", 0, True),
        # the next token of one conversation in a cache of 2048: latency
        _attention("attention_token", 1, 1, 2048, 8, 8, 64, True, 0, 1000, False),
        # the next token of 32 conversations of all lengths, heads that share
        # keys: the cache is read once
        _attention("attention_tokens_32", 32, 1, 8192, 32, 8, 128, True, 0, 100, False),
        # a thousand new tokens behind a cached prompt
        _attention("attention_prompt", 1, 1000, 3500, 16, 4, 80, True, 0, 3500, False),
        # a padded training batch
        _attention("attention_train", 8, 1024, 1024, 8, 8, 64, True, 0, 600, True),
        # long sequences, heads that share keys
        _attention("attention_train_long", 2, 4096, 4096, 16, 4, 128, True, 0, 4096, True),
        # a small vocabulary of odd size, one text
        _distill("distill_small", 128, 1003, 8, 1.0, True),
        # a training batch over a large vocabulary
        _distill("distill_train", 4096, 32000, 64, 2.0, True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm; odd ones too."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# no drawn case costs more than the largest listed ones: bytes, products, and
# the query-key pairs that the plain form holds in memory
MOST_BYTES, MOST_FLOPS, MOST_PAIRS = 1.06e9, 4.9e11, 5.4e8


def draw(rng):
    while True:
        kind = rng.choice(["norm", "norm", "rope", "attention", "attention", "attention", "distill",
                           "distill"])
        if kind == "norm":
            c = _norm("", _log(rng, 1, 16384), _log(rng, 16, 16384), rng.random() < 0.7)
        elif kind == "rope":
            train = rng.random() < 0.5
            dim = rng.choice([32, 64, 80, 128, 2 * rng.randint(8, 64)])
            rot = rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)])
            c = _rope("", _log(rng, 1, 32), _log(rng, 16, 4096) if train else 1, _log(rng, 1, 64),
                      rng.randint(0, 8), dim, rot, rng.random() < 0.5,
                      rng.choice(["none", "linear", "ntk", "parts"]),
                      0 if train else _log(rng, 100, 200000), train)
        elif kind == "attention":
            what = rng.choice(["token", "prompt", "train", "train"])
            group, kv = rng.choice([1, 1, 2, 4, 8]), _log(rng, 1, 16)
            dim = rng.choice([32, 64, 64, 80, 128, rng.randint(16, 128)])
            if what == "token":
                k_rows = _log(rng, 16, 16384)
                c = _attention("", _log(rng, 1, 64), 1, k_rows, group * kv, kv, dim, True, 0,
                               rng.randint(1, k_rows), False)
            elif what == "prompt":
                q_rows = _log(rng, 2, 4096)
                k_rows = q_rows + rng.choice([0, _log(rng, 1, 8192)])
                c = _attention("", _log(rng, 1, 8), q_rows, k_rows, group * kv, kv, dim,
                               rng.random() < 0.8, 0, k_rows, False)
            else:
                rows = _log(rng, 16, 4096)
                c = _attention("", _log(rng, 1, 16), rows, rows, group * kv, kv, dim,
                               rng.random() < 0.8, rng.choice([0, 0, 0, _log(rng, 8, 1024)]),
                               rng.randint(1, rows), True)
        else:
            cols = _log(rng, 100, 131072)
            c = _distill("", _log(rng, 1, 4096), cols, _log(rng, 1, min(cols, 128)),
                         rng.choice([1.0, 2.0, 4.0]), rng.random() < 0.8)
        w = work(c)
        if w["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS:
            continue
        if kind == "attention" and c["batch"] * c["q_heads"] * c["q_rows"] * c["k_rows"] > MOST_PAIRS:
            continue
        del c["name"]
        return c


# ---------------------------------------------------------------- inputs

EPS = 1e-5
BASE = 10000.0
# how positions past the trained length are scaled, in the drawn and listed cases
SCALING = {"none": (0, 1.0, 0.0, 0.0, 0.0), "linear": (1, 4.0, 0.0, 0.0, 0.0),
           "ntk": (2, 4.0, 0.0, 0.0, 0.0), "parts": (3, 8.0, 8192.0, 1.0, 32.0)}


class _State:
    pass


def _lengths(case, seed):
    """What the sequences of a batch hold: even from `shortest` to the whole,
    dealt to the sequences by the seed."""
    n = np.linspace(case["k_rows"], case["shortest"], case["batch"]).astype(np.int32)
    return np.random.default_rng([seed, 1]).permutation(n)


def prepare(case, seed):
    s = _State()
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind == "norm":
        rows, cols = case["rows"], case["cols"]
        # activations with an offset of their own in each column
        s.x = normal(rows, cols) * 1.5 + normal(cols) * 0.5
        s.w, s.b = 1 + 0.1 * normal(cols), 0.1 * normal(cols)
        s.dy = normal(rows, cols) if case["train"] else None
    elif kind == "rope":
        rows, heads, dim = case["batch"] * case["seq"], case["heads"], case["dim"]
        s.buffer = normal(rows, (heads + case["more"]) * dim)
        s.dy = normal(rows, heads * dim) if case["train"] else None
        if case["far"]:
            s.positions = torch.randint(case["far"] // 2, case["far"] + 1, (rows,), generator=g,
                                        device="cuda", dtype=torch.int32)
        else:
            s.positions = torch.arange(case["seq"], device="cuda", dtype=torch.int32).repeat(case["batch"])
    elif kind == "attention":
        B, Lq, Lk, Hq, Hkv, D = (case[n] for n in ("batch", "q_rows", "k_rows", "q_heads", "kv_heads", "dim"))
        s.q, s.k, s.v = normal(B, Lq, Hq, D), normal(B, Lk, Hkv, D), normal(B, Lk, Hkv, D)
        n = _lengths(case, seed)
        s.k_len = torch.from_numpy(n).cuda()
        # a training sequence starts at position 0 and has as many queries as
        # keys; what answers appends its tokens behind what the cache holds
        s.q_len = s.k_len.clone() if case["train"] else None
        s.q_start = torch.zeros_like(s.k_len) if case["train"] else (s.k_len - Lq)
        s.scale = 1.0 / math.sqrt(D)
        if case["train"]:
            valid = torch.arange(Lq, device="cuda")[None, :] < s.q_len[:, None]
            s.dout = normal(B, Lq, Hq, D) * valid[:, :, None, None]
    else:
        rows, cols, top = case["rows"], case["cols"], case["top"]
        s.logits = normal(rows, cols) * 2.0
        # a teacher's top logits: other columns in each row, falling from the first
        first = torch.randint(0, cols, (rows, 1), generator=g, device="cuda")
        step = cols // top
        s.ids = ((first + torch.arange(top, device="cuda")[None, :] * step) % cols).to(torch.int32)
        s.teacher = (8.0 + normal(rows, top)).sort(dim=1, descending=True).values.contiguous()
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return (_OWN if own else _PLAIN)[s.case["kind"]](s)


# the framework's operators: raw device pointers, as its C callers hand them over

_handles = {}


def _framework():
    if not _handles:
        import tinytorch_amd
        _handles["pkg"] = tinytorch_amd
        _handles["lib"] = tinytorch_amd.lib()
    return _handles["pkg"], _handles["lib"]


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"failed with {rc}")


def _own_norm(s):
    _, L = _framework()
    rows, cols = s.x.shape
    y = torch.empty_like(s.x)
    if not s.case["train"]:
        _ok(L.tt_k_layernorm_fwd(s.x.data_ptr(), s.w.data_ptr(), s.b.data_ptr(), y.data_ptr(), None, None,
                                 rows, cols, EPS))
        return y
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dx, dw, db = torch.empty_like(s.x), torch.empty_like(s.w), torch.empty_like(s.b)
    _ok(L.tt_k_layernorm_fwd(s.x.data_ptr(), s.w.data_ptr(), s.b.data_ptr(), y.data_ptr(), mean.data_ptr(),
                             rstd.data_ptr(), rows, cols, EPS))
    _ok(L.tt_k_layernorm_bwd(s.x.data_ptr(), s.w.data_ptr(), s.dy.data_ptr(), mean.data_ptr(),
                             rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), rows, cols, None))
    return [y, dx, dw, db]


def _own_rope(s):
    P, L = _framework()
    c = s.case
    rows, width = s.buffer.shape
    scaling, factor, trained, low, high = SCALING[c["scaling"]]
    r = P.Rope(head_dim=c["dim"], rot_dim=c["rot"], interleaved=int(c["interleaved"]), scaling=scaling,
               base=BASE, factor=factor, trained=trained, low=low, high=high, magnitude=1.0)
    y = torch.empty((rows, c["heads"] * c["dim"]), device="cuda")
    _ok(L.tt_k_rope(r, s.buffer.data_ptr(), y.data_ptr(), s.positions.data_ptr(), rows, c["seq"], c["heads"],
                    width, y.shape[1], 0))
    if not c["train"]:
        return y
    dx = torch.empty_like(y)
    _ok(L.tt_k_rope(r, s.dy.data_ptr(), dx.data_ptr(), s.positions.data_ptr(), rows, c["seq"], c["heads"],
                    y.shape[1], y.shape[1], 1))
    return [y, dx]


def _own_attention(s):
    P, L = _framework()
    c = s.case
    a = P.Attention(batch=c["batch"], q_rows=c["q_rows"], k_rows=c["k_rows"], q_heads=c["q_heads"],
                    kv_heads=c["kv_heads"], head_dim=c["dim"], causal=int(c["causal"]), window=c["window"],
                    scale=s.scale, q_start=s.q_start.data_ptr(),
                    q_len=s.q_len.data_ptr() if s.q_len is not None else None, k_len=s.k_len.data_ptr())
    q, k, v = s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr()
    o = torch.empty_like(s.q)
    if not c["train"]:
        _ok(L.tt_k_attention_fwd(a, q, k, v, o.data_ptr(), None, None))
        return o
    lse = torch.empty((c["batch"], c["q_heads"], c["q_rows"]), device="cuda")
    dq, dk, dv = torch.empty_like(s.q), torch.empty_like(s.k), torch.empty_like(s.v)
    _ok(L.tt_k_attention_fwd(a, q, k, v, o.data_ptr(), lse.data_ptr(), None))
    _ok(L.tt_k_attention_bwd(a, q, k, v, o.data_ptr(), s.dout.data_ptr(), lse.data_ptr(), dq.data_ptr(),
                             dk.data_ptr(), dv.data_ptr(), None))
    return [o, dq, dk, dv]


def _own_distill(s):
    _, L = _framework()
    c = s.case
    loss = torch.empty(c["rows"], device="cuda")
    dz = torch.empty_like(s.logits) if c["train"] else None
    _ok(L.tt_k_distill(s.logits.data_ptr(), s.ids.data_ptr(), s.teacher.data_ptr(), c["top"],
                       c["temperature"], loss.data_ptr(), dz.data_ptr() if c["train"] else None, c["rows"],
                       c["cols"], 1.0 / c["rows"]))
    return [loss, dz] if c["train"] else loss


_OWN = dict(norm=_own_norm, rope=_own_rope, attention=_own_attention, distill=_own_distill)


# the same in elementary operations of 32 bits

def _plain_norm(s):
    d = s.x - s.x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    h = d * r
    y = h * s.w + s.b
    if not s.case["train"]:
        return y
    g = s.dy * s.w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return [y, dx, (s.dy * h).sum(0), s.dy.sum(0)]


def _frequencies(case):
    """Radians a position, in 64 bits: how fast each pair turns."""
    kind, factor, trained, low, high = SCALING[case["scaling"]]
    R = case["rot"]
    base = BASE
    if kind == 2 and R > 2:
        base = BASE * factor ** (R / (R - 2.0))
    f = base ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    if kind == 1:
        f = f / factor
    if kind == 3:
        keep = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = (1 - keep) * f / factor + keep * f
    return f


def _turn(case, x, cos, sin):
    """x (rows, heads, dim) with the pairs of its first `rot` values turned."""
    R = case["rot"]
    first, rest = x[..., :R], x[..., R:]
    if case["interleaved"]:
        a, b = first[..., 0::2], first[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = first[..., :R // 2], first[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, rest], -1)


def _plain_rope(s):
    c = s.case
    rows = s.buffer.shape[0]
    heads, dim = c["heads"], c["dim"]
    angle = s.positions.double()[:, None] * _frequencies(c)
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    y = _turn(c, s.buffer[:, :heads * dim].reshape(rows, heads, dim), cos, sin).reshape(rows, -1)
    if not c["train"]:
        return y
    dx = _turn(c, s.dy.reshape(rows, heads, dim), cos, -sin).reshape(rows, -1)
    return [y, dx]


def _seen(s):
    """(batch, q_rows, k_rows): the keys that each query sees."""
    c = s.case
    i = torch.arange(c["q_rows"], device="cuda")
    j = torch.arange(c["k_rows"], device="cuda")
    at = s.q_start[:, None] + i[None, :]
    seen = (j[None, None, :] < s.k_len[:, None, None]).expand(-1, c["q_rows"], -1)
    if c["causal"]:
        seen = seen & (j[None, None, :] <= at[:, :, None])
    if c["window"]:
        seen = seen & (j[None, None, :] > at[:, :, None] - c["window"])
        if not c["causal"]:
            seen = seen & (j[None, None, :] < at[:, :, None] + c["window"])
    if s.q_len is not None:
        seen = seen & (i[None, :] < s.q_len[:, None])[:, :, None]
    return seen


def _plain_attention(s):
    c = s.case
    B, Lq, Lk, Hq, Hkv, D = (c[n] for n in ("batch", "q_rows", "k_rows", "q_heads", "kv_heads", "dim"))
    G = Hq // Hkv

    def by_head(x, rows):  # (B, rows, Hq, D) -> (B, Hkv, G * rows, D)
        return x.permute(0, 2, 1, 3).reshape(B, Hkv, G * rows, D)

    def back(x, rows):
        return x.reshape(B, Hq, rows, D).permute(0, 2, 1, 3).contiguous()

    q = by_head(s.q, Lq)
    k, v = s.k.permute(0, 2, 1, 3).contiguous(), s.v.permute(0, 2, 1, 3).contiguous()
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s.scale).view(B, Hkv, G, Lq, Lk)
    p.masked_fill_(~_seen(s)[:, None, None], -math.inf)
    most = p.amax(-1, keepdim=True)
    p.sub_(torch.where(most == -math.inf, torch.zeros_like(most), most)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    p = p.view(B, Hkv, G * Lq, Lk)
    o = torch.matmul(p, v)
    if not c["train"]:
        return back(o, Lq)
    do = by_head(s.dout, Lq)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s.scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    return [back(o, Lq), back(dq, Lq), dk.permute(0, 2, 1, 3).contiguous(), dv.permute(0, 2, 1, 3).contiguous()]


def _plain_distill(s):
    c = s.case
    T = c["temperature"]
    t = s.teacher / T
    t = t - t.amax(1, keepdim=True)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    p = log_p.exp()
    z = s.logits / T
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    ids = s.ids.long()
    loss = T * T * (p * (log_p - (z.gather(1, ids) - total.log()))).sum(1)
    if not c["train"]:
        return loss
    dz = (e / total).scatter_add(1, ids, -p) * (T / c["rows"])
    return [loss, dz]


_PLAIN = dict(norm=_plain_norm, rope=_plain_rope, attention=_plain_attention, distill=_plain_distill)


# ---------------------------------------------------------------- what a pass needs

def _pairs(case):
    """Query-key pairs of one head over the batch, from the lengths alone."""
    n = np.linspace(case["k_rows"], case["shortest"], case["batch"]).astype(np.int64)
    total = 0
    for length in n:
        rows = int(length) if case["train"] else case["q_rows"]
        at = np.arange(rows) + (0 if case["train"] else int(length) - case["q_rows"])
        high = np.minimum(at + 1, length) if case["causal"] else np.full(rows, length)
        low = np.zeros(rows, np.int64)
        if case["window"]:
            low = np.maximum(at - case["window"] + 1, 0)
            if not case["causal"]:
                high = np.minimum(at + case["window"], length)
        total += int(np.maximum(high - low, 0).sum())
    return total


def work(case):
    """Inputs read once, outputs written once; the multiply-adds of
    attention's products over the pairs that the masks leave, each once, the
    recomputed scores included."""
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["cols"]
        return dict(bytes=4.0 * ((5 if case["train"] else 2) * n + 2 * case["cols"]),
                    flops=(20.0 if case["train"] else 8.0) * n)
    if kind == "rope":
        n = case["batch"] * case["seq"] * case["heads"] * case["dim"]
        return dict(bytes=(16.0 if case["train"] else 8.0) * n, flops=(6.0 if case["train"] else 3.0) * n)
    if kind == "attention":
        q = case["batch"] * case["q_rows"] * case["q_heads"] * case["dim"]
        held = np.linspace(case["k_rows"], case["shortest"], case["batch"]).astype(np.int64).sum()
        kv = int(held) * case["kv_heads"] * case["dim"]
        products = 7 if case["train"] else 2
        return dict(bytes=4.0 * (8 * q + 6 * kv if case["train"] else 2 * q + 2 * kv),
                    flops=2.0 * products * case["dim"] * case["q_heads"] * _pairs(case))
    n = case["rows"] * case["cols"]
    return dict(bytes=4.0 * n * (2 if case["train"] else 1) + 8.0 * case["rows"] * case["top"],
                flops=(6.0 if case["train"] else 4.0) * n)


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return dict(norm=_exact_norm, rope=_exact_rope, attention=_exact_attention, distill=_exact_distill)[
        case["kind"]](case, s)


def _exact_norm(case, s):
    x = s.x.double().requires_grad_(True)
    w, b = s.w.double().requires_grad_(True), s.b.double().requires_grad_(True)
    var = x.var(1, unbiased=False, keepdim=True)
    y = (x - x.mean(1, keepdim=True)) / (var + EPS).sqrt() * w + b
    if not case["train"]:
        return y.detach()
    y.backward(s.dy.double())
    return [y.detach(), x.grad, w.grad, b.grad]


def _exact_rope(case, s):
    """The pairs as complex numbers, times e^(i angle)."""
    kind, factor, trained, low, high = SCALING[case["scaling"]]
    R, dim, heads = case["rot"], case["dim"], case["heads"]
    rows = s.buffer.shape[0]
    f = []
    for j in range(R // 2):
        base = BASE * factor ** (R / (R - 2.0)) if kind == 2 and R > 2 else BASE
        w = math.exp(-2.0 * j / R * math.log(base))
        if kind == 1:
            w /= factor
        if kind == 3:
            turns = trained * w / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            w = w / factor * (1 - keep) + w * keep
        f.append(w)
    angle = s.positions.double()[:, None] * torch.tensor(f, device="cuda", dtype=torch.float64)
    unit = torch.polar(torch.ones_like(angle), angle)[:, None, :]

    def turn(x, by):
        x = x.double().reshape(rows, heads, dim)
        even, odd = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(x[..., even], x[..., odd]) * by
        out = x.clone()
        out[..., even], out[..., odd] = z.real, z.imag
        return out.reshape(rows, -1)

    y = turn(s.buffer[:, :heads * dim], unit)
    return [y, turn(s.dy, unit.conj())] if case["train"] else y


def _exact_attention(case, s):
    """Head by head; the gradients by differentiation."""
    B, Hq, Hkv = case["batch"], case["q_heads"], case["kv_heads"]
    q, k, v = s.q.double(), s.k.double(), s.v.double()
    o = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    i, j = torch.arange(case["q_rows"], device="cuda")[:, None], torch.arange(case["k_rows"], device="cuda")[None, :]
    lengths, starts = s.k_len.tolist(), s.q_start.tolist()
    for b in range(B):
        hidden = j >= lengths[b]
        if case["causal"]:
            hidden = hidden | (j > i + starts[b])
        if case["window"]:
            gap = i + starts[b] - j
            hidden = hidden | ((gap if case["causal"] else gap.abs()) >= case["window"])
        if s.q_len is not None:
            hidden = hidden | (i >= lengths[b])
        empty = hidden.all(1, keepdim=True)
        for h in range(Hq):
            n = h // (Hq // Hkv)
            one = [t.clone().requires_grad_(case["train"]) for t in (q[b, :, h], k[b, :, n], v[b, :, n])]
            scores = (one[0] @ one[1].t() * s.scale).masked_fill(hidden & ~empty, -math.inf)
            y = torch.softmax(scores, 1).masked_fill(empty, 0.0) @ one[2]
            o[b, :, h] = y.detach()
            if case["train"]:
                y.backward(s.dout[b, :, h].double())
                dq[b, :, h] = one[0].grad
                dk[b, :, n] += one[1].grad
                dv[b, :, n] += one[2].grad
    return [o, dq, dk, dv] if case["train"] else o


def _exact_distill(case, s):
    T = case["temperature"]
    loss, dz = [], []
    for at in range(0, case["rows"], 512):
        z = s.logits[at:at + 512].double().requires_grad_(case["train"])
        p = torch.softmax(s.teacher[at:at + 512].double() / T, 1)
        log_q = torch.log_softmax(z / T, 1).gather(1, s.ids[at:at + 512].long())
        row = T * T * (p * (p.log() - log_q)).sum(1)
        loss.append(row.detach())
        if case["train"]:
            (row.sum() / case["rows"]).backward()
            dz.append(z.grad)
    return [torch.cat(loss), torch.cat(dz)] if case["train"] else torch.cat(loss)
