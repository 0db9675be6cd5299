"""What the operators of a language model's training step are timed on, apart from
those of operators.py: token embeddings, RMS norm with the residual's addition, and
the orthogonalised update of weight matrices, through the device-level entry points
of tt_hip.h, over the sizes they are used with.

Kinds of case:

  embedding  the scaled rows of a table at a batch's tokens; `train`: then the
             table's gradient.  Tokens are as often as words are (the n-th most
             frequent 1 / n as often as the first), `padded` of them are -1.
  rms        h = x + residual (or x alone), y = the RMS norm of h times a weight;
             `train`: then the gradients of x (the residual's is the same) and of the
             weight, from those of y and h.
  orthogonal the matrices that Newton-Schulz steps make of `count` matrices.
  muon       a step of the optimizer on the weight matrices named in `shapes`: the
             momenta and weights after it.

Everything is fp32, the one type the framework computes in.
"""
import ctypes
import functools
import math

import numpy as np
import torch

own = False  # False: the operators in elementary torch operations


# ---------------------------------------------------------------- the cases

def _embedding(name, rows, vocab, cols, padded, train):
    return dict(name=name, kind="embedding", rows=rows, vocab=vocab, cols=cols, padded=padded, train=train)


def _rms(name, rows, cols, residual, train):
    return dict(name=name, kind="rms", rows=rows, cols=cols, residual=residual, train=train)


def _orthogonal(name, count, rows, cols, steps):
    return dict(name=name, kind="orthogonal", count=count, rows=rows, cols=cols, steps=steps)


def _muon(name, shapes, nesterov):
    return dict(name=name, kind="muon", shapes=shapes, nesterov=nesterov)


def listed():
    return [
        # the next tokens of 32 conversations: latency
        _embedding("embedding_tokens_32", 32, 32000, 1024, 0.0, False),
        # a training batch of 8 x 1024 tokens
        _embedding("embedding_train", 8192, 32000, 1024, 0.0, True),
        # a padded batch over a small vocabulary: no row but the first is aligned
        _embedding("embedding_odd", 4099, 1003, 259, 0.1, True),
        # long sequences over a large vocabulary
        _embedding("embedding_train_long", 32768, 131072, 1024, 0.02, True),
        # one token on its way through a trained model: latency
        _rms("rms_token", 1, 1024, True, False),
        # the activations of a training batch of 8 x 1024 tokens
        _rms("rms_train", 8192, 1024, True, True),
        # odd rows and columns, and no residual: a model's last norm
        _rms("rms_odd", 4099, 1003, False, True),
        # wide rows
        _rms("rms_train_wide", 4096, 8192, True, True),
        # the weights of the three-layer MLP that the benchmark trains: latency
        _muon("muon_mlp", "785x256 257x128 129x10", True),
        # a transformer block's weights
        _muon("muon_block", "1024x1024 1024x1024 1024x1024 1024x1024 1024x4096 4096x1024", True),
        # a matrix of odd sides
        _orthogonal("orthogonal_odd", 1, 1003, 517, 5),
        # a large one
        _orthogonal("orthogonal_large", 1, 4096, 4096, 5),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm; odd ones too."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# no drawn case costs more than the largest listed ones
MOST_BYTES, MOST_FLOPS = 1.02e9, 1.37e12


def draw(rng):
    while True:
        kind = rng.choice(["embedding", "embedding", "rms", "rms", "orthogonal", "muon", "muon"])
        if kind == "embedding":
            c = _embedding("", _log(rng, 1, 32768), _log(rng, 100, 131072), _log(rng, 16, 4096),
                           rng.choice([0.0, round(rng.uniform(0.01, 0.6), 2)]), rng.random() < 0.75)
        elif kind == "rms":
            c = _rms("", _log(rng, 1, 16384), _log(rng, 16, 16384), rng.random() < 0.7, rng.random() < 0.7)
        elif kind == "orthogonal":
            c = _orthogonal("", _log(rng, 1, 32), _log(rng, 4, 4096), _log(rng, 4, 4096), rng.choice([5, 5, 3, 6]))
        else:
            shapes = ["%dx%d" % (_log(rng, 4, 4096), _log(rng, 4, 4096)) for _ in range(rng.randint(1, 8))]
            c = _muon("", " ".join(shapes), rng.random() < 0.7)
        w = work(c)
        if w["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS:
            continue
        del c["name"]
        return c


def _shapes(case):
    if case["kind"] == "orthogonal":
        return [(case["rows"], case["cols"])] * case["count"]
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()]


# ---------------------------------------------------------------- inputs

EPS = 1e-5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
STEPS = 5  # Newton-Schulz steps of the optimizer
COEFFICIENTS = 3.4445, -4.7750, 2.0315


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def gradient(rows, cols):
        """As a batch leaves it: a few strong directions over many weak ones."""
        few = max(1, min(rows, cols) // 16)
        return 1e-3 * (normal(rows, few) @ normal(few, cols) / math.sqrt(few) + 0.3 * normal(rows, cols))

    kind = case["kind"]
    if kind == "embedding":
        rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
        s.w = normal(vocab, cols) * 0.02
        rank = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        rank = (torch.exp(rank * math.log(vocab + 1.0)) - 1.0).long().clamp(0, vocab - 1)
        s.ids = torch.randperm(vocab, generator=g, device="cuda")[rank].to(torch.int32)
        s.ids[torch.rand(rows, generator=g, device="cuda") < case["padded"]] = -1
        s.scale = math.sqrt(cols)
        s.dy = normal(rows, cols) if case["train"] else None
    elif kind == "rms":
        rows, cols = case["rows"], case["cols"]
        s.x = normal(rows, cols)
        # a stream whose columns differ in size
        s.residual = normal(rows, cols) * torch.exp(normal(cols)) if case["residual"] else None
        s.w = 1 + 0.1 * normal(cols)
        s.dy = normal(rows, cols) if case["train"] else None
        s.dh = normal(rows, cols) if case["train"] and case["residual"] else None
    elif kind == "orthogonal":
        s.x = torch.stack([gradient(case["rows"], case["cols"]) for _ in range(case["count"])])
    else:
        s.shapes = _shapes(case)
        s.w = [normal(*n) / math.sqrt(n[0]) for n in s.shapes]
        s.g = [gradient(*n) for n in s.shapes]
        s.v = [gradient(*n) * 4 for n in s.shapes]
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return (_OWN if own else _PLAIN)[s.case["kind"]](s)


# the framework's operators: raw device pointers, as its C callers hand them over

@functools.cache
def _framework():
    import tinytorch_amd
    return tinytorch_amd.lib()


def _ok(rc):
    if rc != 0:
        raise RuntimeError(f"failed with {rc}")


def _own_embedding(s):
    L = _framework()
    c = s.case
    y = torch.empty((c["rows"], c["cols"]), device="cuda")
    _ok(L.tt_k_embedding_fwd(s.w.data_ptr(), s.ids.data_ptr(), y.data_ptr(), c["rows"], c["vocab"], c["cols"],
                             s.scale))
    if not c["train"]:
        return y
    dw = torch.empty_like(s.w)
    _ok(L.tt_k_embedding_bwd(s.ids.data_ptr(), s.dy.data_ptr(), dw.data_ptr(), c["rows"], c["vocab"], c["cols"],
                             s.scale, 0, None))
    return [y, dw]


def _own_rms(s):
    L = _framework()
    rows, cols = s.x.shape
    y, rstd = torch.empty_like(s.x), torch.empty(rows, device="cuda")
    h = torch.empty_like(s.x) if s.case["residual"] else None
    _ok(L.tt_k_rmsnorm_fwd(s.x.data_ptr(), s.residual.data_ptr() if s.case["residual"] else None, s.w.data_ptr(),
                           y.data_ptr(), h.data_ptr() if s.case["residual"] else None,
                           rstd.data_ptr() if s.case["train"] else None, rows, cols, EPS))
    out = [y, h] if s.case["residual"] else [y]
    if not s.case["train"]:
        return out
    dx, dw = torch.empty_like(s.x), torch.empty_like(s.w)
    _ok(L.tt_k_rmsnorm_bwd((h if s.case["residual"] else s.x).data_ptr(), s.w.data_ptr(), s.dy.data_ptr(),
                           s.dh.data_ptr() if s.case["residual"] else None, rstd.data_ptr(), dx.data_ptr(),
                           dw.data_ptr(), rows, cols, None))
    return out + [dx, dw]


def _own_orthogonal(s):
    L = _framework()
    y = torch.empty_like(s.x)
    _ok(L.tt_k_newton_schulz(s.x.data_ptr(), y.data_ptr(), s.case["count"], s.case["rows"], s.case["cols"],
                             s.case["steps"], None))
    return y


def _own_muon(s):
    L = _framework()
    n = len(s.shapes)
    w, v = [torch.empty_like(t) for t in s.w], [torch.empty_like(t) for t in s.v]
    for new, old in zip(w + v, s.w + s.v):  # the step is in place, and the state stays as it is
        _ok(L.tt_k_copy(new.data_ptr(), old.data_ptr(), old.numel()))

    def pointers(ts):
        return (ctypes.c_void_p * n)(*[t.data_ptr() for t in ts])

    rows, cols = (ctypes.c_long * n)(*[a for a, _ in s.shapes]), (ctypes.c_long * n)(*[b for _, b in s.shapes])
    _ok(L.tt_k_muon_multi(pointers(w), pointers(s.g), pointers(v), rows, cols, n, LR, MOMENTUM,
                          int(s.case["nesterov"]), DECAY, None))
    return [w, v]


_OWN = dict(embedding=_own_embedding, rms=_own_rms, orthogonal=_own_orthogonal, muon=_own_muon)


# the same in elementary operations of 32 bits

def _plain_embedding(s):
    c = s.case
    has = ((s.ids >= 0) & (s.ids < c["vocab"])).float()[:, None] * s.scale
    at = s.ids.long().clamp(0, c["vocab"] - 1)
    y = s.w[at] * has
    if not c["train"]:
        return y
    return [y, torch.zeros_like(s.w).index_add_(0, at, s.dy * has)]


def _plain_rms(s):
    h = s.x + s.residual if s.case["residual"] else s.x
    r = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * r * s.w
    out = [y, h] if s.case["residual"] else [y]
    if not s.case["train"]:
        return out
    g = s.dy * s.w
    dx = r * g - h * (r * r * r * (g * h).mean(1, keepdim=True))
    if s.case["residual"]:
        dx = dx + s.dh
    return out + [dx, (s.dy * h * r).sum(0)]


def _steps(x, steps):
    """Newton-Schulz steps of matrices x (..., rows, cols), along their shorter side."""
    a, b, c = COEFFICIENTS
    turned = x.shape[-2] > x.shape[-1]
    x = (x.mT if turned else x).contiguous()
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = (x.double() / torch.where(norm == 0, torch.ones_like(norm), norm)).float()
    for _ in range(steps):
        p = x @ x.mT
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.mT.contiguous() if turned else x


def _plain_orthogonal(s):
    return _steps(s.x, s.case["steps"])


def _plain_muon(s):
    w, v = [], []
    for wi, gi, vi in zip(s.w, s.g, s.v):
        m = MOMENTUM * vi + gi
        u = gi + MOMENTUM * m if s.case["nesterov"] else m
        w.append((1 - LR * DECAY) * wi - LR * 0.2 * math.sqrt(max(wi.shape)) * _steps(u, STEPS))
        v.append(m)
    return [w, v]


_PLAIN = dict(embedding=_plain_embedding, rms=_plain_rms, orthogonal=_plain_orthogonal, muon=_plain_muon)


# ---------------------------------------------------------------- what a pass needs

@functools.cache
def _distinct(rows, vocab):
    """How many tokens of the vocabulary a batch holds, as expected."""
    n = np.arange(1, vocab + 1)
    p = np.log((n + 1) / n) / math.log(vocab + 1.0)
    return float((1 - (1 - p) ** rows).sum())


def work(case):
    """Inputs read once, outputs written once; a symmetric product once for each
    pair."""
    kind = case["kind"]
    if kind == "embedding":
        rows, cols = case["rows"] * (1 - case["padded"]), case["cols"]
        values = _distinct(int(math.ceil(rows)), case["vocab"]) * cols + case["rows"] * cols
        if case["train"]:
            values += rows * cols + case["vocab"] * cols
        return dict(bytes=4.0 * (values + case["rows"]), flops=(2.0 if case["train"] else 1.0) * rows * cols)
    if kind == "rms":
        n = case["rows"] * case["cols"]
        passes = 4 if case["residual"] else 2
        if case["train"]:
            passes += 4 if case["residual"] else 3
        return dict(bytes=4.0 * (passes * n + case["cols"]), flops=(14.0 if case["train"] else 5.0) * n)
    values, flops = 0.0, 0.0
    for rows, cols in _shapes(case):
        m, n = min(rows, cols), max(rows, cols)
        values += rows * cols * (2 if kind == "orthogonal" else 5)
        flops += case.get("steps", STEPS) * (m * m * n + m * m * m + 2.0 * m * m * n)
    return dict(bytes=4.0 * values, flops=flops)


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return dict(embedding=_exact_embedding, rms=_exact_rms, orthogonal=_exact_orthogonal,
                muon=_exact_muon)[case["kind"]](case, s)


def _exact_embedding(case, s):
    """With the table's gradient by sorted tokens and the differences of running sums,
    a few columns at a time."""
    vocab, cols = case["vocab"], case["cols"]
    ids = s.ids.long()
    hidden = (ids < 0) | (ids >= vocab)
    y = (s.w.double()[ids.masked_fill(hidden, 0)] * s.scale).masked_fill(hidden[:, None], 0.0)
    if not case["train"]:
        return y
    key, order = ids.masked_fill(hidden, vocab).sort(stable=True)
    ends = torch.searchsorted(key, torch.arange(vocab + 1, device="cuda"))
    dw = torch.empty(vocab, cols, device="cuda", dtype=torch.float64)
    for c in range(0, cols, 64):
        total = torch.zeros(len(order) + 1, min(64, cols - c), device="cuda", dtype=torch.float64)
        torch.cumsum(s.dy[order, c:c + 64].double(), 0, out=total[1:])
        dw[:, c:c + 64] = (total[ends[1:]] - total[ends[:-1]]) * s.scale
    return [y, dw]


def _exact_rms(case, s):
    x = s.x.double()
    h = (x + s.residual.double() if case["residual"] else x).requires_grad_(case["train"])
    w = s.w.double().requires_grad_(case["train"])
    y = h / (h.square().sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * w
    out = [y.detach(), h.detach()] if case["residual"] else [y.detach()]
    if not case["train"]:
        return out
    y.backward(s.dy.double())
    return out + [h.grad + s.dh.double() if case["residual"] else h.grad, w.grad]


def _exact_steps(x, steps):
    """The polynomial of the squares, along the shorter side on the right."""
    a, b, c = COEFFICIENTS
    x = x.double()
    wide = x.shape[1] > x.shape[0]
    x = x.t() if wide else x
    norm = torch.linalg.matrix_norm(x)
    x = x / norm if norm > 0 else x
    one = torch.eye(x.shape[1], device="cuda", dtype=torch.float64)
    for _ in range(steps):
        p = x.t() @ x
        x = x @ (a * one + p @ (b * one + c * p))
    return (x.t() if wide else x).contiguous()


def _exact_orthogonal(case, s):
    return torch.stack([_exact_steps(x, case["steps"]) for x in s.x])


def _exact_muon(case, s):
    w, v = [], []
    for wi, gi, vi in zip(s.w, s.g, s.v):
        wi, gi, vi = wi.double(), gi.double(), vi.double()
        m = vi * MOMENTUM + gi
        u = m * MOMENTUM + gi if case["nesterov"] else m
        v.append(m)
        w.append(wi - LR * (DECAY * wi + 0.2 * math.sqrt(max(wi.shape)) * _exact_steps(u, STEPS)))
    return [w, v]
