"""The regression operators as they are measured: their cases, their inputs, their plain forms and what they cost.

    loss       the log loss of count rows under a linear predictor z = H W' + b, softmax (multinomial) or exp (Dirichlet)
    gradient   the same loss with its gradients in H, W and b: a training step's work
    step       an update matrix replaced by its nearly orthogonal factor: odd matrix polynomials of degree five

With F(z, x) = x z and G(z, x) = x (multinomial), or F = lgamma(e^z + x) - lgamma(e^z) and
G = e^z (psi(e^z + x) - psi(e^z)) (Dirichlet), a row of counts x with total T and l = log sum_k exp z_k has

    loss = F(l, T) - sum_k F(z_k, x_k),      d loss / d z_k = exp(z_k - l) G(l, T) - G(z_k, x_k).
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one document scored against the whole vocabulary, as a service answers: latency and one read of the weights
        {"name": "score_one", "op": "loss", "model": "multinomial", "rows": "csr", "n": 1, "k": 50000, "d": 512, "type": "bf16"},
        # a handful of documents, odd sizes, full precision
        {"name": "score_few", "op": "loss", "model": "dirichlet", "rows": "csr", "n": 7, "k": 20011, "d": 200, "type": "f32"},
        # held-out loss of next-word labels
        {"name": "evaluate_labels", "op": "loss", "model": "multinomial", "rows": "labels", "n": 4096, "k": 50000, "d": 512, "type": "bf16"},
        # held-out loss of a dense count matrix of 1000 categories
        {"name": "evaluate_dense", "op": "loss", "model": "dirichlet", "rows": "dense", "n": 32768, "k": 1000, "d": 128, "type": "bf16"},
        # a training step on labels over the whole vocabulary: the largest
        {"name": "train_labels", "op": "gradient", "model": "multinomial", "rows": "labels", "n": 8192, "k": 50000, "d": 1024, "type": "bf16"},
        # a training step of a topic model's decoder: bags of words, a ragged last tile
        {"name": "train_words", "op": "gradient", "model": "multinomial", "rows": "csr", "n": 4099, "k": 50000, "d": 128, "type": "bf16"},
        # the same in full precision at odd sizes
        {"name": "train_words_f32", "op": "gradient", "model": "multinomial", "rows": "csr", "n": 1024, "k": 10007, "d": 100, "type": "f32"},
        # over-dispersed bags of words: the Dirichlet link
        {"name": "train_dirichlet", "op": "gradient", "model": "dirichlet", "rows": "csr", "n": 4096, "k": 50000, "d": 256, "type": "bf16"},
        # over-dispersed dense rows of 1000 categories in full precision
        {"name": "train_dense", "op": "gradient", "model": "dirichlet", "rows": "dense", "n": 16384, "k": 1000, "d": 64, "type": "f32"},
        # the step of a small weight matrix: launches and latency
        {"name": "step_small", "op": "step", "b": 1, "m": 1000, "n": 64, "type": "f32"},
        # the step of the vocabulary's weights
        {"name": "step_vocabulary", "op": "step", "b": 1, "m": 50000, "n": 256, "type": "bf16"},
        # the step of a large square matrix: products alone
        {"name": "step_square", "op": "step", "b": 1, "m": 4096, "n": 4096, "type": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["loss", "loss", "gradient", "gradient", "step"])
    kind = rng.choice(["bf16", "f32"])
    if op == "step":
        b = rng.choice([1, 1, 1, _spread(rng, 2, 8)])
        m, n = _spread(rng, 64, 20000), _spread(rng, 48, 1024)
        if rng.random() < 0.5:
            m, n = n, m
        return {"op": op, "b": b, "m": m, "n": n, "type": kind}
    rows = rng.choice(["csr", "csr", "labels", "dense"])
    k = _spread(rng, 100, 2000) if rows == "dense" else _spread(rng, 1000, 50000)
    n = _spread(rng, 1, 4096 if kind == "f32" else 8192)
    d = _spread(rng, 16, 512 if kind == "f32" else 1024)
    return {"op": op, "model": rng.choice(["multinomial", "dirichlet"]), "rows": rows, "n": n, "k": k, "d": d, "type": kind}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _csr(n, k, gen, dev):
    """Bags of words: up to 96 draws a row (one row in twenty is empty), columns log-uniform as word ranks are,
    ascending within a row, repeated draws merged into a count."""
    most = 96
    length = torch.exp(torch.randn(n, generator=gen, device=dev) * 0.6 + 3.8).clamp(1, most).long()
    if n > 1:
        length = length * (torch.rand(n, generator=gen, device=dev) >= 0.05)
    col = (float(k) ** torch.rand(n, most, generator=gen, device=dev, dtype=torch.float64)).long().sub_(1).clamp_(0, k - 1)
    col = torch.where(torch.arange(most, device=dev) < length[:, None], col, k)
    col = col.sort(dim=1).values
    first = torch.ones_like(col, dtype=torch.bool)
    first[:, 1:] = col[:, 1:] != col[:, :-1]
    real = col < k
    first &= real
    at = first.reshape(-1).long().cumsum(0) - 1
    nnz = int(at[-1]) + 1
    vals = torch.zeros(max(nnz, 1), dtype=torch.int32, device=dev)
    flat = real.reshape(-1)
    vals.index_add_(0, at[flat], torch.ones(int(flat.sum()), dtype=torch.int32, device=dev))
    rowptr = torch.zeros(n + 1, dtype=torch.int64, device=dev)
    rowptr[1:] = first.sum(1).cumsum(0)
    return rowptr, col[first].to(torch.int32), vals[:nnz]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(1000003 * int(seed) + 17)
    dtype = TYPES[case["type"]]
    if case["op"] == "step":
        b, m, n = case["b"], case["m"], case["n"]
        # a gradient as training gives it: a few strong directions over noise
        r = max(1, min(m, n) // 8)
        scale = torch.arange(1, r + 1, device=dev, dtype=torch.float32) ** -0.5
        left = torch.randn(b, m, r, generator=gen, device=dev) * scale
        right = torch.randn(b, r, n, generator=gen, device=dev)
        g = (left @ right) * (1.5 / math.sqrt(r)) + torch.randn(b, m, n, generator=gen, device=dev)
        g = (g * 1e-3).to(dtype)
        return {"case": case, "g": g[0] if b == 1 else g}
    n, k, d = case["n"], case["k"], case["d"]
    s = {"case": case}
    s["h"] = torch.randn(n, d, generator=gen, device=dev).to(dtype)
    s["w"] = (torch.randn(k, d, generator=gen, device=dev) * (0.7 / math.sqrt(d))).to(dtype)
    # the baseline: log alphas that fall off as word frequencies do
    rank = torch.arange(k, device=dev, dtype=torch.float32)
    s["b"] = 1.0 - 0.9 * torch.log(rank + 3.0) + 0.3 * torch.randn(k, generator=gen, device=dev)
    # how much of each row's weight belongs to this component of a mixture
    s["g"] = torch.rand(n, generator=gen, device=dev)
    if case["rows"] == "labels":
        y = (float(k) ** torch.rand(n, generator=gen, device=dev, dtype=torch.float64)).long().sub_(1).clamp_(0, k - 1)
        s["labels"] = torch.where(torch.rand(n, generator=gen, device=dev) < 0.02, -1, y) if n > 1 else y
    elif case["rows"] == "csr":
        s["rowptr"], s["col"], s["val"] = _csr(n, k, gen, dev)
    else:
        x = torch.empty(n, k, device=dev).exponential_(0.4, generator=gen) - 2.0
        x = x.clamp_(min=0.0).ceil_().to(torch.int32)
        if n > 1:
            x *= (torch.rand(n, 1, generator=gen, device=dev) >= 0.02).to(torch.int32)
        s["x"] = x.to(torch.uint16) if case["type"] == "bf16" else x
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "step":
        return _own_step(state) if own else _plain_step(state)
    return _own_loss(state) if own else _plain_loss(state)


def _own_step(state):
    from bayespy_amd import regression
    return {"step": regression.orthogonal_step(state["g"], steps=5, coefficients=COEFFICIENTS)}


def _own_loss(state):
    from bayespy_amd import regression
    case = state["case"]
    if case["rows"] == "labels":
        rows = regression.CountRows.from_labels(state["labels"], case["k"])
    elif case["rows"] == "csr":
        rows = regression.CountRows.from_csr(state["rowptr"], state["col"], state["val"], case["k"])
    else:
        rows = regression.CountRows.from_dense(state["x"])
    if case["op"] == "loss":
        return {"loss": regression.log_loss(state["h"], state["w"], rows, bias=state["b"], likelihood=case["model"])}
    loss, dh, dw, db = regression.log_loss_gradient(state["h"], state["w"], rows, bias=state["b"], likelihood=case["model"],
                                                    row_weights=state["g"])
    return {"loss": loss, "dfeatures": dh, "dweights": dw, "dbias": db}


def _plain_f(z, x, model):
    """F(z, x) in 64 bits."""
    z, x = z.double(), x.double()
    if model == "multinomial":
        return x * z
    a = z.exp()
    return torch.where(x > 0, torch.lgamma(a + x) - torch.lgamma(a), torch.zeros_like(a))


def _plain_g(z, x, model):
    """G(z, x) in 64 bits."""
    z, x = z.double(), x.double()
    if model == "multinomial":
        return x
    a = z.exp()
    return torch.where(x > 0, a * (torch.digamma(a + x) - torch.digamma(a)), torch.zeros_like(a))


def _plain_loss(state):
    case = state["case"]
    n, model = case["n"], case["model"]
    h, w = state["h"].float(), state["w"].float()
    z = h @ w.t() + state["b"]
    top = z.amax(dim=1, keepdim=True)
    lse = (top + torch.exp(z - top).sum(dim=1, keepdim=True).log()).squeeze(1)
    if case["rows"] == "dense":
        x = state["x"].to(torch.int32)
        total = x.sum(dim=1)
        inner = _plain_f(z, x, model).sum(dim=1)
    else:
        if case["rows"] == "labels":
            row = torch.arange(n, device=z.device)
            col, val = state["labels"].clamp(min=0), (state["labels"] >= 0).long()
        else:
            count = state["rowptr"][1:] - state["rowptr"][:-1]
            row = torch.repeat_interleave(torch.arange(n, device=z.device), count, output_size=state["col"].numel())
            col, val = state["col"].long(), state["val"].long()
        total = torch.zeros(n, dtype=torch.int64, device=z.device).index_add_(0, row, val)
        ze = z[row, col]
        inner = torch.zeros(n, dtype=torch.float64, device=z.device).index_add_(0, row, _plain_f(ze, val, model))
    loss = (_plain_f(lse, total, model) - inner).float()
    if case["op"] == "loss":
        return {"loss": loss}
    dz = torch.exp(z - lse[:, None]) * _plain_g(lse, total, model).float()[:, None]
    if case["rows"] == "dense":
        dz = dz - _plain_g(z, x, model).float()
    else:
        dz[row, col] = dz[row, col] - _plain_g(ze, val, model).float()
    dz = dz * state["g"][:, None]
    return {"loss": loss, "dfeatures": (dz @ w).to(state["h"].dtype), "dweights": (dz.t() @ h).to(state["w"].dtype), "dbias": dz.sum(dim=0)}


def _plain_step(state):
    g = state["g"]
    x = g.float()
    flip = x.shape[-2] > x.shape[-1]
    if flip:
        x = x.transpose(-1, -2).contiguous()
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + 1e-30)
    a, b, c = COEFFICIENTS
    for _ in range(5):
        s = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    if flip:
        x = x.transpose(-1, -2).contiguous()
    return {"step": x.to(g.dtype)}


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "step":
        b, m, n = case["b"], min(case["m"], case["n"]), max(case["m"], case["n"])
        # per product: the symmetric ones by half; one read and one write of the matrix
        return {"bytes": 2.0 * b * m * n * size, "flops": 5.0 * b * (m * m * n + m * m * m + 2.0 * m * m * n)}
    n, k, d = case["n"], case["k"], case["d"]
    rows = {"labels": 8.0 * n, "csr": 8.0 * (n + 1) + 8.0 * 35 * n, "dense": float(size) * n * k}[case["rows"]]
    once = float(size) * (n * d + k * d) + 4.0 * k + rows + 4.0 * n
    if case["op"] == "loss":
        return {"bytes": once, "flops": 2.0 * n * k * d}
    return {"bytes": once + float(size) * (n * d + k * d) + 4.0 * k + 4.0 * n, "flops": 6.0 * n * k * d}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "step":
        return {"step": _exact_step(s["g"])}
    n, k, model = case["n"], case["k"], case["model"]
    w, bias = s["w"].double(), s["b"].double()
    out = {"loss": [], "dfeatures": [], "dweights": torch.zeros_like(w), "dbias": torch.zeros_like(bias)}
    for at in range(0, n, 1024):
        end = min(n, at + 1024)
        x = torch.zeros(end - at, k, dtype=torch.float64, device=w.device)
        if case["rows"] == "dense":
            x += s["x"][at:end].to(torch.int32)
        elif case["rows"] == "labels":
            y = s["labels"][at:end]
            has = torch.nonzero(y >= 0).squeeze(1)
            x[has, y[has]] = 1.0
        else:
            for_row = torch.searchsorted(s["rowptr"], torch.arange(s["col"].numel(), device=w.device), right=True) - 1
            mine = torch.nonzero((for_row >= at) & (for_row < end)).squeeze(1)
            x[for_row[mine] - at, s["col"][mine].long()] = s["val"][mine].double()
        h = s["h"][at:end].double()
        z = torch.addmm(bias, h, w.t())
        total = x.sum(dim=1)
        lse = torch.logsumexp(z, dim=1)
        if model == "multinomial":
            loss = (x * (lse[:, None] - z)).sum(dim=1)
            dz = total[:, None] * torch.softmax(z, dim=1) - x
        else:
            alpha, mass = z.exp(), lse.exp()
            loss = torch.lgamma(mass + total) - torch.lgamma(mass) - (torch.lgamma(alpha + x) - torch.lgamma(alpha)).sum(dim=1)
            dz = alpha * ((torch.digamma(mass + total) - torch.digamma(mass))[:, None] - (torch.digamma(alpha + x) - torch.digamma(alpha)))
        out["loss"].append(loss)
        if case["op"] == "gradient":
            dz *= s["g"][at:end].double()[:, None]
            out["dfeatures"].append(dz @ w)
            out["dweights"] += dz.t() @ h
            out["dbias"] += dz.sum(dim=0)
    if case["op"] == "loss":
        return {"loss": torch.cat(out["loss"])}
    return {"loss": torch.cat(out["loss"]), "dfeatures": torch.cat(out["dfeatures"]), "dweights": out["dweights"], "dbias": out["dbias"]}


def _exact_step(g):
    """The polynomial p(x) = a x + b x^3 + c x^5 applied five times to the singular values' side of g / |g|."""
    if g.dim() == 3:
        return torch.stack([_exact_step(one) for one in g])
    y = g.double()
    tall = y.shape[0] > y.shape[1]
    y = y / torch.linalg.vector_norm(y)
    a, b, c = COEFFICIENTS
    eye = torch.eye(min(y.shape), dtype=torch.float64, device=y.device)
    for _ in range(5):
        s = y.t() @ y if tall else y @ y.t()
        q = a * eye + s @ (b * eye + c * s)
        y = y @ q if tall else q @ y
    return y
