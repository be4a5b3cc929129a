"""Count rows under a linear predictor (bayespy_amd.regression) against the definition in 64 bits.

Tolerances.  With A = |H| |W|' the sum of |products| behind z, 32-bit sums of D terms leave z off by at most
dz = (D + 2) 2^-23 A + 2^-23 |bias|.  l is off by as much as the worst z, F(z, x) by G dz <= x dz, so

    loss:  2 T max(dz) + 2^-22 (|F(l, T)| + sum |F(z, x)|) + 2^-22            (32-bit pieces, one rounding at the end)
    p = exp(z - l): relative error e = 2 max(dz) + 2^-22 (|z| + |l| + 4)      (the exponent's rounding, exp2's last bits)
    d loss / d z:  e |p G| + 2^-22 |G(z, x)|, and u = eps / 2 of the operands' type where it is rounded to that type

and dW = dz' H by |H|' times that, N 2^-23 |dz|' |H| of the 32-bit sum over rows, and u |dW| at the end; dH likewise."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def f_of(z, x, likelihood):
    if likelihood == "multinomial":
        return torch.where(x > 0, x * z, torch.zeros_like(z))
    a = z.exp()
    return torch.where(x > 0, torch.lgamma(a + x) - torch.lgamma(a), torch.zeros_like(z))


def g_of(z, x, likelihood):
    if likelihood == "multinomial":
        return x
    a = z.exp()
    return torch.where(x > 0, a * (torch.digamma(a + x) - torch.digamma(a)), torch.zeros_like(z))


def oracle(h, w, b, x, g, likelihood, dtype):
    """Everything in 64 bits, with how far 32-bit sums and one rounding may be off (see above)."""
    h, w, x, g = h.double().cpu(), w.double().cpu(), x.double().cpu(), g.double().cpu()
    n, d = h.shape
    b = torch.zeros(w.shape[0], dtype=torch.float64) if b is None else b.double().cpu()
    z = h @ w.t() + b
    finite = torch.where(torch.isfinite(z), z, torch.zeros_like(z))
    lse = torch.logsumexp(z, dim=1)
    total = x.sum(dim=1)
    fz, gz = f_of(z, x, likelihood), g_of(z, x, likelihood)
    fl, gl = f_of(lse, total, likelihood), g_of(lse, total, likelihood)
    loss = fl - fz.sum(dim=1)
    loss[total == 0] = 0.0
    p = torch.exp(z - lse[:, None])
    raw = torch.where((total > 0)[:, None], p * gl[:, None] - gz, torch.zeros_like(z))
    dz = raw * g[:, None]
    off = (d + 2) * 2.0**-23 * (h.abs() @ w.abs().t()) + 2.0**-23 * torch.where(torch.isfinite(b), b, torch.zeros_like(b)).abs()
    worst = off.max(dim=1).values
    finite_l = torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))
    tol_loss = 2 * total * worst + 2.0**-22 * (fl.abs() + fz.abs().sum(dim=1)) + 2.0**-22
    e = 2 * worst[:, None] + 2.0**-22 * (finite.abs() + finite_l.abs()[:, None] + 4)
    tol_dz = (e * p * gl[:, None].abs() + (2.0**-22 + (worst[:, None] if likelihood == "dirichlet" else 0)) * gz) * g[:, None].abs()
    tol_dz = torch.where((total > 0)[:, None], tol_dz, torch.zeros_like(tol_dz))
    u = torch.finfo(dtype).eps / 2
    round_dz = tol_dz + u * dz.abs()
    dh, dw, db = dz @ w, dz.t() @ h, dz.sum(dim=0)
    k = w.shape[0]
    tol_dh = round_dz @ w.abs() + k * 2.0**-23 * (dz.abs() @ w.abs())
    tol_dw = round_dz.t() @ h.abs() + n * 2.0**-23 * (dz.abs().t() @ h.abs())
    tol_db = tol_dz.sum(dim=0) + n * 2.0**-23 * dz.abs().sum(dim=0)
    return {"loss": (loss, tol_loss), "dh": (dh, tol_dh * (1 + u) + u * dh.abs()), "dw": (dw, tol_dw * (1 + u) + u * dw.abs()),
            "db": (db, tol_db + 2.0**-24 * db.abs())}


def near(got, want, name):
    value, tol = want
    got = got.double().cpu()
    assert got.shape == value.shape, name
    off = (got - value).abs()
    bad = ~(off <= tol + 1e-30)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g of its tolerance" % (
        name, int(bad.sum()), off.numel(), float((off / (tol + 1e-30)).nan_to_num(nan=float("inf")).max()))


def make(n, k, d, dtype, seed, mean=2.0, density=0.2):
    r = np.random.default_rng(seed)
    h = torch.from_numpy(r.standard_normal((n, d))).to(dtype).cuda()
    w = torch.from_numpy(r.standard_normal((k, d)) * 0.7 / np.sqrt(d)).to(dtype).cuda()
    b = torch.from_numpy(r.standard_normal(k) - 1.0).float().cuda()
    x = (r.poisson(mean, size=(n, k)) + 1) * (r.random((n, k)) < density)
    if n > 2:
        x[n // 2] = 0  # a row without counts
    g = torch.from_numpy(r.random(n) * 2 - 0.5).float().cuda()
    return h, w, b, torch.from_numpy(x.astype(np.int32)), g


def as_rows(x, kind):
    from bayespy_amd.regression import CountRows
    k = x.shape[1]
    if kind == "dense32":
        return CountRows.from_dense(x.cuda())
    if kind == "dense16":
        return CountRows.from_dense(x.to(torch.uint16).cuda())
    rowptr = torch.zeros(x.shape[0] + 1, dtype=torch.int64)
    rowptr[1:] = (x > 0).sum(1).cumsum(0)
    at = (x > 0).nonzero()
    return CountRows.from_csr(rowptr.cuda(), at[:, 1].int().cuda(), x[at[:, 0], at[:, 1]].int().cuda(), k)


SHAPES = [(1, 1, 1), (1, 130, 8), (3, 127, 33), (16, 128, 64), (17, 129, 65), (130, 1000, 40), (257, 300, 128), (129, 2055, 200)]


@pytest.mark.parametrize("likelihood", ["multinomial", "dirichlet"])
@pytest.mark.parametrize("kind", ["csr", "dense16", "dense32"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradient(shape, dtype, kind, likelihood):
    from bayespy_amd import regression
    n, k, d = shape
    h, w, b, x, g = make(n, k, d, TYPES[dtype], sum(shape), density=0.2 if k > 1 else 1.0)
    want = oracle(h, w, b, x, g, likelihood, TYPES[dtype])
    rows = as_rows(x, kind).check()
    near(regression.log_loss(h, w, rows, bias=b, likelihood=likelihood), want["loss"], "loss alone")
    loss, dh, dw, db = regression.log_loss_gradient(h, w, rows, bias=b, likelihood=likelihood, row_weights=g)
    near(loss, want["loss"], "loss")
    near(db, want["db"], "dbias")
    near(dh, want["dh"], "dfeatures")
    near(dw, want["dw"], "dweights")


@pytest.mark.parametrize("likelihood", ["multinomial", "dirichlet"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 5, 3), (9, 700, 24), (200, 1031, 96)])
def test_labels(shape, dtype, likelihood):
    from bayespy_amd import regression
    n, k, d = shape
    h, w, _, _, _ = make(n, k, d, TYPES[dtype], 7)
    r = np.random.default_rng(3)
    y = torch.from_numpy(r.integers(0, k, size=n))
    y[0], y[-1] = k - 1, 0
    if n > 4:
        y[2] = -1
        y[3] = -100
    x = torch.zeros(n, k, dtype=torch.int32)
    has = (y >= 0).nonzero().squeeze(1)
    x[has, y[has]] = 1
    want = oracle(h, w, None, x, torch.ones(n), likelihood, TYPES[dtype])
    rows = regression.CountRows.from_labels(y.cuda(), k).check()
    near(regression.log_loss(h, w, rows, likelihood=likelihood), want["loss"], "loss alone")
    loss, dh, dw, db = regression.log_loss_gradient(h, w, rows, likelihood=likelihood)
    assert db is None
    near(loss, want["loss"], "loss")
    near(dh, want["dh"], "dfeatures")
    near(dw, want["dw"], "dweights")


# ---- the step ----------------------------------------------------------------------------------------------------
#
# One step in working precision v (2^-11 for fp16 operands, k 2^-24 for 32-bit products of k terms): S is off by 2 v |X|^2
# relative to its norm, S S and B by a few more, X' by (a + 4 |b| s^2 + 8 |c| s^4) v |X|_F with singular values s <= 1.2;
# later steps enlarge a difference by at most a = 3.4445 each, as p'(s) <= p'(0).  In Frobenius norm, relative to the
# largest |X| = sqrt(rank) * 1.2; then u of the result's type.

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def step_oracle(g, steps, coefficients=COEFFICIENTS):
    y = g.double().cpu()
    if y.dim() == 3:
        return torch.stack([step_oracle(v, steps, coefficients) for v in y])
    a, b, c = coefficients
    norm = torch.linalg.vector_norm(y)
    if norm == 0:
        return y
    y = y / norm
    for _ in range(steps):
        s = y @ y.t() if y.shape[0] <= y.shape[1] else y.t() @ y
        q = b * s + c * (s @ s)
        y = a * y + (q @ y if y.shape[0] <= y.shape[1] else y @ q)
    return y


def step_tolerance(want, dtype, steps, m, n):
    v = 2.0**-11 if dtype == torch.bfloat16 else max(m, n) * 2.0**-24
    one = 3.4445 + 4 * 4.775 * 1.44 + 8 * 2.0315 * 2.07
    norm = float(torch.linalg.vector_norm(want))
    return norm * (one * v * sum(3.4445**i for i in range(min(steps, 3))) + torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("steps", [1, 2, 5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 200), (33, 7), (64, 64), (130, 257), (500, 100), (3, 70, 129)])
def test_orthogonal_step(shape, dtype, steps):
    from bayespy_amd import regression
    r = np.random.default_rng(len(shape) + shape[-1])
    g = torch.from_numpy(r.standard_normal(shape) * 1e-3).to(TYPES[dtype]).cuda()
    got = regression.orthogonal_step(g, steps=steps)
    assert got.dtype == g.dtype and got.shape == g.shape and got.is_contiguous()
    want = step_oracle(g, steps)
    off = float(torch.linalg.vector_norm(got.double().cpu() - want))
    assert off <= step_tolerance(want, TYPES[dtype], steps, shape[-2], shape[-1])
