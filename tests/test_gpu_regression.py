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
special = pytest.importorskip("scipy.special")

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def f_of(z, x, likelihood):
    """lgamma(a + x) - lgamma(a) = lgamma(x) - log B(a, x): scipy takes the beta function where the difference cancels."""
    if likelihood == "multinomial":
        return torch.where(x > 0, x * z, torch.zeros_like(z))
    a, n = z.exp().numpy(), np.where(x.numpy() > 0, x.numpy(), 1.0)
    with np.errstate(invalid="ignore", divide="ignore"):
        f = torch.from_numpy(special.gammaln(n) - special.betaln(a, n))
    return torch.where(x > 0, f, torch.zeros_like(z))


def g_of(z, x, likelihood):
    """a (psi(a + x) - psi(a)); from a = e^20 on by psi's series, whose next term is below 1 / (12 a^2)."""
    if likelihood == "multinomial":
        return x
    a = z.exp()
    near = a * (torch.digamma(a + x) - torch.digamma(a))
    far = a * (torch.log1p(x / a) + x / (2 * a * (a + x)))
    return torch.where(x > 0, torch.where(z > 20, far, near), torch.zeros_like(z))


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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(256, 640), (640, 256), (193, 1000), (300, 129)])
def test_orthogonal_step_larger(shape, dtype):
    """Several tiles a side, split k, the padding of odd pitches; wide and tall."""
    from bayespy_amd import regression
    r = np.random.default_rng(5)
    g = torch.from_numpy(r.standard_normal(shape)).to(TYPES[dtype]).cuda()
    got, want = regression.orthogonal_step(g), step_oracle(g, 5)
    off = float(torch.linalg.vector_norm(got.double().cpu() - want))
    assert off <= step_tolerance(want, TYPES[dtype], 5, *shape)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(17000, 200), (200, 17001), (17000, 100), (99, 17003), (64, 300, 130), (64, 129, 300), (1500, 1400), (2600, 2500), (4100, 4200)])
def test_orthogonal_step_of_every_tile(shape, dtype):
    """Slabs and every tile side, with ragged ends; in 64 bits on the GPU.  The result is rounded to its type, which is off by at most
    eps / 2 of each value, so of every part of the matrix; the steps before may add as much again (bf16), or `one` times the 2^-21 that
    pairs of halves drop at each step, amplified (fp32, see step_tolerance)."""
    from bayespy_amd import regression
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.randn(shape, generator=gen, device="cuda").to(TYPES[dtype])
    got = regression.orthogonal_step(g).double()
    a, b, c = COEFFICIENTS
    y = g.double().reshape(-1, *shape[-2:])
    y = y / torch.linalg.vector_norm(y, dim=(1, 2), keepdim=True)
    tall = shape[-2] > shape[-1]
    for _ in range(5):
        t = y.transpose(1, 2).contiguous()
        s = t @ y if tall else y @ t
        q = b * s + c * (s @ s)
        y = a * y + (y @ q if tall else q @ y)
    one = 3.4445 + 4 * 4.775 * 1.44 + 8 * 2.0315 * 2.07
    u = torch.finfo(TYPES[dtype]).eps / 2
    tol = 2 * u if dtype == "bf16" else u + one * 2.0**-21 * (1 + 3.4445 + 3.4445**2)
    off = got.reshape(y.shape) - y
    for part in (np.s_[:], np.s_[:, -16:], np.s_[:, :, -16:], np.s_[:, :16], np.s_[:, :, :16], np.s_[-1:]):
        assert float(torch.linalg.vector_norm(off[part])) <= tol * float(torch.linalg.vector_norm(y[part])), part


def test_orthogonal_step_precision():
    """Rounded once from 64 bits bf16 is off by 2^-8 / sqrt(3) / 1.4 of the norm (a uniform rounding error, values spread over a
    power of two); the products in fp16 may add as much again.  fp32: no further off than the same steps in 32-bit arithmetic are, which is
    what weak directions beside strong ones make of roundings of 2^-24 (1.7e-6 of the norm here)."""
    from bayespy_amd import regression
    r = np.random.default_rng(8)
    left, right = r.standard_normal((2000, 16)) * np.arange(1, 17) ** -1.0, r.standard_normal((16, 130))
    g = torch.from_numpy(left @ right + 0.1 * r.standard_normal((2000, 130))).float().cuda()
    want = step_oracle(g, 5)
    off = torch.linalg.vector_norm(regression.orthogonal_step(g).double().cpu() - want) / torch.linalg.vector_norm(want)
    a, b, c = COEFFICIENTS
    y = g.cpu() / torch.linalg.vector_norm(g.cpu().double()).float()
    for _ in range(5):
        t = y.t() @ y
        y = a * y + y @ (b * t + c * (t @ t))
    assert float(off) <= float(torch.linalg.vector_norm(y.double() - want) / torch.linalg.vector_norm(want))
    h = g.bfloat16()
    want = step_oracle(h, 5)
    off = torch.linalg.vector_norm(regression.orthogonal_step(h).double().cpu() - want) / torch.linalg.vector_norm(want)
    assert float(off) < 2 * 2.0**-8 / 3**0.5 / 1.4


def test_orthogonal_step_strides_zero_and_scale():
    from bayespy_amd import regression
    r = np.random.default_rng(2)
    whole = torch.from_numpy(r.standard_normal((6, 90, 200))).float().cuda()
    for view in (whole[:, 3:70, 5:140], whole[:, 3:70, 5:140].transpose(1, 2), whole[::2, ::3, ::2], whole[1:2].expand(3, 90, 200),
                 whole[0].t(), whole[0, :33, ::3], whole[0, ::3, :33].t()):
        want = step_oracle(view, 5)
        off = float(torch.linalg.vector_norm(regression.orthogonal_step(view).double().cpu() - want))
        assert off <= step_tolerance(want, torch.float32, 5, view.shape[-2], view.shape[-1])
    for dtype in (torch.float32, torch.bfloat16):
        zero = torch.zeros(70, 130, dtype=dtype, device="cuda")
        assert not bool(regression.orthogonal_step(zero).any())
        # |G| beyond the range of its squares, powers of two: the same result to the bit
        g = whole[0].to(dtype)
        one = regression.orthogonal_step(g)
        for scale in (2.0**100, 2.0**-100):
            assert torch.equal(regression.orthogonal_step(g * scale), one)
        pair = torch.stack([g, zero[:1, :1].expand_as(g)])
        got = regression.orthogonal_step(pair)
        assert torch.equal(got[0], one) and not bool(got[1].any())
        g = g.clone()
        g[3, 4] = float("nan")
        assert bool(torch.isnan(regression.orthogonal_step(g)).all())
    assert regression.orthogonal_step(torch.zeros(0, 5, 7, device="cuda")).shape == (0, 5, 7)
    narrow = regression.orthogonal_step(whole[0], steps=3, coefficients=(1.5, -0.5, 0.0))  # the cubic iteration
    want = step_oracle(whole[0], 3, (1.5, -0.5, 0.0))
    assert float(torch.linalg.vector_norm(narrow.double().cpu() - want)) <= step_tolerance(want, torch.float32, 3, 90, 200)


# ---- masks, empty rows, formats ----------------------------------------------------------------------------------

def test_columns_taken_out():
    """bias = -inf: probability 0, no gradient, whatever the weights hold; a count there costs +inf."""
    from bayespy_amd import regression
    for n, k, d in ((5, 300, 24), (40, 300, 24)):
        h, w, b, x, g = make(n, k, d, torch.float32, 11)
        out = torch.zeros(k, dtype=torch.bool)
        out[[0, 7, 129, 255, 299]] = True
        x[:, out] = 0
        keep = ~out
        b = b.clone()
        b[out.cuda()] = -float("inf")
        for likelihood in ("multinomial", "dirichlet"):
            want = oracle(h, w[keep.cuda()], b[keep.cuda()], x[:, keep], g, likelihood, torch.float32)
            for kind in ("csr", "dense32"):
                loss, dh, dw, db = regression.log_loss_gradient(h, w, as_rows(x, kind), bias=b, likelihood=likelihood, row_weights=g)
                near(loss, want["loss"], "loss")
                near(dh, want["dh"], "dfeatures")
                near(dw[keep.cuda()], want["dw"], "dweights")
                near(db[keep.cuda()], want["db"], "dbias")
                assert not bool(dw[out.cuda()].any()) and not bool(db[out.cuda()].any())
                broken = w.clone()
                broken[7], broken[299] = float("nan"), float("inf")
                near(regression.log_loss(h, broken, as_rows(x, kind), bias=b, likelihood=likelihood), want["loss"], "NaN in weights that are out")
        y = x.clone()
        y[1, 7] = 2
        for kind in ("csr", "dense32"):
            loss = regression.log_loss(h, w, as_rows(y, kind), bias=b)
            assert loss[1] == float("inf") and bool(torch.isfinite(loss[[0, 2, 3, 4]]).all())


@pytest.mark.parametrize("n", [3, 70])
def test_masks_of_the_lowest_value(n):
    """All columns at the type's lowest value are all alike: the loss is T log K; one spared column takes everything."""
    from bayespy_amd import regression
    k, d = 500, 16
    h, w, _, x, _ = make(n, k, d, torch.bfloat16, 3)
    low = torch.full((k,), torch.finfo(torch.float32).min, device="cuda")
    y = torch.arange(n, device="cuda") % k
    loss = regression.log_loss(h, w, regression.CountRows.from_labels(y, k), bias=low)
    assert bool(((loss - np.log(k)).abs() <= 2.0**-20).all())  # log, exp and one rounding of a value near 6
    for kind in ("csr", "dense32"):  # every likelihood and form of rows; the gradient's p is 1 / K
        one = torch.zeros(n, k, dtype=torch.int32)
        one[torch.arange(n), y.cpu()] = 1
        for likelihood in ("multinomial", "dirichlet"):
            loss, _, _, db = regression.log_loss_gradient(h, w, as_rows(one, kind), bias=low, likelihood=likelihood)
            assert bool(((loss - np.log(k)).abs() <= 2.0**-20).all())
            assert bool(((db.cpu() - (n / k - one.sum(0))).abs() <= n * 2.0**-22).all())
    low[9] = 0.0
    y[:] = 9
    loss = regression.log_loss(h, w, regression.CountRows.from_labels(y, k), bias=low)
    # l = z_9, which is summed twice in two orders: once among the row's columns, once for the label; each is off by d 2^-24 sum |h w| at most
    assert bool((loss.abs() <= 2 * d * 2.0**-24 * float((h.double().abs() @ w[9].double().abs()).max())).all())


def test_rows_without_counts_and_no_rows():
    from bayespy_amd import regression
    k, d = 200, 40
    for n in (4, 50):
        h, w, b, x, g = make(n, k, d, torch.float32, 1)
        x[:] = 0
        labels = torch.full((n,), -1, device="cuda")
        for rows in (as_rows(x, "csr"), as_rows(x, "dense16"), regression.CountRows.from_labels(labels, k)):
            h2 = h.clone()
            loss, dh, dw, db = regression.log_loss_gradient(h2, w, rows, bias=b, row_weights=g, likelihood="dirichlet")
            for t in (loss, dh, dw, db):
                assert not bool(t.any())
    for dtype in (torch.float32, torch.bfloat16):
        for rows in (regression.CountRows.from_labels(torch.zeros(0, dtype=torch.int64, device="cuda"), 7),
                     regression.CountRows.from_dense(torch.zeros(0, 7, dtype=torch.int32, device="cuda")),
                     regression.CountRows.from_csr(torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"),
                                                   torch.zeros(0, dtype=torch.int32, device="cuda"), 7)):
            h, w = torch.zeros(0, 3, dtype=dtype, device="cuda"), torch.ones(7, 3, dtype=dtype, device="cuda")
            loss, dh, dw, db = regression.log_loss_gradient(h, w, rows.check(), bias=torch.zeros(7, device="cuda"))
            assert loss.shape == (0,) and dh.shape == (0, 3) and not bool(dw.any()) and not bool(db.any())
            assert regression.log_loss(h, w, rows).shape == (0,)


def test_rows_that_break_their_format():
    """check() names it; the loss of such a row is NaN, other rows keep theirs, and nothing out of range is followed."""
    from bayespy_amd import regression
    k, d = 300, 8
    for n in (6, 40):
        h, w, b, x, _ = make(n, k, d, torch.float32, 4)
        x[n // 2, 5] = 1
        good = as_rows(x, "csr")
        want = regression.log_loss(h, w, good, bias=b, likelihood="dirichlet")
        rowptr, col, val = good._tensors
        first = int(rowptr[1])
        breaks = {"ascend strictly": lambda p, c, v: c.__setitem__(first + 1, int(c[first])), "out of range": lambda p, c, v: c.__setitem__(first, k),
                  "column is out": lambda p, c, v: c.__setitem__(first, -3), "negative": lambda p, c, v: v.__setitem__(first, -1)}
        for text, change in breaks.items():
            p, c, v = rowptr.clone(), col.clone(), val.clone()
            change(p, c, v)
            rows = regression.CountRows.from_csr(p, c, v, k)
            with pytest.raises(ValueError):
                rows.check()
            loss = regression.log_loss(h, w, rows, bias=b, likelihood="dirichlet")
            other = [i for i in range(n) if i != 1]
            assert bool(torch.isnan(loss[1])) and torch.equal(loss[other], want[other])
            loss, dh, dw, db = regression.log_loss_gradient(h, w, rows, bias=b, likelihood="dirichlet")
            assert bool(torch.isnan(dh[1]).all()) and bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all()) and bool(torch.isfinite(dh[other]).all())
        for i, value in ((1, 1 << 40), (1, -5), (2, 0)):
            p = rowptr.clone()
            p[i] = value
            rows = regression.CountRows.from_csr(p, col, val, k)
            with pytest.raises(ValueError, match="rowptr"):
                rows.check()
            assert bool(torch.isnan(regression.log_loss(h, w, rows, bias=b)[i - 1 if value != 0 else 1]))
        y = torch.zeros(n, dtype=torch.int64, device="cuda")
        y[1], y[2] = k, 1 << 50
        rows = regression.CountRows.from_labels(y, k)
        with pytest.raises(ValueError, match="below K"):
            rows.check()
        loss = regression.log_loss_gradient(h, w, rows, bias=b)[0]
        assert torch.isnan(loss).tolist() == [i in (1, 2) for i in range(n)]
        z = x.clone()
        z[1, 3] = -1
        rows = as_rows(z, "dense32")
        with pytest.raises(ValueError, match="negative"):
            rows.check()
        assert torch.isnan(regression.log_loss(h, w, rows, bias=b)).tolist() == [i == 1 for i in range(n)]


@pytest.mark.parametrize("likelihood", ["multinomial", "dirichlet"])
@pytest.mark.parametrize("kind", ["csr", "dense32"])
def test_large_counts_and_far_values(kind, likelihood):
    """Counts to 2^30, z from -80 to 80: where 32-bit lgamma and exp would leave their range."""
    from bayespy_amd import regression
    n, k, d = 20, 150, 16
    h, w, b, x, g = make(n, k, d, torch.float32, 21)
    r = np.random.default_rng(0)
    b = torch.from_numpy(r.uniform(-80, 80, size=k)).float().cuda()
    b[:20] = torch.linspace(-8, 8, 20)
    big = torch.from_numpy(np.floor(2.0 ** r.uniform(0, 30, size=(n, k))).astype(np.int32))
    x = torch.where(torch.from_numpy(r.random((n, k)) < 0.1), big, x)
    x[:3] = 0
    x[0, 4], x[1, 120], x[2, 10] = 17, 16, 1 << 30
    want = oracle(h, w, b, x, g, likelihood, torch.float32)
    loss, dh, dw, db = regression.log_loss_gradient(h, w, as_rows(x, kind), bias=b, likelihood=likelihood, row_weights=g)
    near(loss, want["loss"], "loss")
    near(dh, want["dh"], "dfeatures")
    near(dw, want["dw"], "dweights")
    near(db, want["db"], "dbias")


# ---- layout --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [7, 90])
def test_pitches_and_alignment(n, dtype):
    from bayespy_amd import regression
    k, d = 333, 56
    h, w, b, x, g = make(n, k, d, TYPES[dtype], 9)
    plain = regression.log_loss_gradient(h, w, as_rows(x, "dense16"), bias=b, row_weights=g)
    for shift in (1, 2, 8):
        big_h = torch.full((n, d + 19), float("nan"), dtype=h.dtype, device="cuda")
        big_w = torch.full((k, d + 24), float("nan"), dtype=h.dtype, device="cuda")
        big_x = torch.full((n, k + 13), 9, dtype=torch.int32, device="cuda").to(torch.uint16)
        hh, ww, xx = big_h[:, shift:shift + d], big_w[:, shift:shift + d], big_x[:, shift:shift + k]
        hh.copy_(h), ww.copy_(w), xx.copy_(x.to(torch.uint16))
        bb = torch.empty(k + 1, device="cuda")[1:]
        bb.copy_(b)
        got = regression.log_loss_gradient(hh, ww, regression.CountRows.from_dense(xx), bias=bb, row_weights=g)
        for a, c in zip(plain, got):  # the same sums in the same order, whatever the layout
            assert torch.equal(a, c)


@pytest.mark.parametrize("d", [2500, 5000])
def test_few_rows_of_many_features(d):
    """Rows too long for LDS take tiles."""
    from bayespy_amd import regression
    for dtype in ("bf16", "f32"):
        h, w, b, x, g = make(3, 200, d, TYPES[dtype], 2)
        want = oracle(h, w, b, x, g, "multinomial", TYPES[dtype])
        near(regression.log_loss(h, w, as_rows(x, "csr"), bias=b), want["loss"], "loss")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_tiles(dtype):
    """Enough work for tiles of 256, with ragged ends and a pitch."""
    from bayespy_amd import regression
    n, k, d = 4100, 6001, 72
    h, w, b, x, g = make(n, k, d, TYPES[dtype], 12, density=0.003)
    want = oracle(h, w, b, x, g, "multinomial", TYPES[dtype])
    wide = torch.zeros(k, d + 8, dtype=TYPES[dtype], device="cuda")
    wide[:, :d] = w
    loss, dh, dw, db = regression.log_loss_gradient(h, wide[:, :d], as_rows(x, "csr"), bias=b, row_weights=g)
    near(loss, want["loss"], "loss")
    near(dh, want["dh"], "dfeatures")
    near(dw, want["dw"], "dweights")
    near(db, want["db"], "dbias")


def test_more_rows_than_a_block():
    from bayespy_amd import regression
    n, k, d = 16384 + 37, 140, 8
    h, w, b, x, g = make(n, k, d, torch.float32, 6, density=0.05)
    want = oracle(h, w, b, x, g, "dirichlet", torch.float32)
    for kind in ("csr", "dense16"):
        loss, dh, dw, db = regression.log_loss_gradient(h, w, as_rows(x, kind), bias=b, likelihood="dirichlet", row_weights=g)
        near(loss, want["loss"], "loss")
        near(dh, want["dh"], "dfeatures")
        near(dw, want["dw"], "dweights")
        near(db, want["db"], "dbias")


def test_more_rows_than_a_block_of_losses():
    from bayespy_amd import regression
    n, k, d = 65536 + 37, 20, 4
    h, w, b, x, g = make(n, k, d, torch.float32, 8)
    want = oracle(h, w, b, x, g, "dirichlet", torch.float32)
    for kind in ("csr", "dense16"):
        near(regression.log_loss(h, w, as_rows(x, kind), bias=b, likelihood="dirichlet"), want["loss"], "loss")


def test_dense_counts_of_every_size():
    """Lists that fill up, counts at the borders of their forms (1, 2, 15 to 17, 30 to 32), z far out to both sides."""
    from bayespy_amd import regression
    r = np.random.default_rng(2)
    for n, k, d in ((9, 300, 8), (140, 517, 16)):
        h, w, b, _, g = make(n, k, d, torch.float32, 3)
        b = torch.from_numpy(r.choice([-30.0, -3.0, 0.0, 3.0, 25.0], size=k)).float().cuda()
        x = torch.from_numpy(r.choice([1, 2, 3, 15, 16, 17, 30, 31, 32, 100000], size=(n, k)).astype(np.int32))
        x[1] = 17   # a row for the 64-bit functions alone
        x[2] = 16
        x[3] = 0
        want = oracle(h, w, b, x, g, "dirichlet", torch.float32)
        for kind in ("dense32", "csr"):
            loss, dh, dw, db = regression.log_loss_gradient(h, w, as_rows(x, kind), bias=b, likelihood="dirichlet", row_weights=g)
            near(loss, want["loss"], "loss")
            near(dh, want["dh"], "dfeatures")
            near(dw, want["dw"], "dweights")
            near(db, want["db"], "dbias")


def test_more_columns_than_a_piece():
    """d loss / d z of 1500 x 60000 in fp32 is 360 MB: two pieces."""
    from bayespy_amd import regression
    n, k, d = 1500, 60000, 8
    h, w, b, _, g = make(n, 16, d, torch.float32, 6)
    r = np.random.default_rng(1)
    w = torch.from_numpy(r.standard_normal((k, d)) * 0.2).float().cuda()
    b = torch.from_numpy(r.standard_normal(k)).float().cuda()
    y = torch.from_numpy(r.integers(0, k, size=n))
    x = torch.zeros(n, k, dtype=torch.int32)
    x[torch.arange(n), y] = 1
    want = oracle(h, w, b, x, g, "multinomial", torch.float32)
    loss, dh, dw, db = regression.log_loss_gradient(h, w, regression.CountRows.from_labels(y.cuda(), k), bias=b, row_weights=g)
    near(loss, want["loss"], "loss")
    near(dh, want["dh"], "dfeatures")
    near(dw, want["dw"], "dweights")
    near(db, want["db"], "dbias")


@pytest.mark.parametrize("n", [2, 130])
def test_weights_beyond_32_bit_offsets(n):
    """2^31 + values: zero but for the last columns."""
    from bayespy_amd import regression
    d = 1024
    k = (1 << 31) // d + 1000
    w = torch.zeros(k, d, dtype=torch.bfloat16, device="cuda")
    w[-3:] = 0.125
    h = torch.ones(n, d, dtype=torch.bfloat16, device="cuda") * 0.0625
    y = torch.full((n,), k - 2, device="cuda")
    loss, dh, dw, _ = regression.log_loss_gradient(h, w, regression.CountRows.from_labels(y, k))
    z = 0.125 * 0.0625 * d
    mass = (k - 3) + 3 * np.exp(z)
    # l and z in 32 bits: a few roundings of 2^-24 of values up to 15
    assert bool(((loss - (np.log(mass) - z)).abs() <= 2.0**-19).all())
    u = 2.0**-8
    p = np.exp(z) / mass
    assert float((dw[-2].double() - n * (p - 1) * 0.0625).abs().max()) <= 3 * u * n * 0.0625
    assert float((dw[-1].double() - n * p * 0.0625).abs().max()) <= 3 * u * n * p * 0.0625
    assert float((dw[0].double() - n / mass * 0.0625).abs().max()) <= 3 * u * n / mass * 0.0625
    assert float((dh.double() - 0.125 * (3 * p - 1)).abs().max()) <= 3 * u * 0.125 * (1 + 3 * p)


def test_more_tiles_than_a_launch_takes():
    """16384 rows of 2^25 columns: tiles of 256 with a thread for 128 values each would be 2^32 threads."""
    from bayespy_amd import regression
    n, k, d = 16384, 1 << 25, 8
    w = torch.zeros(k, d, dtype=torch.bfloat16, device="cuda")
    w[-3:] = 0.5
    h = torch.zeros(n, d, dtype=torch.bfloat16, device="cuda")
    z = torch.tensor([0.0, 4.0, 8.0, 16.0], dtype=torch.float64)
    h[:] = (z[torch.arange(n) % 4, None] / (0.5 * d)).to(torch.bfloat16).cuda()  # exact
    y = torch.full((n,), k - 1, device="cuda")
    loss = regression.log_loss(h, w, regression.CountRows.from_labels(y, k))
    want = (torch.log((k - 3) + 3 * z.exp()) - z)[torch.arange(n) % 4]
    # l - m in 64 bits from pieces that hold at most 2^14 ones each, and one rounding of a value up to 18
    assert bool(((loss.cpu().double() - want).abs() <= 2.0**-19).all())


def test_a_weight_at_the_end_of_its_range():
    """weight * count leaves 32 bits in one row: its column is lost, columns without it are not."""
    from bayespy_amd import regression
    n, k, d = 40, 600, 16
    h, w, b, x, _ = make(n, k, d, torch.float32, 4)
    g = torch.ones(n, device="cuda")
    b[:] = 0.0
    b[300:] = -200.0  # p = 0 in 32 bits there
    x[:, 300:] = 0
    x[1:, 400] = 3000000
    x[0, :] = 0
    x[0, 5] = 2
    g[0] = 3e38
    for likelihood in ("multinomial", "dirichlet"):
        _, _, _, db = regression.log_loss_gradient(h, w, as_rows(x, "csr"), bias=b, likelihood=likelihood, row_weights=g)
        want = oracle(h[1:], w, b, x[1:], g[1:], likelihood, torch.float32)["db"]
        near(db[300:], (want[0][300:], want[1][300:]), "dbias of columns that the row has not")


# ---- how they are run ------------------------------------------------------------------------------------------------

def _call_all(h, w, b, x, g, kind, likelihood):
    from bayespy_amd import regression
    loss, dh, dw, db = regression.log_loss_gradient(h, w, as_rows(x, kind), bias=b, likelihood=likelihood, row_weights=g)
    return [regression.log_loss(h, w, as_rows(x, kind), bias=b, likelihood=likelihood), loss, dh, dw, db, regression.orthogonal_step(dw)]


@pytest.mark.parametrize("kind", ["csr", "dense32"])
def test_same_bits_every_time_and_on_any_stream(kind):
    h, w, b, x, g = make(300, 700, 72, torch.bfloat16, 13)
    want = _call_all(h, w, b, x, g, kind, "dirichlet")
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in side * 3:  # calls that overlap
        with torch.cuda.stream(s):
            got.append(_call_all(h, w, b, x, g, kind, "dirichlet"))
    torch.cuda.synchronize()
    for one in got:
        for a, c in zip(want, one):
            assert torch.equal(a, c)


def test_captured_and_replayed():
    """Two graphs, replayed in turn with eager calls between: each replay gives the eager bits for the inputs of the time."""
    from bayespy_amd import regression
    cases = []
    for n, k, d in ((200, 500, 64), (6, 900, 32)):
        h, w, b, x, g = make(n, k, d, torch.float32, n)
        rows = as_rows(x, "csr")
        run = lambda h=h, w=w, b=b, rows=rows, g=g: (lambda r: list(r) + [regression.orthogonal_step(r[2])])(  # noqa: E731
            regression.log_loss_gradient(h, w, rows, bias=b, likelihood="dirichlet", row_weights=g))
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        cases.append((graph, out, run, h))
    for turn in range(4):
        for graph, out, run, h in cases:
            h.mul_(1.125)
            graph.replay()
            kept = [t.clone() for t in out]
            want = run()
            torch.cuda.synchronize()
            for a, c in zip(want, kept):
                assert torch.equal(a, c)


def test_gradient_against_differences():
    """Central differences of the loss in 64 bits (its definition, which the tests above hold the kernels to) against the kernels' fp32
    gradient: step e = 1e-4, truncation e^2 / 6 of the third derivative (below 1e-6 here) and fp32's 2^-24 of sums near 100."""
    from bayespy_amd import regression
    n, k, d = 12, 60, 5
    h, w, b, x, g = make(n, k, d, torch.float32, 17)
    for likelihood in ("multinomial", "dirichlet"):
        _, dh, dw, db = regression.log_loss_gradient(h, w, as_rows(x, "csr"), bias=b, likelihood=likelihood, row_weights=g)

        def total(h, w, b):
            return float((oracle(h, w, b, x, torch.ones(n), likelihood, torch.float32)["loss"][0] * g.double().cpu()).sum())
        at = [h.double().cpu(), w.double().cpu(), b.double().cpu()]
        for i, (grad, where) in enumerate(((dh, (2, 3)), (dw, (10, 1)), (dw, (59, 4)), (db, (0,)), (db, (33,)))):
            which = 0 if grad is dh else 1 if grad is dw else 2
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in at]
                moved[which][where] += sign * 1e-4
                ends.append(total(*moved))
            assert abs((ends[0] - ends[1]) / 2e-4 - float(grad[where])) < 1e-4


def test_bias_alone_is_the_prior_s_likelihood():
    """weights = 0, bias = log(alphas): the loss summed over rows is the total loss that the estimator minimises."""
    from bayespy_amd import dirichletMultinomialEstimation as DME
    from bayespy_amd import regression
    r = np.random.default_rng(4)
    k = 30
    x = r.poisson(1.5, size=(400, k)).astype(np.int32)
    data = DME.CompressedRowData(k)
    data.appendMatrix(x)
    priors = DME.findDirichletPriors(data, [1.0] * k, 50)
    want = DME.getTotalLoss(priors, data)
    h, w = torch.ones(400, 8, device="cuda"), torch.zeros(k, 8, device="cuda")
    b = torch.log(torch.tensor(priors, dtype=torch.float64)).float().cuda()
    rows = regression.CountRows.from_dense(torch.from_numpy(x).cuda())
    loss, _, _, db = regression.log_loss_gradient(h, w, rows, bias=b, likelihood="dirichlet")
    # each alpha is off by the 2^-24 |log alpha| of its bias's rounding, a loss by 2^-20 of its terms
    assert abs(float(loss.double().sum()) - want) <= 2.0**-20 * abs(want)
    # at the maximum the gradient vanishes: what is left is the solver's stop (|g|^2 < 2^-10, here times alpha) and the sums' rounding
    assert float(db.abs().max()) <= 2.0**-5 * max(priors) + 2.0**-20 * float(x.sum())


def test_a_run_of_them():
    """A few steps of a decoder as a user takes them: loss, gradient, orthogonalised step, weights; every step against the same in 64 bits."""
    from bayespy_amd import regression
    n, k, d = 200, 400, 32
    h, w, b, x, g = make(n, k, d, torch.float32, 30)
    rows = as_rows(x, "csr").check()
    for _ in range(3):
        want = oracle(h, w, b, x, g, "dirichlet", torch.float32)
        loss, dh, dw, db = regression.log_loss_gradient(h, w, rows, bias=b, likelihood="dirichlet", row_weights=g)
        near(loss, want["loss"], "loss")
        near(dw, want["dw"], "dweights")
        step = regression.orthogonal_step(dw)
        exact = step_oracle(dw, 5)
        assert float(torch.linalg.vector_norm(step.double().cpu() - exact)) <= step_tolerance(exact, torch.float32, 5, k, d)
        w = w - 0.02 * step
        b = b - 1e-4 * db


def test_refusals():
    from bayespy_amd import regression as R
    h, w = torch.zeros(4, 8, device="cuda"), torch.zeros(9, 8, device="cuda")
    rows = R.CountRows.from_labels(torch.zeros(4, dtype=torch.int64, device="cuda"), 9)
    for bad in (lambda: R.log_loss(h.half(), w.half(), rows), lambda: R.log_loss(h, w.bfloat16(), rows), lambda: R.log_loss(h[:3], w, rows),
                lambda: R.log_loss(h, w[:8], rows), lambda: R.log_loss(h[:, :7], w, rows), lambda: R.log_loss(h, w, rows, likelihood="poisson"),
                lambda: R.log_loss(h, w, "rows"), lambda: R.log_loss(h, w, rows, bias=torch.zeros(8, device="cuda")),
                lambda: R.log_loss(h, w, rows, bias=torch.zeros(9)), lambda: R.log_loss(h.cpu(), w, rows), lambda: R.log_loss(h[:1].expand(4, 8), w, rows),
                lambda: R.log_loss(torch.zeros(8, 4, device="cuda").t(), w, rows), lambda: R.log_loss_gradient(h, w, rows, row_weights=torch.zeros(3, device="cuda")),
                lambda: R.log_loss_gradient(h, w, rows, row_weights=torch.zeros(4, dtype=torch.float64, device="cuda")),
                lambda: R.CountRows.from_dense(torch.zeros(4, 9, device="cuda")), lambda: R.CountRows.from_dense(torch.zeros(9, 4, dtype=torch.int32, device="cuda").t()),
                lambda: R.orthogonal_step(h.half()), lambda: R.orthogonal_step(h[0]), lambda: R.orthogonal_step(h, steps=0), lambda: R.orthogonal_step(h[:0]),
                lambda: R.orthogonal_step(h, coefficients=(9.0, 0.0, 0.0)), lambda: R.orthogonal_step(h, coefficients=(float("nan"), 0.0, 0.0))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        R.orthogonal_step(h.cpu())
