"""Log losses of count rows and their gradient where values are far apart: masks of any size, against the definition in 64 bits.

The inputs are whole numbers and quarters, few of them, so that every product and every 32-bit sum of them is exact and z is z = fp32(dot + bias)
whatever the order: what is left to be off by are the functions of z.  With d = z - m (m the row's largest z)

    e^d: 2^-22 (|d| + 4) of it (the exponent's rounding, exp2's last bits; below 2^-126 it may be 0);  s = sum e^d: 2^-18 of it besides
    (at most 64 additions of 2^-24 in a lane's sum)
    loss:  2^-22 times the sum of its terms' sizes, 2^-18 T for log s, one rounding at the end
    d loss / d z = p G(l, T) - G(z, x):  e = 2^-18 + 2^-22 (|d| + 4) of the first, 2^-22 of the second, then the operands' rounding."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def rest_of(z, x):
    """R(z, x) = sum_{1 <= n < x} log(e^z + n), 64 bits, any z."""
    r = torch.zeros_like(z)
    for n in range(1, int(x.max()) if x.numel() else 0):
        term = torch.where(z > 0, z + torch.log1p(n * torch.exp(-z.clamp(min=0))), torch.log(torch.exp(z.clamp(max=0)) + n))
        r += torch.where(x > n, term, torch.zeros_like(z))
    return r


def g_of(z, x):
    """G(z, x) = sum_{n < x} e^z / (e^z + n), 64 bits, any z."""
    g = (x > 0).to(z.dtype)
    for n in range(1, int(x.max()) if x.numel() else 0):
        g += torch.where(x > n, 1.0 / (1.0 + n * torch.exp(-z)), torch.zeros_like(z))
    return g


def exact(h, w, b, x, weight, likelihood, dtype):
    """Loss and gradient and what they may be off by (see above); on the device of h."""
    h, w, x, weight = h.double(), w.double(), x.double(), weight.double()
    z = ((h @ w.t()) + b.double()).float().double()
    m = z.max(dim=1, keepdim=True).values
    d = z - m
    at = (x > 0).nonzero(as_tuple=True)
    ze, xe, de = z[at], x[at], d[at]
    total = x.sum(dim=1)
    p = torch.exp(d)
    s = p.sum(dim=1)
    p = p / s[:, None]
    over = torch.log(s)
    mass = torch.zeros_like(total)

    def rows(v):
        return mass.index_add(0, at[0], v)
    if likelihood == "multinomial":
        loss = total * over + rows(-xe * de)
        size = total * over + rows(xe * de.abs())
        ge, gl = xe, total
    else:
        j, l = rows(torch.ones_like(xe)), m.squeeze(1) + over
        re, rl = rest_of(ze, xe), rest_of(l, total)
        loss = over + rl - rows(de + re) + (1 - j) * m.squeeze(1)
        size = over + rl.abs() + rows(de.abs() + re.abs()) + ((1 - j) * m.squeeze(1)).abs()
        ge, gl = g_of(ze, xe), g_of(l, total)
    loss = torch.where(total > 0, loss, mass)
    tol_loss = 2.0**-22 * size + 2.0**-18 * total + 2.0**-24 * loss.abs()
    loss = loss.float().double()  # two counts at a mask of the type's lowest value: beyond 32 bits, which is inf
    have = (total > 0).double()[:, None]
    first = p * gl[:, None] * have
    dz = first.clone()
    dz[at] -= ge
    e = 2.0**-18 + 2.0**-22 * (d.abs().clamp(max=104.0) + 4)
    tol = e * first + 2.0**-120
    tol[at] += 2.0**-22 * ge
    dz, tol = dz * weight[:, None], tol * weight.abs()[:, None]
    u = torch.finfo(dtype).eps / 2
    off = tol + u * dz.abs()
    n, k = x.shape
    out = {"loss": (loss, tol_loss), "dbias": (dz.sum(dim=0), tol.sum(dim=0) + n * 2.0**-23 * dz.abs().sum(dim=0))}
    for name, value, t in (("dfeatures", dz @ w, off @ w.abs() + k * 2.0**-23 * (dz.abs() @ w.abs())),
                           ("dweights", dz.t() @ h, off.t() @ h.abs() + n * 2.0**-23 * (dz.abs().t() @ h.abs()))):
        out[name] = (value, t * (1 + u) + u * value.abs())
    return out


def near(got, want, name):
    value, tol = want
    assert got.shape == value.shape, name
    off = torch.where(got.double() == value, 0.0, (got.double() - value).abs())
    bad = ~(off <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g of its tolerance" % (
        name, int(bad.sum()), off.numel(), float((off / tol).nan_to_num(nan=float("inf")).max()))


def rows_of(x, kind, labels=None):
    from bayespy_amd.regression import CountRows
    if kind == "labels":
        return CountRows.from_labels(labels, x.shape[1])
    if kind == "dense":
        return CountRows.from_dense(x.int().contiguous())
    rowptr = torch.zeros(x.shape[0] + 1, dtype=torch.int64, device=x.device)
    rowptr[1:] = (x > 0).sum(1).cumsum(0)
    at = (x > 0).nonzero()
    return CountRows.from_csr(rowptr, at[:, 1].int().contiguous(), x[at[:, 0], at[:, 1]].int().contiguous(), x.shape[1])


def all_of_it(h, w, b, x, weight, kind, likelihood, dtype, labels=None):
    from bayespy_amd import regression
    want = exact(h, w, b, x, weight, likelihood, dtype)
    rows = rows_of(x, kind, labels)
    near(regression.log_loss(h, w, rows, bias=b, likelihood=likelihood), want["loss"], "loss alone")
    got = regression.log_loss_gradient(h, w, rows, bias=b, likelihood=likelihood, row_weights=weight)
    for value, name in zip(got, ("loss", "dfeatures", "dweights", "dbias")):
        near(value, want[name], name)


def whole_numbers(n, k, d, dtype, seed):
    r = np.random.default_rng(seed)
    h = torch.from_numpy(r.integers(-1, 2, size=(n, d))).to(dtype).cuda()
    w = torch.from_numpy(r.integers(-1, 2, size=(k, d))).to(dtype).cuda()
    b = torch.from_numpy(r.integers(-8, 9, size=k) / 4).float().cuda()
    x = np.zeros((n, k), dtype=np.int32)
    for i in range(n):
        x[i, r.choice(k, size=min(k, 12), replace=False)] = r.choice([1, 1, 2, 3, 7, 17], size=min(k, 12))
    x[n // 2] = 0  # a row without counts
    weight = torch.from_numpy(r.integers(1, 9, size=n) / 8).float().cuda()
    return h, w, b, torch.from_numpy(x).cuda(), weight


# every tile side in both types: 16 x 128 and single loads, 64, 128 and 256
SHAPES = [(3, 900, 8), (17, 900, 8), (70, 900, 8), (1000, 6001, 8), (2000, 6001, 8), (4100, 6001, 8)]
MASKS = [1e7, -1e7, -1e9, -1e10, -1e20, -1e30, 1e10]


@pytest.mark.parametrize("kind", ["labels", "csr", "dense"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_runs_of_masked_columns(shape, dtype, kind):
    """A run of more than two tiles' columns and the ragged end at one far value: tiles without an ordinary column.  Counts lie inside and
    outside of it."""
    n, k, d = shape
    h, w, b, x, weight = whole_numbers(n, k, d, TYPES[dtype], n)
    labels = None
    if kind == "labels":
        labels = torch.from_numpy(np.random.default_rng(1).integers(-1, k, size=n)).cuda()
        labels[0], labels[-1] = k - 1, 300
        x = torch.zeros_like(x)
        x[torch.arange(n, device="cuda")[labels >= 0], labels[labels >= 0]] = 1
    for mask in MASKS:
        far = b.clone()
        far[256:min(k - 140, 1300)] = mask
        far[k - 130:] = mask
        for likelihood in ("multinomial", "dirichlet"):
            all_of_it(h, w, far, x, weight, kind, likelihood, TYPES[dtype], labels)


@pytest.mark.parametrize("kind", ["csr", "dense"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_all_columns_far_out(shape, dtype, kind):
    """The row's own largest z is far out: only what lies above it counts."""
    n, k, d = shape
    h, w, b, x, weight = whole_numbers(n, k, d, TYPES[dtype], n + 1)
    for mask in MASKS:
        for likelihood in ("multinomial", "dirichlet"):
            all_of_it(h, w, torch.full_like(b, mask), x, weight, kind, likelihood, TYPES[dtype])


@pytest.mark.parametrize("n", [5, 40, 600])
def test_two_masks_beside_each_other(n):
    """Masks of several sizes and -inf in turn, so that a tile's largest z is now an ordinary one, now one mask or the other."""
    k, d = 2100, 8
    h, w, b, x, weight = whole_numbers(n, k, d, torch.bfloat16, 5)
    b[128:256] = -1e10
    b[256:512] = -1e30
    b[512:768] = -float("inf")
    b[768:1024] = torch.finfo(torch.float32).min
    b[1024:1100] = -1e6
    b[1100:1400] = -3e9
    x[:, 512:768] = 0
    for kind in ("csr", "dense"):
        for likelihood in ("multinomial", "dirichlet"):
            all_of_it(h, w, b, x, weight, kind, likelihood, torch.bfloat16)


@pytest.mark.parametrize("kind", ["labels", "csr", "dense"])
@pytest.mark.parametrize("n", [12, 60, 700])
def test_bias_gradient_of_light_rows(n, kind):
    """Rows of a responsibility near 1 and rows of next to none, each with columns of its own: the light rows' columns have the gradient of
    those rows, relative to its own size.  (The heavy rows' p is 0 in 32 bits there, and the light rows' in theirs.)"""
    k, d = 9001, 8
    r = np.random.default_rng(n)
    heavy = torch.arange(n, device="cuda") % 2 == 0
    h = torch.zeros(n, d, device="cuda")
    h[:, 0] = torch.where(heavy, 100.0, -100.0)
    w = torch.zeros(k, d, device="cuda")
    w[:, 0] = torch.where(torch.arange(k, device="cuda") < k // 2, 2.0, -2.0)
    b = torch.from_numpy(r.integers(-8, 9, size=k) / 4).float().cuda()
    x = np.zeros((n, k), dtype=np.int32)
    labels = np.zeros(n, dtype=np.int64)
    for i in range(n):
        at = (0 if i % 2 == 0 else k // 2) + r.choice(k // 2, size=9, replace=False)
        labels[i] = at[0]
        if kind == "labels":
            x[i, at[0]] = 1
        else:
            x[i, at] = r.choice([1, 2, 3, 1000000], size=9) if i % 2 == 0 else r.choice([1, 2, 3], size=9)
    x, labels = torch.from_numpy(x).cuda(), torch.from_numpy(labels).cuda()
    for light in (1e-6, 1e-13, 1e-25):
        weight = torch.where(heavy, 1.0, light)
        want = exact(h, w, b, x, weight, "multinomial", torch.float32)
        from bayespy_amd import regression
        got = regression.log_loss_gradient(h, w, rows_of(x, kind, labels), bias=b, row_weights=weight)[3]
        near(got[:k // 2], [v[:k // 2] for v in want["dbias"]], "dbias of the heavy rows' columns")
        near(got[k // 2:], [v[k // 2:] for v in want["dbias"]], "dbias of the light rows' columns, weight %g" % light)


@pytest.mark.parametrize("kind", ["labels", "csr", "dense"])
@pytest.mark.parametrize("n", [9, 500])
def test_losses_of_sure_rows_are_not_negative(n, kind):
    """The label's z is far above all others: the loss is 0, up to the rounding of z (d + 2 roundings of 2^-23 of sum |h w| for each of its two
    sums), and not below it."""
    from bayespy_amd import regression
    k, d = 700, 300
    gen = torch.Generator(device="cuda").manual_seed(n)
    h = torch.randn(n, d, generator=gen, device="cuda")
    w = torch.randn(k, d, generator=gen, device="cuda") * 0.01
    labels = torch.arange(n, device="cuda") % k
    w[labels[:k]] += h[:k] * 0.2
    x = torch.zeros(n, k, dtype=torch.int32, device="cuda")
    x[torch.arange(n, device="cuda"), labels] = 1 if kind == "labels" else 3
    for t in (torch.float32, torch.bfloat16):
        hh, ww = h.to(t), w.to(t)
        off = 2 * (d + 2) * 2.0**-23 * (hh.double().abs() @ ww.double().abs().t()).max(dim=1).values + 2.0**-18
        for likelihood in ("multinomial", "dirichlet"):
            loss = regression.log_loss(hh, ww, rows_of(x, kind, labels), likelihood=likelihood)
            want = exact(hh, ww, torch.zeros(k, device="cuda"), x, torch.ones(n, device="cuda"), likelihood, t)["loss"][0]
            assert float(want.max()) < 1e-3 and bool((loss >= 0).all())
            assert bool(((loss.double() - want).abs() <= 2 * x.sum(1) * off).all())
