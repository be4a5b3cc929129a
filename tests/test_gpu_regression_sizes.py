"""Log losses at sizes where a kernel changes its way, on random operands: features beyond a register buffer and beyond 512, rows and columns
enough for split sums, rows that lie anywhere.  Definition and tolerances as in test_gpu_regression."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_regression import TYPES, as_rows, make, near, oracle  # noqa: E402


def moved(t, shift, more):
    """The same values with a pitch, `shift` values from the beginning; NaN between them."""
    big = torch.full((t.shape[0], t.shape[1] + more), float("nan"), dtype=t.dtype, device=t.device)
    view = big[:, shift:shift + t.shape[1]]
    view.copy_(t)
    return view


def label_rows(x):
    from bayespy_amd.regression import CountRows
    y = torch.where(x.sum(1) > 0, x.argmax(1), -1)
    one = torch.zeros_like(x)
    has = (y >= 0).nonzero().squeeze(1)
    one[has, y[has]] = 1
    return one, CountRows.from_labels(y.cuda(), x.shape[1])


@pytest.mark.parametrize("n", [1, 7, 16])
@pytest.mark.parametrize("dtype,d", [("bf16", d) for d in (8, 255, 256, 257, 511, 512, 513, 900, 1500, 1877)] + [("f32", d) for d in (4, 127, 128, 129, 200, 201, 513, 900)])
def test_few_rows(n, dtype, d):
    """Up to 16 rows' weights go from memory to registers, 512 bytes of a row at a time, from where they lie."""
    from bayespy_amd import regression
    h, w, b, x, g = make(n, 333, d, TYPES[dtype], d + n)
    one, labels = label_rows(x)
    for counts, rows in ((x, as_rows(x, "csr")), (one, labels)):
        for likelihood in ("multinomial", "dirichlet"):
            want = oracle(h, w, b, counts, g, likelihood, TYPES[dtype])["loss"]
            for hh, ww in ((h, w), (moved(h, 1, 3), moved(w, 3, 8)), (moved(h, 2, 18), w), (h, moved(w, 1, 1)), (moved(h, 8, 16), moved(w, 8, 24))):
                near(regression.log_loss(hh, ww, rows, bias=b, likelihood=likelihood), want, "loss")


@pytest.mark.parametrize("kind", ["csr", "dense16"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(300, 700, 520), (2050, 260, 1000), (40, 3000, 520), (9, 1500, 1000), (1000, 1031, 777)])
def test_gradients_of_many_features(shape, dtype, kind):
    """More than 512 features: the two products are launched one after the other, each cut in its own way."""
    from bayespy_amd import regression
    n, k, d = shape
    h, w, b, x, g = make(n, k, d, TYPES[dtype], n, density=0.02)
    want = oracle(h, w, b, x, g, "multinomial", TYPES[dtype])
    for hh, ww in ((h, w), (moved(h, 1, 9), moved(w, 2, 5))):
        loss, dh, dw, db = regression.log_loss_gradient(hh, ww, as_rows(x, kind), bias=b, row_weights=g)
        near(loss, want["loss"], "loss")
        near(dh, want["dh"], "dfeatures")
        near(dw, want["dw"], "dweights")
        near(db, want["db"], "dbias")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["csr", "labels", "dense16"])
def test_pieces_of_both_sums(kind, dtype):
    """More rows than a block: dW goes on from block to block, dbias too, with a ragged last block."""
    from bayespy_amd import regression
    n, k, d = 2 * 16384 + 21, 150, 12
    h, w, b, x, g = make(n, k, d, TYPES[dtype], 40, density=0.03)
    rows = None
    if kind == "labels":
        x, rows = label_rows(x)
    want = oracle(h, w, b, x, g, "multinomial", TYPES[dtype])
    loss, dh, dw, db = regression.log_loss_gradient(h, w, rows or as_rows(x, kind), bias=b, row_weights=g)
    near(loss, want["loss"], "loss")
    near(dh, want["dh"], "dfeatures")
    near(dw, want["dw"], "dweights")
    near(db, want["db"], "dbias")


def test_rows_cut_from_a_larger_matrix():
    """A part of rowptr is a CSR matrix of its own, whatever comes before and after its entries."""
    from bayespy_amd import regression
    from bayespy_amd.regression import CountRows
    h, w, b, x, g = make(120, 400, 24, torch.float32, 50)
    rowptr, col, val = as_rows(x, "csr")._tensors
    for first, last in ((0, 7), (7, 60), (60, 120), (119, 120), (30, 30)):
        rows = CountRows.from_csr(rowptr[first:last + 1], col, val, 400).check()
        whole = as_rows(x[first:last], "csr") if last > first else None
        for likelihood in ("multinomial", "dirichlet"):
            got = regression.log_loss_gradient(h[first:last], w, rows, bias=b, likelihood=likelihood, row_weights=g[first:last])
            if whole is None:
                assert got[0].shape == (0,) and not bool(got[2].any()) and not bool(got[3].any())
                continue
            want = oracle(h[first:last], w, b, x[first:last], g[first:last], likelihood, torch.float32)
            for value, name in zip(got, ("loss", "dh", "dw", "db")):
                near(value, want[name], name)


def test_a_bias_gradient_that_leaves_32_bits():
    """weight * count beyond 32 bits: no number, in its column alone."""
    from bayespy_amd import regression
    h, w, b, x, _ = make(40, 600, 16, torch.float32, 4)
    b[:] = 0.0
    b[300:] = -200.0
    x[:, 300:] = 0
    x[1:, 400] = 3
    x[0, :] = 0
    x[0, 5] = 2
    g = torch.ones(40, device="cuda")
    g[0] = 3e38
    db = regression.log_loss_gradient(h, w, as_rows(x, "csr"), bias=b, row_weights=g)[3]
    assert bool(torch.isnan(db[5])) and bool(torch.isfinite(db[300:]).all())


@pytest.mark.parametrize("kind", ["csr", "labels"])
def test_bias_gradient_of_a_wide_vocabulary(kind):
    """Column sums by ranges of every width, up to the widest.  Weights of 0: z is the bias, p the same for all rows, and the gradient
    p sum_i g_i T_i - sum_i g_i x_ik.  p is off by 2^-22 (|b - l| + 4) + 2^-17 (its sum), each sum over n rows by n 2^-23 of its terms."""
    from bayespy_amd import regression
    from bayespy_amd.regression import CountRows
    gen = torch.Generator(device="cuda").manual_seed(9)
    n = 3000
    for k in (1023, 5000, 70001, 300007):
        b = torch.randn(k, generator=gen, device="cuda")
        g = torch.rand(n, generator=gen, device="cuda")
        each = 1 if kind == "labels" else 40
        col = (torch.rand(n, each, generator=gen, device="cuda").pow(3) * k).long().clamp(max=k - 1)
        val = torch.randint(1, 50, (n, each), generator=gen, device="cuda") if kind == "csr" else torch.ones_like(col)
        if kind == "labels":
            rows = CountRows.from_labels(col[:, 0].contiguous(), k)
        else:
            col = col.sort(dim=1).values
            val[:, 1:] *= col[:, 1:] != col[:, :-1]  # a column once
            at = (val > 0).nonzero(as_tuple=True)
            rowptr = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
            rowptr[1:] = (val > 0).sum(1).cumsum(0)
            rows = CountRows.from_csr(rowptr, col[at].int(), val[at].int(), k).check()
        h, w = torch.randn(n, 4, generator=gen, device="cuda"), torch.zeros(k, 4, device="cuda")
        got = regression.log_loss_gradient(h, w, rows, bias=b, row_weights=g)[3].double()
        total, counts = val.sum(1).double(), torch.zeros(k, dtype=torch.float64, device="cuda")
        counts.index_add_(0, col.reshape(-1), (val * g.double()[:, None]).reshape(-1))
        z = b.double()
        l = torch.logsumexp(z, 0)
        first = torch.exp(z - l) * (g.double() * total).sum()
        tol = first * (2.0**-22 * ((z - l).abs() + 4) + 2.0**-17 + n * 2.0**-23) + (n + 1) * 2.0**-23 * counts + 2.0**-24 * (first + counts)
        assert bool(((got - (first - counts)).abs() <= tol).all()), k
