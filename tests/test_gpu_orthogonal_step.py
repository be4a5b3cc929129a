"""orthogonal_step where one launch makes a step (up to 64 singular values, up to 4096 the other way), on both sides of that border, and from strides:
held to its type's rounding.

The result's own rounding is off by u = eps / 2 of each value at most, so by u of any part of the matrix in norm; the steps before may add as much again in bf16.
In fp32 a step's products are off by 2^-24 sqrt(n) at a sum of n terms (32-bit products), or 2^-21 (pairs of halves), times
`one` = a + 4 |b| 1.2^2 + 8 |c| 1.2^4 (see test_gpu_regression), and each of the two steps after a step enlarges that by a at most
before the singular values are near 1."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

A, B, C = 3.4445, -4.7750, 2.0315
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def steps_of(g, steps=5):
    y = g.double().reshape(-1, *g.shape[-2:])
    norm = torch.linalg.vector_norm(y, dim=(1, 2), keepdim=True)
    y = y / norm
    tall = y.shape[1] > y.shape[2]
    for _ in range(steps):
        t = y.transpose(1, 2).contiguous()
        s = t @ y if tall else y @ t
        q = B * s + C * (s @ s)
        y = A * y + (y @ q if tall else q @ y)
    return y


def hold(g, steps=5):
    from bayespy_amd import regression
    got, want = regression.orthogonal_step(g, steps=steps), steps_of(g, steps)
    assert got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    u = torch.finfo(g.dtype).eps / 2
    one = A - 4 * B * 1.44 + 8 * C * 2.07
    tol = 2 * u if g.dtype == torch.bfloat16 else u + one * 2.0**-21 * (1 + A + A**2)
    off = got.double().reshape(want.shape) - want
    rows, cols = want.shape[1:]
    for r in (slice(None), slice(0, 16), slice(max(rows - 16, 0), None)):
        for c in (slice(None), slice(0, 16), slice(max(cols - 16, 0), None)):
            for m in (slice(None), slice(-1, None)):
                part = (m, r, c)
                assert float(torch.linalg.vector_norm(off[part])) <= tol * float(torch.linalg.vector_norm(want[part])), part


@pytest.mark.parametrize("steps", [1, 2, 5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 200), (33, 7), (64, 64), (48, 65), (1000, 64), (64, 1025), (1024, 64), (4096, 48), (64, 4096), (50, 3001), (2, 1500, 64),
                                   (5, 40, 130), (3, 64, 2000), (4097, 64), (5000, 48), (48, 5000), (17000, 50), (64, 17001), (130, 257), (500, 100), (3, 70, 129)])
def test_every_value(shape, dtype, steps):
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    hold((torch.randn(shape, generator=gen, device="cuda") * 1e-3).to(TYPES[dtype]), steps)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_any_strides(dtype):
    """Views of a larger tensor: pitches, turned, spread out, the same matrix again; on either side of 64 singular values."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    whole = torch.randn(6, 1100, 200, generator=gen, device="cuda").to(TYPES[dtype])
    for view in (whole[:, 3:70, 5:140], whole[:, 3:70, 5:140].transpose(1, 2), whole[::2, ::3, ::4], whole[1:2].expand(3, 1100, 200), whole[0].t(), whole[0, :33, ::3],
                 whole[0, ::3, :33].t(), whole[:, :, 7:60], whole[:, 1:, 7:60].transpose(1, 2), whole[2, :, ::4], whole[2, :, ::4].t(), whole[1:2, :, :50].expand(3, 1100, 50)):
        hold(view)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1000, 64), (64, 3000), (9000, 60), (2000, 130), (20000, 200)])
def test_strong_directions_over_weak_noise(shape, dtype):
    """A gradient's spectrum.  Weak directions enlarge what the first steps round off by a each, so fp32 is held to what the same steps are
    off by in 32-bit arithmetic, and bf16 to its rounding as everywhere."""
    from bayespy_amd import regression
    gen = torch.Generator(device="cuda").manual_seed(4)
    m, n = shape
    left = torch.randn(m, 16, generator=gen, device="cuda") / torch.arange(1, 17, device="cuda")
    g = left @ torch.randn(16, n, generator=gen, device="cuda") + 0.1 * torch.randn(m, n, generator=gen, device="cuda")
    if dtype == "bf16":
        hold(g.bfloat16())
        return
    want = steps_of(g)[0]
    y = g / torch.linalg.vector_norm(g.double()).float()
    for _ in range(5):
        t = y.t().contiguous()
        s = t @ y if m > n else y @ t
        q = B * s + C * (s @ s)
        y = A * y + (y @ q if m > n else q @ y)
    off = float(torch.linalg.vector_norm(regression.orthogonal_step(g).double() - want))
    # the 32-bit arithmetic's own error is one sample of what roundings make; ours may be another, and rounds its result
    assert off <= 2 * float(torch.linalg.vector_norm(y.double() - want)) + 2.0**-24 * float(torch.linalg.vector_norm(want))
