"""How the regression operators are called: what autograd does not see, rows cut from larger ones."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_a_graph_that_would_be_missing_is_refused():
    """log_loss and orthogonal_step record none; log_loss_gradient takes parameters, its results are the gradient."""
    from bayespy_amd import regression as R
    gen = torch.Generator(device="cuda").manual_seed(2)
    h, w, b = (torch.randn(s, generator=gen, device="cuda") for s in ((30, 16), (50, 16), (50,)))
    rows = R.CountRows.from_labels(torch.arange(30, device="cuda"), 50)
    want, grads = R.log_loss(h, w, rows, bias=b), R.log_loss_gradient(h, w, rows, bias=b)
    for i in range(3):
        t = [h, w, b]
        t[i] = t[i].clone().requires_grad_()
        with pytest.raises(ValueError, match="log_loss_gradient"):
            R.log_loss(t[0], t[1], rows, bias=t[2])
        with torch.no_grad():
            assert torch.equal(R.log_loss(t[0], t[1], rows, bias=t[2]), want)
        for got, one in zip(R.log_loss_gradient(t[0], t[1], rows, bias=t[2]), grads):
            assert torch.equal(got, one) and not got.requires_grad
    p = w.clone().requires_grad_()
    with pytest.raises(ValueError, match="no graph"):
        R.orthogonal_step(p)
    assert torch.equal(R.orthogonal_step(p.detach()), R.orthogonal_step(w))
