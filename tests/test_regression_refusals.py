"""Refusals of the regression functions that need no GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_a_step_that_autograd_would_record():
    from bayespy_amd import regression
    update = torch.zeros(3, 4, requires_grad=True)
    with pytest.raises(ValueError, match="no graph"):
        regression.orthogonal_step(update)
    if not torch.cuda.is_available():
        with torch.no_grad(), pytest.raises(RuntimeError):  # taken as it is: then there is no GPU
            regression.orthogonal_step(update)
