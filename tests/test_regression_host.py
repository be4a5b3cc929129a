"""CPU-only checks of the regression entries: what they refuse before anything is launched, through the C ABI and in Python."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def _rows(**kw):
    from bayespy_amd import _lib
    a = _lib.CountRowsArg()
    a.kind = kw.pop("kind", 0)
    a.labels = kw.pop("labels", 4096)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bytes(rows, type_=0, N=10, K=100, D=16, ldh=None, ldw=None, H=4096, W=8192, gradient=1):
    from bayespy_amd import _lib
    return _lib.lib().dme_log_loss_workspace_bytes(H, D if ldh is None else ldh, W, D if ldw is None else ldw, type_, N, K, D, ctypes.addressof(rows), gradient)


def test_workspace_of_what_is_taken_and_refused():
    assert _bytes(_rows()) > 0
    assert _bytes(_rows(), N=0) > 0
    assert _bytes(_rows(), gradient=0) < _bytes(_rows())
    assert _bytes(_rows(), D=15, ldh=16, ldw=16) > _bytes(_rows(), D=16)  # copies of the operands
    for bad in (dict(type_=2), dict(N=-1), dict(K=0), dict(D=0), dict(ldh=8), dict(ldw=8), dict(H=0), dict(W=0), dict(W=8193), dict(K=1 << 31), dict(K=(1 << 29) + 1),
                dict(D=(1 << 20) + 1)):
        assert _bytes(_rows(), **bad) == -1, bad
    for rows in (_rows(kind=3), _rows(labels=0), _rows(kind=1, rowptr=0), _rows(kind=1, rowptr=8, nnz=-1), _rows(kind=1, rowptr=8, nnz=5),
                 _rows(kind=2, X=0, elem=2, ld=100), _rows(kind=2, X=8, elem=3, ld=100), _rows(kind=2, X=8, elem=4, ld=99)):
        assert _bytes(rows) == -1


def test_calls_refused_before_any_launch():
    from bayespy_amd import _lib
    L, rows = _lib.lib(), _rows()
    need = _bytes(rows)

    def call(likelihood=0, ws=1 << 20, size=need, loss=4096, dh=4096, dw=4096):
        return L.dme_log_loss_gradient(4096, 16, 8192, 16, 0, 0, 10, 100, 16, ctypes.addressof(rows), likelihood, 0, loss, dh, dw, 0, ws, size, 0)
    assert call(likelihood=7) == _lib.ERR_INVALID_ARG
    assert call(dw=0) == call(dh=0) == call(loss=0) == call(dw=4104) == call(dh=4097) == _lib.ERR_INVALID_ARG
    assert call(size=need - 1) == call(ws=0) == call(ws=(1 << 20) + 128) == _lib.ERR_WORKSPACE
    assert L.dme_log_loss(4096, 16, 8192, 16, 0, 0, 10, 100, 16, ctypes.addressof(rows), 0, 4096, 0, 0, 0) == _lib.ERR_WORKSPACE
    assert L.dme_log_loss(4096, 16, 8192, 16, 0, 0, 10, 100, 16, 0, 0, 4096, 0, 0, 0) == _lib.ERR_INVALID_ARG
    assert L.dme_log_loss(4096, 16, 8192, 16, 0, 0, 0, 100, 16, ctypes.addressof(rows), 0, 0, 0, 0, 0) == _lib.OK  # no rows: nothing to do


def test_step_refused_before_any_launch():
    from bayespy_amd import _lib
    L = _lib.lib()
    need = L.dme_orthogonal_step_workspace_bytes(0, 1, 300, 200)
    assert need > 0 and L.dme_orthogonal_step_workspace_bytes(1, 3, 300, 200) > 0
    assert L.dme_orthogonal_step_workspace_bytes(0, 0, 300, 200) >= 0  # no matrices
    for bad in ((2, 1, 3, 3), (0, -1, 3, 3), (0, 1, 0, 3), (0, 1, 3, 0), (0, 1, 1 << 17, 1 << 17), (0, 65536, 3, 3)):
        assert L.dme_orthogonal_step_workspace_bytes(*bad) == -1

    def call(steps=5, a=3.4445, b=-4.775, c=2.0315, out=4096, size=need, batch=1, G=4096):
        return L.dme_orthogonal_step(G, 0, 200, 1, 0, batch, 300, 200, steps, a, b, c, out, 1 << 20, size, 0)
    assert call(steps=0) == call(steps=65) == call(out=0) == call(G=0) == _lib.ERR_INVALID_ARG
    # singular values that begin at 1 grow beyond 3, or the polynomial is no number
    assert call(a=4.0, b=0.0, c=0.0) == call(a=1.0, b=0.0, c=100.0) == call(a=float("nan")) == call(b=float("inf")) == _lib.ERR_INVALID_ARG
    assert call(size=need - 1) == _lib.ERR_WORKSPACE
    assert call(batch=0) == _lib.OK


def test_python_refusals_without_a_gpu():
    from bayespy_amd import regression as R
    with pytest.raises(ValueError):
        R.CountRows.from_labels(torch.zeros(3, dtype=torch.int32), 5)
    with pytest.raises(ValueError):
        R.CountRows.from_labels(torch.zeros(3, 1, dtype=torch.int64), 5)
    with pytest.raises(ValueError):
        R.CountRows.from_labels(torch.zeros(3, dtype=torch.int64), 0)
    with pytest.raises(ValueError):
        R.CountRows.from_csr(torch.zeros(0, dtype=torch.int64), torch.zeros(0, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), 5)
    with pytest.raises(ValueError):
        R.CountRows.from_csr(torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 5)
    with pytest.raises(ValueError):
        R.CountRows.from_dense(torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="GPU"):
        R.CountRows.from_labels(torch.zeros(3, dtype=torch.int64), 5)
    with pytest.raises(ValueError):
        R.orthogonal_step(torch.zeros(3, dtype=torch.float32))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            R.orthogonal_step(torch.zeros(3, 4))
