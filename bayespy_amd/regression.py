"""Count rows under a linear predictor: the log loss, its gradient, and the step of its weights.

`dirichletMultinomialEstimation` fits one parameter vector to all rows.  Here every row has one of its own,
z = features @ weights.T + bias, under the same likelihoods (DE/dme.py:16-48 with alpha = exp(z), or the multinomial's
softmax(z)); bias = log(priors) of `findDirichletPriors` is the start that leaves the prior's fit unchanged, as the
reference's DirichletRegression/dirichletRegression.py:137-141 starts from it.

    rows = CountRows.from_csr(rowptr, colidx, vals, K)      # or from_labels(labels, K), from_dense(X)
    loss = log_loss(features, weights, rows, bias=bias, likelihood="dirichlet")
    loss, dfeatures, dweights, dbias = log_loss_gradient(features, weights, rows, bias=bias, row_weights=r)
    weights -= rate * orthogonal_step(dweights)
    features_of_an_encoder.backward(dfeatures)              # where the features are learned too

Everything is enqueued on the current stream of the operands' device and nothing waits; scratch memory comes from
torch's allocator, call by call, so calls on several streams and captured graphs share none.  All computation is in
libdme_hip.so (include/dme_hip.h: dme_log_loss, dme_log_loss_gradient, dme_orthogonal_step).
"""
import ctypes

import torch

from . import _lib
from .device import _on, _ptr, _stream, require_gpu

_TYPES = {torch.float32: 0, torch.bfloat16: 1}          # DME_TYPE_*
_LIKELIHOODS = {"multinomial": 0, "dirichlet": 1}       # DME_LIKELIHOOD_*
_LABELS, _CSR, _DENSE = 0, 1, 2                         # DME_ROWS_*


def _flat(t, dtype, name, device):
    if not torch.is_tensor(t) or t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")


class CountRows:
    """N rows of counts over K columns, in one of three forms.  Holds references: rows whose tensors change in place
    are read as they are when a call runs.  A row that breaks its form has loss NaN (and makes the gradient NaN);
    check() says what is wrong."""

    def __init__(self, kind, N, K, device, tensors, elem=0, ld=0):
        self.N, self.K, self.device = int(N), int(K), device
        self._kind, self._tensors, self._elem, self._ld = kind, tensors, int(elem), int(ld)
        if self.K < 1:
            raise ValueError("K must be positive")
        if device.type != "cuda":
            raise RuntimeError("bayespy_amd runs on the GPU only")

    @classmethod
    def from_labels(cls, labels, K):
        """One count per row, in column labels[i] (int64 [N]); a negative label is a row without counts."""
        _flat(labels, torch.int64, "labels", None)
        return cls(_LABELS, labels.numel(), K, labels.device, (labels,))

    @classmethod
    def from_csr(cls, rowptr, colidx, vals, K):
        """rowptr int64 [N+1], colidx int32 [nnz] strictly ascending within a row, vals int32 [nnz] >= 0."""
        _flat(rowptr, torch.int64, "rowptr", None)
        _flat(colidx, torch.int32, "colidx", rowptr.device)
        _flat(vals, torch.int32, "vals", rowptr.device)
        if rowptr.numel() < 1:
            raise ValueError("rowptr has N + 1 values")
        if colidx.numel() != vals.numel():
            raise ValueError("colidx and vals differ in length")
        return cls(_CSR, rowptr.numel() - 1, K, rowptr.device, (rowptr, colidx, vals))

    @classmethod
    def from_dense(cls, X):
        """X: uint16 or int32 [N, K], values contiguous within a row, any row pitch."""
        if not torch.is_tensor(X) or X.dtype not in (torch.uint16, torch.int32) or X.dim() != 2:
            raise ValueError("X must be a 2-D uint16 or int32 tensor")
        ld = _pitch(X, "X")
        return cls(_DENSE, X.shape[0], X.shape[1], X.device, (X,), elem=X.element_size(), ld=ld)

    def check(self):
        """Raises ValueError where a row breaks the form (waits for the device)."""
        if self._kind == _LABELS:
            if bool((self._tensors[0] >= self.K).any()):
                raise ValueError("a label is not below K")
        elif self._kind == _DENSE:
            X = self._tensors[0]
            if X.dtype == torch.int32 and bool((X < 0).any()):
                raise ValueError("negative counts")
        else:
            rowptr, col, val = self._tensors
            nnz = col.numel()
            if bool((rowptr < 0).any()) or bool((rowptr > nnz).any()) or bool((rowptr[1:] < rowptr[:-1]).any()):
                raise ValueError("rowptr must ascend within 0..nnz")
            first, last = (int(rowptr[0]), int(rowptr[-1]))
            col, val = col[first:last], val[first:last]
            if bool((col < 0).any()) or bool((col >= self.K).any()):
                raise ValueError("a column is out of range")
            if bool((val < 0).any()):
                raise ValueError("negative counts")
            begins = torch.zeros(last - first + 1, dtype=torch.bool, device=col.device)
            begins[rowptr - first] = True
            if bool(((col[1:] <= col[:-1]) & ~begins[1:last - first]).any()):
                raise ValueError("columns must ascend strictly within a row")
        return self

    def _arg(self):
        t = self._tensors
        if self._kind == _LABELS:
            return _lib.CountRowsArg(_LABELS, 0, t[0].data_ptr())
        if self._kind == _CSR:
            return _lib.CountRowsArg(_CSR, 0, None, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), t[1].numel())
        return _lib.CountRowsArg(_DENSE, self._elem, None, None, None, None, 0, t[0].data_ptr(), self._ld)


def _pitch(t, name):
    """Row pitch, in values, of a matrix whose rows are contiguous and do not overlap."""
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must be contiguous within a row")
    if rows <= 1:
        return max(cols, 1)
    if t.stride(0) < cols:
        raise ValueError(f"the rows of {name} overlap")
    return t.stride(0)


def _operand(t, name, device):
    """(rows, columns, pointer, pitch) of features or weights."""
    if not isinstance(t, torch.Tensor) or t.dtype not in _TYPES or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D float32 or bfloat16 tensor")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    n, d = t.shape
    return n, d, t.data_ptr(), max(d, 1) if t.is_contiguous() else _pitch(t, name)


def _call(features, weights, rows, bias, likelihood):
    """Checks what log_loss and log_loss_gradient share; returns the arguments up to the likelihood."""
    if not isinstance(rows, CountRows):
        raise ValueError("rows must be a CountRows")
    if likelihood not in _LIKELIHOODS:
        raise ValueError(f"likelihood must be one of {', '.join(_LIKELIHOODS)}")
    device = rows.device  # a GPU: CountRows takes no other
    N, D, h, ldh = _operand(features, "features", device)
    K, width, w, ldw = _operand(weights, "weights", device)
    if features.dtype != weights.dtype:
        raise ValueError("features and weights differ in type")
    if N != rows.N or K != rows.K or width != D or D < 1:
        raise ValueError(f"features {tuple(features.shape)} and weights {tuple(weights.shape)} do not fit {rows.N} rows of {rows.K} columns")
    if bias is not None:
        _flat(bias, torch.float32, "bias", device)
        if bias.numel() != K:
            raise ValueError(f"bias must have {K} values")
    return (h, ldh, w, ldw), (N, K, D)


def _records_nothing(what, instead, *tensors):
    """Results carry no graph; a loss that silently lacks its gradient is refused instead, as torch refuses out=."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} records no graph for a backward pass and an argument requires a gradient: {instead}, "
                         "or call it under torch.no_grad() or with detached tensors")


_NEEDS = {}  # scratch bytes by what they depend on: sizes, pitches, alignment


def _workspace(operands, kind, shape, rows, arg, gradient):
    key = (operands[0] % 16, operands[1], operands[2] % 16, operands[3], kind, shape, rows._kind, arg.nnz, gradient)
    need = _NEEDS.get(key)
    if need is None:
        need = _lib.lib().dme_log_loss_workspace_bytes(*operands, kind, *shape, ctypes.addressof(arg), gradient)
        if need < 0:
            _lib.check(_lib.ERR_INVALID_ARG)
        if len(_NEEDS) >= 1024:
            _NEEDS.clear()
        _NEEDS[key] = need
    return torch.empty(max(need, 256), dtype=torch.uint8, device=rows.device)


def log_loss(features, weights, rows, bias=None, likelihood="multinomial"):
    """Negative log-likelihood of each row, float32 [N] (without the coefficient that does not depend on z).

    features [N, D] and weights [K, D]: float32 or bfloat16; bias: float32 [K] or None (-inf takes a column out).
    No graph is recorded: where autograd would record one (gradients enabled, an argument that requires one) the call is refused."""
    operands, shape = _call(features, weights, rows, bias, likelihood)
    _records_nothing("log_loss", "take log_loss_gradient", features, weights, bias)
    with _on(rows.device):
        loss = torch.empty(rows.N, dtype=torch.float32, device=rows.device)
        if rows.N == 0:
            return loss
        arg, kind = rows._arg(), _TYPES[features.dtype]
        ws = _workspace(operands, kind, shape, rows, arg, 0)
        _lib.check(_lib.lib().dme_log_loss(*operands, _ptr(bias), kind, *shape, ctypes.addressof(arg),
                                           _LIKELIHOODS[likelihood], loss.data_ptr(), ws.data_ptr(), ws.numel(), _stream()))
    return loss


def log_loss_gradient(features, weights, rows, bias=None, likelihood="multinomial", row_weights=None):
    """(loss, dfeatures, dweights, dbias): the loss of each row, unweighted, and the gradient of
    sum_i row_weights[i] * loss[i] (float32 [N], None = ones: the responsibilities of a mixture's component, or 1 / N).
    dfeatures and dweights have the features' type, dbias is float32 and None where there is no bias.

    The results are plain tensors, whatever the arguments require: the gradient is in them, and the loss beside it has no graph.
    The derivative in z is rounded once to the features' type before its products with the weights and the features (dbias is summed before
    that): in bfloat16 dfeatures and dweights are off by about 0.0022 of their norm, where one rounding of the result alone is 0.0016."""
    operands, shape = _call(features, weights, rows, bias, likelihood)
    if row_weights is not None:
        _flat(row_weights, torch.float32, "row_weights", rows.device)
        if row_weights.numel() != rows.N:
            raise ValueError(f"row_weights must have {rows.N} values")
    dev = rows.device
    with _on(dev):
        loss = torch.empty(rows.N, dtype=torch.float32, device=dev)
        dfeatures = torch.empty(features.shape, dtype=features.dtype, device=dev)
        dweights = torch.empty(weights.shape, dtype=weights.dtype, device=dev)
        dbias = None if bias is None else torch.empty(rows.K, dtype=torch.float32, device=dev)
        arg, kind = rows._arg(), _TYPES[features.dtype]
        ws = _workspace(operands, kind, shape, rows, arg, 1)
        _lib.check(_lib.lib().dme_log_loss_gradient(
            *operands, _ptr(bias), kind, *shape, ctypes.addressof(arg), _LIKELIHOODS[likelihood], _ptr(row_weights),
            loss.data_ptr(), dfeatures.data_ptr(), dweights.data_ptr(), _ptr(dbias), ws.data_ptr(), ws.numel(), _stream()))
    return loss, dfeatures, dweights, dbias


def orthogonal_step(update, steps=5, coefficients=(3.4445, -4.7750, 2.0315)):
    """The update matrix with its singular values brought near one: X = update / |update|, then `steps` times
    X <- a X + (b S + c S S) X with S = X X'.  The coefficients are those of Jordan et al. 2024 (Muon): five steps take singular values
    from 0.005 of |update| on to between 0.68 and 1.16.  update: float32 or bfloat16, [rows, cols] or a batch [B, rows, cols], any
    strides; the result is contiguous and of the same type, and has no graph (refused where autograd would record one).  A zero matrix
    gives zeros.  The step from the gradient alone that stands beside device.predicted_step, which needs a Hessian."""
    if not torch.is_tensor(update) or update.dtype not in _TYPES or update.dim() not in (2, 3):
        raise ValueError("update must be a float32 or bfloat16 matrix or a batch of them")
    if update.shape[-1] < 1 or update.shape[-2] < 1:
        raise ValueError("empty matrix")
    if not 1 <= int(steps) <= 64:
        raise ValueError("steps must be in 1..64")
    _records_nothing("orthogonal_step", "take the gradient's values", update)
    a, b, c = (float(v) for v in coefficients)
    dev = require_gpu(update.device)
    batch = update.shape[0] if update.dim() == 3 else 1
    rows, cols = update.shape[-2:]
    with _on(dev):
        out = torch.empty(update.shape, dtype=update.dtype, device=dev)
        L, kind = _lib.lib(), _TYPES[update.dtype]
        need = L.dme_orthogonal_step_workspace_bytes(kind, batch, rows, cols)
        if need < 0:
            _lib.check(_lib.ERR_INVALID_ARG)
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
        _lib.check(L.dme_orthogonal_step(
            update.data_ptr(), update.stride(0) if update.dim() == 3 else 0, update.stride(-2), update.stride(-1), kind,
            batch, rows, cols, int(steps), a, b, c, out.data_ptr(), ws.data_ptr(), ws.numel(), _stream()))
    return out
