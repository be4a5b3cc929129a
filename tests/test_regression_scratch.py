"""What the regression entries ask for as scratch memory: no more than the header lists.  No GPU."""
import ctypes


def _bytes(N, K, D, gradient, type_=1, kind=0, nnz=0):
    from bayespy_amd import _lib
    rows = _lib.CountRowsArg()
    rows.kind, rows.labels, rows.rowptr, rows.colidx, rows.vals, rows.nnz = kind, 4096, 4096, 4096, 4096, nnz
    rows.X, rows.ld, rows.elem = 4096, K, 2
    return _lib.lib().dme_log_loss_workspace_bytes(4096, D, 8192, D, type_, N, K, D, ctypes.addressof(rows), gradient)


def test_sums_of_dbias_take_the_place_of_the_forward_pieces():
    """16384 labels, 2^20 columns: tiles of 256 leave 8 bytes for 256 columns of each row; dbias's sums, 8 and 4 bytes of each column for 256 rows,
    are 1.5 times that and lie in the same place.  Beside them 256 MB of d loss / d z, dW in 32 bits where its sum is split (no more pieces than two),
    dH in 32 bits in at most 64 pieces, and a few bytes a row."""
    n, k, d = 16384, 1 << 20, 64
    forward, sums = n * (k // 256) * 8, k * (n // 256) * 12
    loss, gradient = _bytes(n, k, d, 0), _bytes(n, k, d, 1)
    assert forward <= loss <= forward + n * 4 + 1024
    rest = (256 << 20) + 2 * k * d * 4 + 64 * n * d * 4 + n * 32 + 4096
    assert sums <= gradient <= sums + rest


def test_dense_rows_leave_more_than_dbias_needs():
    n, k, d = 16384, 4096, 64
    forward, sums = n * (k // 128) * 32, k * (n // 128) * 4
    assert sums < forward
    gradient = _bytes(n, k, d, 1, kind=2)
    dz = n * k * 2
    assert forward + dz <= gradient <= forward + dz + 64 * (n + k) * d * 4 + n * 32 + 4096


def test_no_empty_pieces_of_a_step_s_square():
    """Every piece that k is cut into has slices (64 halves each) of its own.  The rest of what a step of matrices beyond 64 singular values takes is
    its pairs, S and B, so the pieces' number follows from the bytes."""
    from bayespy_amd import _lib
    up = lambda v, to: (v + to - 1) // to * to  # noqa: E731
    several = 0
    for type_ in (0, 1):
        for m, n in ((250, 2000), (2000, 250), (100, 8300), (129, 129), (300, 5000), (512, 4097), (70, 20000), (250, 8321), (1000, 1030)):
            rows, cols = m, n
            ldx, small = up(cols, 8), min(m, n)
            lds, parts = up(small, 8), 2 if type_ == 0 else 1
            sizes = [256 * 8] + [rows * ldx * 2] * 4 + [small * lds * 2] * 2 * parts + [lds * 4] * 2
            if type_ == 0:
                sizes += [rows * ldx * 4, small * lds * 4]
            left = _lib.lib().dme_orthogonal_step_workspace_bytes(type_, 1, rows, cols) - sum(up(s, 256) for s in sizes)
            slices = -(-max(m, n) * 2 // 128)
            pieces = left // (small * lds * 4)
            assert left == up(pieces * small * lds * 4, 256)
            if pieces:
                several += 1
                assert -(-slices // -(-slices // pieces)) == pieces, (type_, m, n, slices, pieces)
    assert several > 6
