"""Device-resident operands: calls layer 2 of the C ABI (``comet_b200_dev_*``) on
torch CUDA tensors.  torch supplies device memory and streams only; every
computation is done by the kernels of ``libcomet_b200``.

Beside the sparse operations: the largest entries of rows of logits as a CSR matrix, and two losses of such a matrix beside
logits (``top_entries``, ``distill_loss``, ``balance_loss``).

Used by the benchmark (inputs already in HBM when the clock starts), by the
multi-GPU sharding layer and by the device-level parity tests.
"""
import ctypes

import numpy as np
import torch

from . import _lib
from .api import PLUS_PAIR, PLUS_TIMES, as_sparse  # noqa: F401


class DeviceCSR:
    """A CSR (or DCSR when ``row_ids`` is set) matrix in device memory, int64 indices.

    The sparse operations take float64 values and refuse others; ``top_entries`` gives float32 values, which ``distill_loss`` takes.  Of
    such a matrix S, ``DeviceCSR(S.nrows, S.ncols, S.pos, S.crd, S.val.double())`` is one for the sparse operations."""

    def __init__(self, nrows, ncols, pos, crd, val, row_ids=None):
        self.nrows, self.ncols = int(nrows), int(ncols)
        self.pos, self.crd, self.val, self.row_ids = pos, crd, val, row_ids
        self.nnz = int(crd.shape[0])

    @property
    def nstored(self):
        return int(self.pos.shape[0]) - 1


def to_device(A, device="cuda", pin=False):
    """Host COMET arrays / scipy matrix -> DeviceCSR (COO is not taken here)."""
    A = as_sparse(A)
    if A.format == "COO":
        raise ValueError("to_device: pass CSR or DCSR (the host entry points convert COO)")

    def up(a):
        t = torch.from_numpy(np.ascontiguousarray(a))
        if pin:
            t = t.pin_memory()
        return t.to(device, non_blocking=pin)

    i64 = lambda a: np.asarray(a, dtype=np.int64)       # the device entry points take int64 indices
    row_ids = up(i64(A.a1crd[:int(A.a1pos[1])])) if A.format == "DCSR" else None
    return DeviceCSR(A.nrows, A.ncols, up(i64(A.a2pos)), up(i64(A.a2crd)), up(A.val), row_ids)


def _p(t):
    return 0 if t is None else t.data_ptr()


def _stream():
    # torch.cuda.current_stream() builds a Stream object (2 us); the handle is all that is needed
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _check_cuda(*ts):
    for t in ts:
        if t is not None and not (t.is_cuda and t.is_contiguous()):
            raise ValueError("device entry points need contiguous CUDA tensors")


def _check_f64(*ts):
    """Values that the f64 entry points read or write by their address."""
    for t in ts:
        if t is not None:
            if not (t.is_cuda and t.is_contiguous()):
                raise ValueError("device entry points need contiguous CUDA tensors")
            if t.dtype is not torch.float64:
                raise ValueError("this operation takes float64 values, not %s; convert them with .double()" % t.dtype)


_ready = None


def _call(name, *args):
    """Calls a device entry point (integers and addresses only); raises on a non-zero status."""
    global _ready
    if _ready is None:
        _lib.load()
        from . import _pycall
        _ready = _pycall.call_i32
    st = _ready(_lib.address(name), *args)
    if st:
        _lib.check(st)


def spmv(A, x, y=None, semiring=PLUS_TIMES, accumulate=False):
    _check_cuda(A.pos, A.crd)
    _check_f64(A.val, x, y)
    if y is None:
        # rows the matrix does not store, and the values that are added to, start at zero; any other row is written
        new = torch.zeros if A.row_ids is not None or A.nstored < A.nrows or accumulate else torch.empty
        y = new(A.nrows, dtype=torch.float64, device=x.device)
    _call("comet_b200_dev_spmv_f64_i64", A.nstored, A.nnz, _p(A.row_ids), A.pos.data_ptr(), A.crd.data_ptr(),
          A.val.data_ptr(), x.data_ptr(), y.data_ptr(), semiring, int(accumulate), _stream())
    return y


def spmm(A, B, C=None, semiring=PLUS_TIMES, accumulate=False, variant=0):
    """B may be a column slice of a wider row-major array (unit column stride); its row stride is passed on."""
    _check_cuda(A.pos, A.crd)
    _check_f64(A.val, C)
    if not B.is_cuda or B.dim() != 2 or B.stride(1) != 1 or B.dtype is not torch.float64:
        raise ValueError("B must be a CUDA matrix of float64 values with unit column stride")
    k = B.shape[1]
    if C is None:
        C = torch.empty((A.nrows, k), dtype=torch.float64, device=B.device)
        if A.row_ids is not None:
            C.zero_()
    _call("comet_b200_dev_spmm_f64_i64", A.nstored, A.ncols, A.nnz, k, _p(A.row_ids), A.pos.data_ptr(),
          A.crd.data_ptr(), A.val.data_ptr(), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0),
          semiring, int(accumulate), int(variant), _stream())
    return C


def sddmm(S, X, Y, out=None):
    """Y is [ncols, K] row-major."""
    _check_cuda(S.pos, S.crd)
    _check_f64(S.val, X, Y, out)
    if out is None:
        out = torch.empty(S.nnz, dtype=torch.float64, device=X.device)
    _call("comet_b200_dev_sddmm_f64_i64", S.nrows, S.nnz, X.shape[1], S.pos.data_ptr(), S.crd.data_ptr(),
          S.val.data_ptr(), X.data_ptr(), X.stride(0), Y.data_ptr(), Y.stride(0), out.data_ptr(), _stream())
    return out


class SpgemmResult:
    def __init__(self, nrows, ncols, pos, crd, val):
        self.nrows, self.ncols, self.pos, self.crd, self.val = nrows, ncols, pos, crd, val
        self.nnz = int(crd.shape[0])


def spgemm_symbolic(A, B, M=None, semiring=PLUS_TIMES):
    """Returns (handle, cpos tensor, nnz)."""
    _check_cuda(A.pos, A.crd, B.pos, B.crd)
    _check_f64(A.val, B.val)
    cpos = torch.empty(A.nrows + 1, dtype=torch.int64, device=A.pos.device)
    out = (ctypes.c_int64 * 2)()
    at = ctypes.addressof(out)
    _call("comet_b200_dev_spgemm_symbolic_f64_i64",
          A.nrows, B.ncols, B.nnz, A.pos.data_ptr(), A.crd.data_ptr(), A.val.data_ptr(), B.pos.data_ptr(),
          B.crd.data_ptr(), B.val.data_ptr(), M.pos.data_ptr() if M is not None else 0,
          M.crd.data_ptr() if M is not None else 0, semiring, cpos.data_ptr(), at, at + 8, _stream())
    return out[1], cpos, out[0]


def spgemm_numeric(handle, nnz, device, keep=False, crd=None, val=None):
    if crd is None:
        crd = torch.empty(max(nnz, 1), dtype=torch.int64, device=device)[:nnz]
        val = torch.empty(max(nnz, 1), dtype=torch.float64, device=device)[:nnz]
    if val.dtype is not torch.float64:
        raise ValueError("this operation writes float64 values, not %s" % val.dtype)
    _call("comet_b200_dev_spgemm_numeric_f64_i64", handle, crd.data_ptr(), val.data_ptr(), int(keep), _stream())
    return crd, val


def spgemm(A, B, M=None, semiring=PLUS_TIMES):
    handle, cpos, nnz = spgemm_symbolic(A, B, M, semiring)
    crd, val = spgemm_numeric(handle, nnz, A.pos.device)
    return SpgemmResult(A.nrows, B.ncols, cpos, crd, val)


def masked_pair_count(A, B, M, row_lo=0, row_hi=None, out=None):
    """Device int64 scalar tensor: products of rows [row_lo, row_hi) of A that land on M's pattern."""
    _check_cuda(A.pos, A.crd, B.pos, B.crd, M.pos, M.crd)
    row_hi = A.nrows if row_hi is None else row_hi
    if out is None:
        out = torch.empty(1, dtype=torch.int64, device=A.pos.device)       # cleared by the call
    _call("comet_b200_dev_masked_spgemm_count_f64_i64", row_lo, row_hi, B.ncols, A.nnz, B.nnz, M.nnz,
          A.pos.data_ptr(), A.crd.data_ptr(), B.pos.data_ptr(), B.crd.data_ptr(), M.pos.data_ptr(), M.crd.data_ptr(),
          out.data_ptr(), _stream())
    return out


# Rows of logits beside a CSR matrix.  The logits are CUDA matrices with unit column stride, in bf16, f16 or f32; the
# results are new tensors without a graph (the gradients are for torch.autograd.backward), and every call is asynchronous on the
# current stream.  A gradient written in place of the logits counts as an operation in place: a graph that has saved them refuses its
# backward pass.
_LOGITS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
_TOP, _DISTILL, _BALANCE = ({t: "comet_b200_dev_%s_%s_i64" % (op, name) for t, name in _LOGITS.items()}
                            for op in ("top_entries", "distill_loss", "balance_loss"))
_numbers = {}


def _floats(*v):
    """The address of host doubles, and what keeps them alive (the calls take integers and addresses)."""
    got = _numbers.get(v)
    if got is None:
        if len(_numbers) >= 256:
            _numbers.clear()
        a = (ctypes.c_double * len(v))(*v)
        got = _numbers[v] = (ctypes.addressof(a), a)
    return got


def _check_logits(what, X):
    """(rows, columns, row stride) of a matrix of logits.  The checks are few: they are most of a small call's time on the host."""
    if not (isinstance(X, torch.Tensor) and X.is_cuda and X.dtype in _LOGITS):
        raise ValueError(what + ": the logits must be a CUDA matrix of bfloat16, float16 or float32")
    shape, stride = X.shape, X.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] != 1):
        raise ValueError(what + ": the logits must be a matrix with unit column stride")
    if X.get_device() != torch._C._cuda_getDevice():
        raise ValueError(what + ": the logits must be on the current device")
    n, m = shape
    if m < 1:
        raise ValueError(what + ": the logits have no columns")
    ld = stride[0] if n > 1 else m
    if ld < m:
        raise ValueError(what + ": rows of the logits must not overlap")
    return n, m, ld


def _check_vector(what, v, dtype, n):
    if v.dtype is not dtype or v.shape != (n,) or not v.is_contiguous() or v.get_device() != torch._C._cuda_getDevice():
        raise ValueError("%s: expected %d contiguous values of %s on the logits' device" % (what, n, dtype))
    return v.data_ptr()


def _check_beside(what, S, n, m):
    """Addresses of pos and crd of a CSR matrix of the logits' shape, with int64 indices."""
    if S.row_ids is not None:
        raise ValueError(what + ": the sparse operand must be CSR (a row that stores nothing is empty there)")
    if S.nrows != n or S.ncols != m:
        raise ValueError(what + ": the sparse operand and the logits must have the same shape")
    return _check_vector(what, S.pos, torch.int64, n + 1), _check_vector(what, S.crd, torch.int64, S.nnz)


def _gradient(what, X, shape, grad):
    """(gradient, its address, its row stride): new, none, or the caller's (the logits themselves, say)."""
    if grad is True:
        grad = X.new_empty(shape)
        return grad, grad.data_ptr(), shape[1]
    if grad is None or grad is False:
        return None, 0, 0
    if grad.dtype is not X.dtype or grad.shape != shape:
        raise ValueError(what + ": the gradient must have the logits' shape, type and device")
    ld = _check_logits(what, grad)[2]
    torch.autograd.graph.increment_version(grad)       # written by its address: a graph that has saved it has to know
    return grad, grad.data_ptr(), ld


def top_entries(X, k, temperature=1.0, lse=False):
    """The k largest entries of each row of X (1 <= k <= 1024) as a DeviceCSR with float32 values, columns ascending; of equal entries the lower
    column, NaN above all numbers.  Returns (matrix, the log of the sum of each row's exp(X / temperature), or None); the sparse operations take the
    matrix with its values converted to float64."""
    n, m, ld = _check_logits("top_entries", X)
    k = int(k)
    if not 1 <= k <= min(1024, m):
        raise ValueError("top_entries: k must be between 1 and 1024, and at most the number of columns")
    new = X.new_empty
    pos, crd, val = new(n + 1, dtype=torch.int64), new(n * k, dtype=torch.int64), new(n * k, dtype=torch.float32)
    sums = new(n, dtype=torch.float32) if lse else None
    options = _floats(float(temperature))
    _call(_TOP[X.dtype], n, m, X.data_ptr(), ld, k, options[0], pos.data_ptr(), crd.data_ptr(), val.data_ptr(), _p(sums), _stream())
    return DeviceCSR(n, m, pos, crd, val), sums


def distill_loss(S, X, temperature=1.0, lse=None, weight=None, scale=1.0, grad=True):
    """Distillation from a teacher's top logits: S holds them (DeviceCSR of X's shape, float32 or float64 values, columns of a row ascending), X the
    student's.  With q = softmax(X / temperature) and p = exp(S / temperature) over the sum of the row's entries, a row's loss is
    sum p (log p - log q) over the entries.  lse: the log of the sum of exp(teacher / temperature) over the teacher's whole rows, as top_entries gives
    it; p is then a part of the whole row, and all that is not stored counts as one outcome (none, where the list's p are 1 but for rounding and the
    student gives nothing to the rest).  Rows that store nothing, or whose weight is 0, are
    left out.  One entry in each row: the cross entropy with that column.

    Returns (scale * sum of weight * rows, rows, the gradient of the first with respect to X).  grad: True (a new tensor), False (none), or a tensor to write
    it to, such as X."""
    n, m, ld = shape = _check_logits("distill_loss", X)
    pos, crd = _check_beside("distill_loss", S, n, m)
    width = 4 if S.val.dtype is torch.float32 else 8
    val = _check_vector("distill_loss", S.val, torch.float32 if width == 4 else torch.float64, S.nnz)
    sums = 0 if lse is None else _check_vector("distill_loss", lse, torch.float32, n)
    weights = 0 if weight is None else _check_vector("distill_loss", weight, torch.float32, n)
    out, to, ldg = _gradient("distill_loss", X, shape[:2], grad)
    rows, loss = X.new_empty(n, dtype=torch.float32), X.new_empty((), dtype=torch.float32)
    options = _floats(float(temperature), float(scale))
    _call(_DISTILL[X.dtype], n, m, pos, crd, val, width, sums, weights, X.data_ptr(), ld, to, ldg, options[0], rows.data_ptr(), loss.data_ptr(), _stream())
    return loss, rows, out


def balance_loss(S, R, seq=None, mask=None, scores="softmax", scale=1.0, grad=True):
    """Balance loss of a router: S (DeviceCSR of R's shape, at most 1024 columns; its values are not looked at) says which experts take which tokens, R
    holds the router's logits.  seq: int64 bounds of the sequences, from 0 to the number of rows (None: one); mask: bool, rows that count (rows that store
    nothing do not).  The loss is scale * the mean over sequences with such rows of E * sum_e f_e P_e, f_e the share of the sequence's entries in column e and
    P_e the mean over its rows of p_e, with p = softmax(R) or, for scores="sigmoid", sigmoid(R) over the row's sum.

    Returns (loss, counts[sequences, E] as int64, gradient with respect to R).  grad: True (a new tensor), False (none), or a tensor to write it to, such
    as R.  Calls on one device share the memory that counts, and must not overlap."""
    n, m, ld = shape = _check_logits("balance_loss", R)
    pos, crd = _check_beside("balance_loss", S, n, m)
    if scores not in ("softmax", "sigmoid"):
        raise ValueError("balance_loss: scores must be 'softmax' or 'sigmoid'")
    if m > 1024:
        raise ValueError("balance_loss: at most 1024 experts")
    nseq, bounds = 1, 0
    if seq is not None:
        nseq = seq.numel() - 1
        if nseq < 1:
            raise ValueError("balance_loss: seq holds the bounds of one sequence or more")
        bounds = _check_vector("balance_loss", seq, torch.int64, nseq + 1)
    on = 0 if mask is None else _check_vector("balance_loss", mask, torch.bool, n)
    out, to, ldg = _gradient("balance_loss", R, shape[:2], grad)
    counts, loss = R.new_empty((nseq, m), dtype=torch.int64), R.new_empty((), dtype=torch.float32)
    options = _floats(float(scale))
    _call(_BALANCE[R.dtype], n, m, pos, crd, nseq, bounds, on, int(scores == "sigmoid"), R.data_ptr(), ld, to, ldg, options[0], counts.data_ptr(),
          loss.data_ptr(), _stream())
    return loss, counts, out
