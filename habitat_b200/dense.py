"""Dense layers in 8-bit integers, and orthogonalised weight updates.

* `quantize_rows`, `int8_matmul`, `int8_matmul_quantized`: rows (queries, tokens) in 8-bit integers with one scale each,
  times 8-bit weights with one scale per output channel.  `RuntimePredictor(precision="int8")` runs on them.
* `orthogonalize`: the update of a weight matrix made nearly orthogonal by Newton-Schulz steps.
  `RuntimePredictor.update_hidden` steps the predictors' hidden layers with it.

All take CUDA tensors, queue their work on the current stream without synchronising, allocate results and workspaces
through torch, and run in the library's sm_100a kernels (habitat_b200/csrc/dense_int8.cu, orthogonalize.cu).  The first
call on a GPU sets up a status word there: make it before a stream capture.
"""
import ctypes

import torch

from habitat_b200 import _native

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr() if t is not None else 0)


def _rows_of(t, dtypes, name, device=None):
    """A CUDA matrix whose rows are contiguous -> its pitch."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype not in dtypes:
        raise TypeError("%s must have dtype %s, got %s" % (name, " or ".join(str(d) for d in dtypes), t.dtype))
    if t.ndim != 2:
        raise ValueError("%s must be a matrix" % name)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("%s must have contiguous rows" % name)
    pitch = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if pitch < t.shape[1]:
        raise ValueError("%s must have rows that do not overlap" % name)
    return pitch


def _vector(t, n, name, device):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype != torch.float32:
        raise TypeError("%s must have dtype torch.float32, got %s" % (name, t.dtype))
    if t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError("%s must be a contiguous vector of %d values" % (name, n))


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _rows_of_bytes(rows, cols, device):
    """An int8 matrix whose rows start on 16-byte boundaries."""
    pitch = (cols + 15) // 16 * 16
    t = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return t[:, :cols]


def quantize_rows(x):
    """Rows of a float32, bfloat16 or float16 matrix in 8-bit integers: (q [rows, cols] int8, scales [rows] float32), so that
    q[i, j] * scales[i] is x[i, j] to within half a scale.  In float32: scale = max |x| / 127, q = rint(x * (127 / max |x|)),
    ties to even.  Rows of zeros (magnitudes below 2^-119) get the scale 0, rows with an infinity or a NaN zeros and the scale
    NaN.  q's rows start on 16-byte boundaries, as the products want them."""
    pitch = _rows_of(x, tuple(_TYPES), "x")
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x must have at least one column")
    q = _rows_of_bytes(rows, cols, x.device)
    scales = torch.empty((rows,), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _native.check(_native.load().hb_quantize_rows(
            _ptr(x), _TYPES[x.dtype], rows, cols, pitch, _ptr(q), (cols + 15) // 16 * 16, _ptr(scales), _stream(x.device)))
    return q, scales


def _product_arguments(q, scales, weight, weight_scales, bias):
    q_pitch = _rows_of(q, (torch.int8,), "q")
    w_pitch = _rows_of(weight, (torch.int8,), "weight", q.device)
    m, k = q.shape
    n = weight.shape[0]
    if weight.shape[1] != k:
        raise ValueError("q has %d columns, weight has %d" % (k, weight.shape[1]))
    if not 1 <= k <= 131071:
        raise ValueError("the rows have 1 to 131071 columns (the sums are 32-bit integers), not %d" % k)
    _vector(scales, m, "scales", q.device)
    _vector(weight_scales, n, "weight_scales", q.device)
    if bias is not None:
        _vector(bias, n, "bias", q.device)
    return q_pitch, w_pitch, m, n, k


def _workspace(lib, q, q_pitch, weight, w_pitch, m, n, k, quantized):
    size = lib.hb_int8_workspace_bytes(_ptr(q), q_pitch, _ptr(weight), w_pitch, m, n, k, quantized)
    return (torch.empty((size,), dtype=torch.uint8, device=q.device) if size else None), size


def int8_matmul(q, scales, weight, weight_scales, bias=None, relu=False, out_dtype=torch.float32):
    """q [M, K] int8 with scales [M] times weight [N, K] int8 with weight_scales [N], plus bias [N] float32, then ReLU: [M, N] in
    out_dtype (float32, bfloat16, float16).  The integer sums are exact; (sum * weight scale) * scale + bias in float32, then one
    rounding to out_dtype.  Rows may start anywhere; those that do not start on 16-byte boundaries are copied first."""
    q_pitch, w_pitch, m, n, k = _product_arguments(q, scales, weight, weight_scales, bias)
    if out_dtype not in _TYPES:
        raise TypeError("out_dtype must be float32, bfloat16 or float16, got %s" % (out_dtype,))
    lib = _native.load()
    out = torch.empty((m, n), dtype=out_dtype, device=q.device)
    with torch.cuda.device(q.device):
        ws, size = _workspace(lib, q, q_pitch, weight, w_pitch, m, n, k, 0)
        _native.check(lib.hb_int8_matmul(
            _ptr(q), q_pitch, _ptr(scales), _ptr(weight), w_pitch, _ptr(weight_scales), _ptr(bias), int(bool(relu)), m, n, k,
            _ptr(out), _TYPES[out_dtype], n, _ptr(ws), size, _stream(q.device)))
    return out


def int8_matmul_quantized(q, scales, weight, weight_scales, bias=None, relu=False):
    """quantize_rows(int8_matmul(...)) of the float32 product, bit for bit, as (int8 rows, scales); with up to 1,024 output
    channels the product does not go through memory."""
    q_pitch, w_pitch, m, n, k = _product_arguments(q, scales, weight, weight_scales, bias)
    if n < 1:
        raise ValueError("weight must have at least one row")
    lib = _native.load()
    out = _rows_of_bytes(m, n, q.device)
    out_scales = torch.empty((m,), dtype=torch.float32, device=q.device)
    with torch.cuda.device(q.device):
        ws, size = _workspace(lib, q, q_pitch, weight, w_pitch, m, n, k, 1)
        _native.check(lib.hb_int8_matmul_quantized(
            _ptr(q), q_pitch, _ptr(scales), _ptr(weight), w_pitch, _ptr(weight_scales), _ptr(bias), int(bool(relu)), m, n, k,
            _ptr(out), (n + 15) // 16 * 16, _ptr(out_scales), _ptr(ws), size, _stream(q.device)))
    return out, out_scales


def orthogonalize(update, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """The update of a weight matrix, or of a batch of equal ones ([..., rows, cols], contiguous), with its singular values driven
    towards one by Newton-Schulz steps: X = update / (|update|_F + eps), then `steps` times X <- (a I + b A + c A^2) X with
    A = X X^T and (a, b, c) = coefficients.  Same shape and dtype as the update.

    float32 and float16 updates are multiplied in three half-precision products each (22-bit operands), bfloat16 ones in one
    (11-bit operands, float32 sums), so that the result's own rounding is the larger error.  Elements of the result smaller than 2^-32 are lost; an update with an infinity or a NaN
    gives NaN everywhere.  Coefficients that would let singular values grow beyond 12 are refused."""
    if not isinstance(update, torch.Tensor) or not update.is_cuda:
        raise TypeError("update must be a CUDA tensor")
    if update.dtype not in _TYPES:
        raise TypeError("update must have dtype float32, bfloat16 or float16, got %s" % update.dtype)
    if update.ndim < 2:
        raise ValueError("update must be a matrix or a batch of matrices")
    if not update.is_contiguous():
        raise ValueError("update must be contiguous")
    if len(coefficients) != 3:
        raise ValueError("coefficients must be three numbers")
    rows, cols = update.shape[-2:]
    batch = update[..., 0, 0].numel() if rows and cols else 0
    out = torch.empty_like(update)
    lib = _native.load()
    split = int(update.dtype != torch.bfloat16)
    with torch.cuda.device(update.device):
        size = lib.hb_orthogonalize_workspace_bytes(batch, rows, cols, split)
        ws = torch.empty((size,), dtype=torch.uint8, device=update.device)
        _native.check(lib.hb_orthogonalize(
            _ptr(update), _TYPES[update.dtype], batch, rows, cols, cols, rows * cols, int(steps),
            (ctypes.c_double * 3)(*coefficients), float(eps), split, _ptr(out), cols, rows * cols, _ptr(ws), size,
            _stream(update.device)))
    return out


def check_status():
    """Synchronises the current GPU and raises if a launch of this module gave up on a bounded device wait (reported once)."""
    code = ctypes.c_int32(0)
    _native.check(_native.load().hb_dense_status(ctypes.byref(code)))
