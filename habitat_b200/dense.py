"""Dense layers in 8-bit integers, and orthogonalised weight updates.

* `quantize_rows`, `int8_matmul`, `int8_matmul_quantized`: rows (queries, tokens) in 8-bit integers with one scale each,
  times 8-bit weights with one scale per output channel.  `RuntimePredictor(precision="int8")` runs on them.
* `orthogonalize`: the update of a weight matrix made nearly orthogonal by Newton-Schulz steps.
  `RuntimePredictor.update_hidden` steps the predictors' hidden layers with it.

All take CUDA tensors, queue their work on the current stream without synchronising, allocate results and workspaces
through torch, and run in the library's sm_100a kernels (habitat_b200/csrc/dense_int8.cu, orthogonalize.cu).  The first
call on a GPU sets up a status word there: make it before a stream capture.  Results carry no gradient, whatever the
arguments require.
"""
import ctypes

import torch

from habitat_b200 import _native

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_rows(t, dtypes, name, device=None):
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
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("%s must have rows that do not overlap" % name)


def _check_vector(t, n, name, device):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype != torch.float32:
        raise TypeError("%s must have dtype torch.float32, got %s" % (name, t.dtype))
    if t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError("%s must be a contiguous vector of %d values" % (name, n))


def quantize_rows(x):
    """Rows of a float32, bfloat16 or float16 matrix in 8-bit integers: (q [rows, cols] int8, scales [rows] float32), so that
    q[i, j] * scales[i] is x[i, j] to within half a scale.  In float32: scale = max |x| / 127, q = rint(x * (127 / max |x|)),
    ties to even.  Rows of zeros (magnitudes below 2^-119, whose scale would be subnormal) get the scale 0, rows with an infinity
    or a NaN zeros and the scale NaN.  q's rows start on 16-byte boundaries, as the products want them."""
    res = _native.binding().quantize_rows(x)
    if res is None:
        _check_rows(x, tuple(_TYPES), "x")
        raise ValueError("x must have at least one column")
    return res


def _check_product(q, scales, weight, weight_scales, bias):
    _check_rows(q, (torch.int8,), "q")
    _check_rows(weight, (torch.int8,), "weight", q.device)
    k = q.shape[1]
    if weight.shape[1] != k:
        raise ValueError("q has %d columns, weight has %d" % (k, weight.shape[1]))
    if not 1 <= k <= 131071:
        raise ValueError("the rows have 1 to 131071 columns (the sums are 32-bit integers), not %d" % k)
    _check_vector(scales, q.shape[0], "scales", q.device)
    _check_vector(weight_scales, weight.shape[0], "weight_scales", q.device)
    if bias is not None:
        _check_vector(bias, weight.shape[0], "bias", q.device)
    raise ValueError("weight must have at least one row")


def int8_matmul(q, scales, weight, weight_scales, bias=None, relu=False, out_dtype=torch.float32):
    """q [M, K] int8 with scales [M] times weight [N, K] int8 with weight_scales [N], plus bias [N] float32, then ReLU: [M, N] in
    out_dtype (float32, bfloat16, float16).  The integer sums are exact; (sum * weight scale) * scale + bias in float32, then one
    rounding to out_dtype.  Rows may start anywhere; those that do not start on 16-byte boundaries are copied first."""
    if out_dtype not in _TYPES:
        raise TypeError("out_dtype must be float32, bfloat16 or float16, got %s" % (out_dtype,))
    res = _native.binding().int8_product(q, scales, weight, weight_scales, bias, relu, _TYPES[out_dtype])
    if res is None:
        _check_product(q, scales, weight, weight_scales, bias)
    return res


def int8_matmul_quantized(q, scales, weight, weight_scales, bias=None, relu=False):
    """quantize_rows(int8_matmul(...)) of the float32 product, bit for bit, as (int8 rows, scales); with up to 1,024 output
    channels the product of large batches does not go through memory."""
    res = _native.binding().int8_product(q, scales, weight, weight_scales, bias, relu, -1)
    if res is None:
        _check_product(q, scales, weight, weight_scales, bias)
    return res


def orthogonalize(update, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, operand_bits=22):
    """The update of a weight matrix, or of a batch of equal ones ([..., rows, cols], contiguous), with its singular values driven
    towards one by Newton-Schulz steps: X = update / (|update|_F + eps), then `steps` times X <- (a I + b A + c A^2) X with
    A = X X^T and (a, b, c) = coefficients.  Same shape and dtype as the update.

    operand_bits: what X, A and B = a I + b A + c A^2 are held in between the products.  22: as pairs of half-precision numbers, three
    products for each one of the formula, close to float32 for updates of all three types.  11: as single ones, a third of the
    products; bfloat16 results are then off by 2.0e-3 instead of the 1.7e-3 that their own rounding is (2-norm).  The sums are
    float32 either way.  With a shorter side of up to 32 everything is float64, whatever operand_bits.  Elements of the result
    smaller than 2^-32 may be lost; an update with an infinity or a NaN gives NaN everywhere.  Coefficients that would let singular
    values grow beyond 12 are refused."""
    if operand_bits not in (11, 22):
        raise ValueError("operand_bits must be 22 or 11, got %r" % (operand_bits,))
    a, b, c = coefficients
    res = _native.binding().orthogonalize(update, steps, a, b, c, eps, operand_bits == 22)
    if res is None:
        if not isinstance(update, torch.Tensor) or not update.is_cuda:
            raise TypeError("update must be a CUDA tensor")
        if update.dtype not in _TYPES:
            raise TypeError("update must have dtype float32, bfloat16 or float16, got %s" % update.dtype)
        if update.ndim < 2:
            raise ValueError("update must be a matrix or a batch of matrices")
        raise ValueError("update must be contiguous")
    return res


def check_status():
    """Synchronises the current GPU and raises if a launch of this module gave up on a bounded device wait.  The calls above raise for
    that, too, without synchronising.  Each thread is told once, whichever thread launched it."""
    code = ctypes.c_int32(0)
    _native.check(_native.load().hb_dense_status(ctypes.byref(code)))


def failures(synchronise=False):
    """How often a launch of this module is known to have given up on the current GPU.  Results are good if the count from before their
    calls is still the one that `failures(synchronise=True)` gives behind them, whichever thread was told in between."""
    count = ctypes.c_int64(0)
    _native.check(_native.load().hb_dense_failures(int(synchronise), ctypes.byref(count)))
    return count.value


def check_since(count):
    """Synchronises and raises if a launch has given up since `failures` gave `count`."""
    if failures(synchronise=True) != count:
        check_status()            # raises unless this thread has been told by another call
        raise _native.HabitatNativeError(_native.HB_ERR_DEVICE_TIMEOUT, "a dense-layer launch gave up on a bounded wait")
