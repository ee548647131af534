"""The dense-layer operators against their definitions.

8-bit layers: the integer sums are exact and every float32 operation of the definition is rounded on its own, so results
are compared bit for bit with numpy.  Orthogonalised updates are compared with the formula in 64 bits; the tolerance is worked
out from the 64-bit iterates (`_newton_schulz`).
"""
import ctypes

import numpy as np
import pytest
import torch

from habitat_b200 import _native, dense

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# -- quantisation -------------------------------------------------------------

def _rows(rows, cols, seed, dtype=torch.float32):
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, cols)) * np.exp(2 * g.standard_normal((rows, 1)))
    x[::3] = np.maximum(x[::3], 0.0)
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


def _quantized(x):
    """The definition in numpy float32: x [rows, cols] float32 -> int8, float32."""
    amax = np.abs(x).max(axis=1)
    bad, zero = ~np.isfinite(amax), amax < np.float32(2.0 ** -119)
    with np.errstate(all="ignore"):
        inverse = np.where(bad | zero, np.float32(0), np.float32(127) / amax)
        scale = np.where(bad, np.float32(np.nan), np.where(zero, np.float32(0), amax / np.float32(127)))
        q = np.rint(x * inverse[:, None])
    q[bad] = 0
    return q.astype(np.int8), scale.astype(np.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 1024), (3, 7), (9, 500), (33, 777), (5, 1025), (8, 2048), (7, 2056), (2, 8192), (2, 16384),
                                        (3, 16392), (2, 40000), (700, 64)])
def test_quantize_rows(rows, cols, dtype):
    x = _rows(rows, cols, rows * 1000 + cols, dtype)
    q, s = dense.quantize_rows(x)
    want_q, want_s = _quantized(x.float().cpu().numpy())
    assert q.shape == (rows, cols) and q.stride(0) % 16 == 0
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


def test_quantize_rows_with_a_pitch_and_an_odd_start():
    big = _rows(20, 300, 5)
    for view in (big[:, :256], big[:, 1:258], big[::2, 4:260], big[3:4, 3:]):
        q, s = dense.quantize_rows(view)
        want_q, want_s = _quantized(view.cpu().numpy())
        assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)


def test_quantize_rows_extreme_values():
    x = _rows(12, 130, 6)
    x[0] = 0.0
    x[1, 5] = float("inf")
    x[2, 129] = float("nan")
    x[3, 0] = float("-inf")
    x[4] *= 1e-38 / x[4].abs().max()              # counts as zeros
    x[5] *= 3e38 / x[5].abs().max()
    x[6] *= 2.0 ** -118 / x[6].abs().max()        # the smallest that do not
    x[7] = 0.0
    x[7, 0] = 127.0
    x[7, 1:6] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5])     # ties go to even
    x[8] = -0.0
    q, s = dense.quantize_rows(x)
    want_q, want_s = _quantized(x.cpu().numpy())
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert q[7, 1:6].tolist() == [0, 2, 2, 0, -2]
    assert torch.isnan(s[1:4]).all() and not q[1:5].any()


def test_quantize_no_rows():
    q, s = dense.quantize_rows(torch.empty((0, 5), device="cuda"))
    assert q.shape == (0, 5) and s.shape == (0,)


# -- products -----------------------------------------------------------------

def _layer(m, n, k, seed, bias=True):
    g = np.random.default_rng(seed)
    q = g.integers(-127, 128, size=(m, k), dtype=np.int8)
    w = g.integers(-128, 128, size=(n, k), dtype=np.int8)
    s = np.exp(g.standard_normal(m)).astype(np.float32)
    ws = (np.exp(0.3 * g.standard_normal(n)) / 127 / np.sqrt(k)).astype(np.float32)
    b = g.standard_normal(n).astype(np.float32) * 20 if bias else None
    return q, s, w, ws, b


def _product(q, s, w, ws, b, relu):
    acc = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)      # whole numbers below 2^31: exact sums
    with np.errstate(all="ignore"):
        y = acc * ws * s[:, None]
        if b is not None:
            y = y + b
    return np.maximum(y, np.float32(0)) if relu else y      # numpy's maximum keeps NaN


def _cuda(*arrays):
    return [None if a is None else torch.from_numpy(a).cuda() for a in arrays]


SHAPES = [(1, 1, 1), (1, 1024, 1024), (2, 3, 16), (3, 5, 17), (7, 64, 33), (16, 100, 128), (17, 31, 129), (127, 1024, 1024), (128, 65, 500),
          (129, 128, 1000), (255, 257, 256), (257, 300, 777), (300, 1003, 96), (1000, 24, 2000), (1, 5000, 640), (5, 130, 8192), (2049, 512, 64)]


@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("out", DTYPES)
def test_int8_matmul(m, n, k, out):
    relu, bias = (m + n) % 2 == 0, k % 2 == 0
    arrays = _layer(m, n, k, m + 3 * n + 7 * k, bias)
    got = dense.int8_matmul(*_cuda(*arrays[:4]), bias=_cuda(arrays[4])[0], relu=relu, out_dtype=out)
    want = torch.from_numpy(_product(*arrays, relu)).to(out)
    dense.check_status()
    assert got.dtype == out and got.shape == (m, n)
    assert torch.equal(got.cpu(), want)


def test_int8_matmul_sums_at_the_limits():
    k = 131071                                                     # 128 * 128 * K is just below 2^31
    q, w = torch.full((3, k), -128, dtype=torch.int8, device="cuda"), torch.full((70, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = torch.ones((70,), device="cuda")
    got = dense.int8_matmul(q, one[:3], w, one)
    assert got[:, 0].tolist() == [float(np.float32(128 * 128 * k))] * 3
    assert got[:, 1].tolist() == [float(np.float32(-128 * 127 * k))] * 3


def test_int8_matmul_scales_that_are_not_finite():
    q, s, w, ws, b = _layer(40, 70, 64, 3)
    s[3], s[7], ws[5], b[9], b[10] = np.nan, np.inf, np.nan, np.inf, np.nan
    s[11] = 0.0
    for relu in (False, True):
        got = dense.int8_matmul(*_cuda(q, s, w, ws), bias=_cuda(b)[0], relu=relu).cpu().numpy()
        want = _product(q, s, w, ws, b, relu)
        assert np.array_equal(got, want, equal_nan=True)
        assert np.isnan(got[3]).all()


@pytest.mark.parametrize("m", [1, 40])
def test_int8_matmul_rows_that_start_anywhere(m):
    q, s, w, ws, b = _layer(m, 50, 100, 9)
    want = torch.from_numpy(_product(q, s, w, ws, b, False))
    big = torch.zeros((m + 50, 260), dtype=torch.int8, device="cuda")
    for at in (0, 1, 3, 16, 37, 159):
        big[:m, at:at + 100], big[m:, at:at + 100] = torch.from_numpy(q).cuda(), torch.from_numpy(w).cuda()
        got = dense.int8_matmul(big[:m, at:at + 100], *_cuda(s), big[m:, at:at + 100], *_cuda(ws, b))
        assert torch.equal(got.cpu(), want), at
    padded = torch.zeros((m + 50, 112), dtype=torch.int8, device="cuda")
    padded[:m, :100], padded[m:, :100] = torch.from_numpy(q).cuda(), torch.from_numpy(w).cuda()
    padded[:, 100:] = 77                                           # what lies behind a row does not count
    got = dense.int8_matmul(padded[:m, :100], *_cuda(s), padded[m:, :100], *_cuda(ws, b))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("k", [1, 15, 16, 17, 40, 63, 64, 65, 200, 777])
def test_int8_matmul_few_rows_of_weights_that_start_anywhere(k):
    """The kernel for up to 16 rows reads unaligned weights as they are, in whole words: every start, every end."""
    g = np.random.default_rng(k)
    for m in (1, 9):
        q, s, w, ws, b = _layer(m, 37, k, 11 + m)
        want = torch.from_numpy(_product(q, s, w, ws, b, True))
        for start in range(5):
            room = torch.from_numpy(g.integers(-128, 128, size=37 * (k + 3) + 8, dtype=np.int8)).cuda()
            view = room[start:start + 37 * (k + 3)].view(37, k + 3)[:, :k]
            view.copy_(torch.from_numpy(w))
            got = dense.int8_matmul(*_cuda(q, s), view, *_cuda(ws, b), relu=True)
            assert torch.equal(got.cpu(), want), (m, start)
            got_q, got_s = dense.int8_matmul_quantized(*_cuda(q, s), view, *_cuda(ws, b), relu=True)
            want_q, want_s = _quantized(want.numpy())
            assert np.array_equal(got_q.cpu().numpy(), want_q) and np.array_equal(got_s.cpu().numpy(), want_s)


@pytest.mark.parametrize("m, k", [(1, 3000), (16, 2100), (17, 300), (512, 300), (513, 300), (300, 3000)])
def test_int8_matmul_quantized_in_one_launch_and_in_two(m, k):
    arrays = _layer(m, 900, k, m + k)
    q, s = dense.int8_matmul_quantized(*_cuda(*arrays[:4]), bias=_cuda(arrays[4])[0], relu=True)
    want_q, want_s = _quantized(_product(*arrays, True))
    assert np.array_equal(s.cpu().numpy(), want_s) and np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("m, n, k", [(19000, 1000, 200), (18433, 1024, 1024), (38000, 300, 77), (76000, 200, 64)])
def test_int8_matmul_long_batches(m, n, k):
    """Weights that stay in shared memory for all of an SM pair's rows."""
    arrays = _layer(m, n, k, m + n)
    got = dense.int8_matmul(*_cuda(*arrays[:4]), bias=_cuda(arrays[4])[0], relu=True, out_dtype=torch.bfloat16)
    dense.check_status()
    assert torch.equal(got.cpu(), torch.from_numpy(_product(*arrays, True)).to(torch.bfloat16))


@pytest.mark.parametrize("m, n, k", [(15361, 1000, 200), (20000, 1024, 1024), (21000, 700, 90), (31000, 500, 64), (62000, 130, 40)])
def test_int8_matmul_quantized_long_batches(m, n, k):
    arrays = _layer(m, n, k, m + n)
    q, s = dense.int8_matmul_quantized(*_cuda(*arrays[:4]), bias=_cuda(arrays[4])[0], relu=True)
    want_q, want_s = _quantized(_product(*arrays, True))
    dense.check_status()
    assert np.array_equal(s.cpu().numpy(), want_s) and np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("m", [5, 100, 700])
@pytest.mark.parametrize("relu", [False, True])
def test_int8_matmul_far_below_zero(m, relu):
    """Results that ReLU drops, by however much they are below zero, and zeros of either sign, bit for bit."""
    q, s, w, ws, b = _layer(m, 300, 96, m)
    b[::7], b[3::11] = np.float32(-1e30), np.float32(-3e7)
    if relu:
        b[5::13] = -np.inf
    q[m // 2], b[1::9] = 0, np.float32(-0.0)
    want = _product(q, s, w, ws, b, relu)
    got_q, got_s = dense.int8_matmul_quantized(*_cuda(q, s, w, ws, b), relu=relu)
    want_q, want_s = _quantized(want)
    assert np.array_equal(got_s.cpu().numpy(), want_s) and np.array_equal(got_q.cpu().numpy(), want_q)
    for dtype, bits in ((torch.float32, torch.int32), (torch.bfloat16, torch.int16), (torch.float16, torch.int16)):
        got = dense.int8_matmul(*_cuda(q, s, w, ws, b), relu=relu, out_dtype=dtype)
        assert torch.equal(got.cpu().view(bits), torch.from_numpy(want + np.float32(0) if relu else want).to(dtype).view(bits))


def test_int8_matmul_of_nothing():
    q, s, w, ws, b = _cuda(*_layer(4, 6, 16, 1))
    assert dense.int8_matmul(q[:0], s[:0], w, ws, b).shape == (0, 6)
    assert dense.int8_matmul(q, s, w[:0], ws[:0], b[:0]).shape == (4, 0)


def test_product_arguments_are_checked():
    q, s, w, ws, b = _cuda(*_layer(4, 6, 16, 1))
    with pytest.raises(ValueError, match="columns"):
        dense.int8_matmul(q, s, w[:, :8].contiguous(), ws)
    with pytest.raises(ValueError, match="contiguous rows"):
        dense.int8_matmul(torch.zeros((16, 4), dtype=torch.int8, device="cuda").t(), s, w, ws)
    with pytest.raises(ValueError, match="overlap"):
        dense.int8_matmul(q[:1].expand(4, 16), s, w, ws)
    with pytest.raises(ValueError, match="weight_scales"):
        dense.int8_matmul(q, s, w, ws[:5])
    with pytest.raises(TypeError, match="bias"):
        dense.int8_matmul(q, s, w, ws, b.double())
    with pytest.raises(TypeError, match="out_dtype"):
        dense.int8_matmul(q, s, w, ws, out_dtype=torch.float64)
    with pytest.raises(TypeError, match="int8"):
        dense.int8_matmul(q.short(), s, w, ws)
    with pytest.raises(ValueError, match="scales"):
        dense.int8_matmul_quantized(q, s[:3], w, ws)
    with pytest.raises(ValueError, match="at least one column"):
        dense.quantize_rows(torch.empty((3, 0), device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        dense.orthogonalize(torch.zeros((4, 6), device="cuda").t())
    with pytest.raises(TypeError, match="dtype"):
        dense.orthogonalize(torch.zeros((4, 6), device="cuda", dtype=torch.float64))
    with pytest.raises(_native.HabitatNativeError, match="grow"):
        dense.orthogonalize(torch.zeros((4, 6), device="cuda"), coefficients=(4.0, 0.0, 0.0))


@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 1024, 1024), (3, 5, 17), (17, 256, 64), (130, 257, 128), (300, 500, 500), (700, 700, 33), (256, 768, 100),
                                     (2500, 1000, 200), (40, 1025, 70), (9000, 1024, 64)])
def test_int8_matmul_quantized(m, n, k):
    arrays = _layer(m, n, k, m + n + k)
    q, s = dense.int8_matmul_quantized(*_cuda(*arrays[:4]), bias=_cuda(arrays[4])[0], relu=k % 3 == 1)
    want_q, want_s = _quantized(_product(*arrays, k % 3 == 1))
    dense.check_status()
    assert q.shape == (m, n) and q.stride(0) % 16 == 0
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


def test_int8_matmul_quantized_rows_that_are_not_finite_or_zero():
    q, s, w, ws, b = _layer(300, 600, 64, 4, bias=False)
    s[3], s[5], s[280] = np.nan, 0.0, 1e-38
    got_q, got_s = dense.int8_matmul_quantized(*_cuda(q, s, w, ws))
    want_q, want_s = _quantized(_product(q, s, w, ws, None, False))
    assert np.array_equal(got_s.cpu().numpy(), want_s, equal_nan=True)
    assert np.array_equal(got_q.cpu().numpy(), want_q)
    assert torch.isnan(got_s[3]) and not got_q[3].any()


@pytest.mark.parametrize("m, width, layers, dtype", [(1, 1024, 8, torch.float32), (37, 500, 4, torch.bfloat16), (1500, 1024, 3, torch.float32),
                                                     (260, 1100, 3, torch.float16)])
def test_stack_of_layers(m, width, layers, dtype):
    """As a network uses them: rows quantised once, handed from layer to layer in 8 bits, the last result in 16."""
    x = _rows(m, width, m + width, dtype)
    q, s = dense.quantize_rows(x)
    y = x.float().cpu().numpy()
    for i in range(layers):
        _, _, w, ws, b = _layer(1, width, width, i)
        wt, wst, bt = _cuda(w, ws, b)
        if i < layers - 1:
            q, s = dense.int8_matmul_quantized(q, s, wt, wst, bias=bt, relu=True)
        else:
            got = dense.int8_matmul(q, s, wt, wst, bias=bt, relu=True, out_dtype=torch.bfloat16)
        y = _product(*_quantized(y), w, ws, b, True)
    assert torch.equal(got.cpu(), torch.from_numpy(y).to(torch.bfloat16))


# -- orthogonalised updates ---------------------------------------------------

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _newton_schulz(g, steps, coefficients, eps, unit):
    """The formula in 64 bits, and how far a result whose operands are rounded to within `unit` may be from it (2-norms,
    relative).  Each step rounds X, A and B once: four units of the iterate's norm with what A's rounding does to B, and what
    is off grows by at most the polynomial's largest slope in each later step."""
    a, b, c = coefficients
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT if flip else x
    t = torch.linspace(0, 1.3, 1001, dtype=torch.float64)
    slope = float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max().clamp_min(1.0))
    off = 0.0
    for _ in range(steps):
        off = (off + 4 * unit * float(x.norm())) * min(slope, max(abs(a), 1.0))
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if flip else x), off / max(float(x.norm()), 1e-300)


def _update(shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    r, c = shape[-2:]
    k = max(1, min(r, c) // 8)
    u, v = torch.randn(shape[:-1] + (k,), generator=g), torch.randn(shape[:-2] + (k, c), generator=g)
    return (1e-3 * (u @ v / k ** 0.5 + torch.randn(shape, generator=g))).to(dtype).cuda()


def _check(update, got, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    unit = 2.0 ** -12 if update.dtype == torch.bfloat16 else 2.0 ** -22
    want, off = _newton_schulz(update.cpu(), steps, coefficients, eps, unit)
    assert got.shape == update.shape and got.dtype == update.dtype
    # and the result's own rounding, and float32 sums over up to K terms (random: sqrt(K) / 2^24)
    tol = off + torch.finfo(update.dtype).eps / 2 + max(update.shape[-2:]) ** 0.5 * 2.0 ** -24 * 4
    err = float((got.double().cpu() - want).norm() / want.norm())
    assert err <= tol, (err, tol)


ORTHO_SHAPES = [(1, 1), (1, 9), (9, 1), (2, 3), (12, 1024), (1024, 12), (63, 65), (64, 64), (128, 128), (129, 200), (256, 256), (257, 255), (300, 1000),
                (777, 300), (3, 40, 70), (2, 2, 130, 33), (8, 256, 512), (5, 520, 260), (1024, 1024)]


@pytest.mark.parametrize("shape", ORTHO_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_orthogonalize(shape, dtype):
    update = _update(shape, sum(shape), dtype)
    got = dense.orthogonalize(update)
    dense.check_status()
    _check(update, got)


# the shorter side around what is kept on chip (32, 128), the longer one around what a cluster holds of it
@pytest.mark.parametrize("shape", [(32, 33), (33, 32), (32, 10048), (32, 10400), (31, 30000), (1, 70000), (5, 40000), (20000, 20), (128, 129), (129, 128),
                                   (128, 3300), (128, 6000), (9000, 100), (70, 14000), (130, 9000), (2, 160, 5000), (300, 256), (520, 700)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize_long_and_short_sides(shape, dtype):
    update = _update(shape, sum(shape), dtype)
    _check(update, dense.orthogonalize(update))


# shorter sides kept on chip, with rows that start on 16, 8, 4 and 2 bytes
@pytest.mark.parametrize("shape", [(64, 128), (100, 100), (90, 102), (40, 101), (2, 64, 100), (3, 50, 102), (128, 1004), (60, 2002), (128, 6000), (100, 100, 44)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_orthogonalize_on_chip(shape, dtype):
    update = _update(shape, sum(shape), dtype)
    got = dense.orthogonalize(update)
    _check(update, got)
    assert torch.equal(got, dense.orthogonalize(update))


# single matrices, whose products are split along K over the pairs of a cluster or over launches, with slots that do not divide by the shares
@pytest.mark.parametrize("shape", [(400, 400), (768, 768), (777, 1000), (1000, 777), (513, 1100), (900, 900), (300, 3000), (150, 8000), (2, 650, 700),
                                   (4, 510, 520), (1200, 1100)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_orthogonalize_single_matrices(shape, dtype):
    update = _update(shape, sum(shape), dtype)
    got = dense.orthogonalize(update)
    _check(update, got)
    for _ in range(3):
        assert torch.equal(got, dense.orthogonalize(update))


# read in pieces of eight elements or one by one: rows that are no multiple of eight, that start on any element, and both
@pytest.mark.parametrize("shape", [(129, 204), (131, 260), (129, 1030), (3, 131, 204), (1030, 129), (131, 2056)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_orthogonalize_updates_that_start_anywhere(shape, dtype, shift):
    update = _update(shape, sum(shape), dtype)
    flat = torch.full((shift + update.numel(),), float("nan"), dtype=dtype, device="cuda")
    flat[shift:] = update.flatten()
    _check(update, dense.orthogonalize(flat[shift:].view(shape)))


# blocks of 128 rows per side, and enough matrices for tiles of two such blocks
@pytest.mark.parametrize("blocks, batch", [(2, 40), (3, 30), (4, 20), (5, 12), (6, 10), (7, 8), (8, 8), (9, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize_batches_of_equal_updates(blocks, batch, dtype):
    update = _update((128 * blocks - 37, 128 * blocks - 16), blocks, dtype)
    got = dense.orthogonalize(update.expand((batch,) + update.shape).contiguous())
    _check(update, got[0])
    for x in got:
        assert torch.equal(x, got[0])


@pytest.mark.parametrize("steps, coefficients", [(1, COEFFICIENTS), (2, COEFFICIENTS), (3, (1.5, -0.5, 0.0)), (10, (1.875, -1.25, 0.375))])
def test_orthogonalize_steps_and_coefficients(steps, coefficients):
    for dtype in (torch.float32, torch.bfloat16):
        update = _update((100, 180), steps, dtype)
        _check(update, dense.orthogonalize(update, steps=steps, coefficients=coefficients), steps, coefficients)


@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e-3, 1e4, 1e18, 1e36])
def test_orthogonalize_sizes_of_updates(scale):
    g = _update((90, 140), 3, torch.float32) * 1e3 * scale      # (1e3 * 1e36 is no float32)
    for eps in (0.0, 1e-7):
        if scale < 1e-20 and eps:
            continue            # next to eps nothing is left of it, see below
        _check(g, dense.orthogonalize(g, eps=eps), eps=eps)


def test_orthogonalize_zero_and_not_finite():
    z = torch.zeros((2, 30, 50), device="cuda")
    assert not dense.orthogonalize(z).any()
    z[1, 3, 4] = float("nan")
    got = dense.orthogonalize(z)
    assert not got[0].any() and torch.isnan(got[1]).all()
    z[1, 3, 4] = float("inf")
    assert torch.isnan(dense.orthogonalize(z)[1]).all()
    tiny = _update((30, 50), 1, torch.float32) * 1e-20          # far below eps: no larger than its share of it
    assert float(dense.orthogonalize(tiny).abs().max()) < 1e-9


def test_orthogonalize_of_nothing():
    for shape in ((0, 5), (5, 0), (0, 3, 4)):
        assert dense.orthogonalize(torch.empty(shape, device="cuda")).shape == shape


def test_orthogonalize_makes_orthogonal():
    """What it is for: singular values within the band the default coefficients leave (0.67 to 1.21), from spread ones."""
    for dtype in DTYPES:
        s = torch.linalg.svdvals(dense.orthogonalize(_update((200, 300), 2, dtype)).float().cpu())
        assert 0.6 < float(s.min()) and float(s.max()) < 1.3


# -- streams, graphs, errors --------------------------------------------------

def test_on_another_stream_and_in_a_graph():
    q, s, w, ws, b = _cuda(*_layer(300, 500, 100, 2))
    x, u = _rows(300, 100, 3), _update((130, 70), 4, torch.float32)

    def all_of_them():
        qq, ss = dense.quantize_rows(x)
        q2, s2 = dense.int8_matmul_quantized(qq, ss, w, ws, b, relu=True)
        return dense.int8_matmul(q2, s2, w.t().contiguous(), ss[:100], out_dtype=torch.bfloat16), dense.orthogonalize(u)
    want = all_of_them()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of_them()
    side.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(all_of_them())
        graphs.append(g)
    x.mul_(-3.0)
    u.mul_(0.5).add_(1e-4)
    want = all_of_them()
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, e) for a, e in zip(out, want))


def test_first_use_of_a_kernel_inside_a_capture():
    """One call sets up the GPU's status word; whatever kernel a later capture is the first to use may be captured."""
    code = """
import torch
from habitat_b200 import dense
w, s = torch.ones((600, 64), dtype=torch.int8, device="cuda"), torch.ones((600,), device="cuda")
q, qs = dense.quantize_rows(torch.ones((1, 64), device="cuda"))
dense.int8_matmul(q, qs, w, s)
x, u, v, t = (torch.randn(n, device="cuda") for n in ((700, 64), (300, 200), (100, 90), (20, 30)))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = dense.quantize_rows(x)
    b = dense.int8_matmul_quantized(*a, w, s)
    c = dense.int8_matmul(*a, w, s, out_dtype=torch.bfloat16)
    d = [dense.orthogonalize(y) for y in (u, v, t)]
g.replay()
torch.cuda.synchronize()
assert torch.equal(c, dense.int8_matmul(*dense.quantize_rows(x), w, s, out_dtype=torch.bfloat16))
assert all(torch.equal(y, dense.orthogonalize(z)) for y, z in zip(d, (u, v, t)))
assert torch.equal(b[0], dense.int8_matmul_quantized(*a, w, s)[0])
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_streams_at_once_and_repeated_calls_agree():
    a, c = _cuda(*_layer(2000, 1024, 1024, 5)), _update((512, 700), 6, torch.bfloat16)
    want = dense.int8_matmul(*a), dense.int8_matmul_quantized(*a)[0], dense.orthogonalize(c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = []
        for st in streams:
            with torch.cuda.stream(st):
                got.append((dense.int8_matmul(*a), dense.int8_matmul_quantized(*a)[0], dense.orthogonalize(c)))
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(x, y) for x, y in zip(g, want))


def test_clusters_of_several_calls_and_graphs_at_once():
    updates = [_update((777, 1000), 1, torch.float16), _update((100, 4000), 2, torch.float32), _update((3, 300, 320), 3, torch.float32),
               _update((150, 5000), 4, torch.bfloat16)]
    layer = _cuda(*_layer(1500, 700, 300, 5))
    run = lambda: [dense.orthogonalize(u) for u in updates] + list(dense.int8_matmul_quantized(*layer, relu=True))
    want = run()
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = []
        for st in streams[2:]:
            with torch.cuda.stream(st):
                eager.append(run())
        torch.cuda.synchronize()
        for got in results + eager:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    dense.check_status()


def test_a_launch_that_gave_up_is_reported():
    q, s, w, ws, b = _cuda(*_layer(4, 6, 16, 1))
    lib = _native.load()
    _native.check(lib.hb_dense_inject_status(0x511))
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        dense.int8_matmul(q, s, w, ws)
    dense.int8_matmul(q, s, w, ws)                               # reported once
    _native.check(lib.hb_dense_inject_status(0x522))
    with pytest.raises(_native.HabitatNativeError, match="gave up"):
        dense.check_status()
    dense.check_status()


def test_workspaces_that_are_too_small_are_refused():
    q, s, w, ws, b = _cuda(*_layer(4, 6, 17, 1))
    out = torch.empty((4, 6), device="cuda")
    lib, p = _native.load(), lambda t: ctypes.c_void_p(t.data_ptr())
    room = torch.empty((1024,), dtype=torch.uint8, device="cuda")
    for space, size in ((None, 0), (p(room), 511), (ctypes.c_void_p(room.data_ptr() + 16), 512)):
        assert lib.hb_int8_matmul(p(q), 17, p(s), p(w), 17, p(ws), None, 0, 4, 6, 17, p(out), 0, 6, space, size,
                                  _native.current_stream_ptr()) == _native.HB_ERR_INVALID_ARGUMENT
    u = torch.ones((4, 6), device="cuda")
    size = lib.hb_orthogonalize_workspace_bytes(1, 4, 6, 1)
    assert lib.hb_orthogonalize(p(u), 0, 1, 4, 6, 6, 24, 5, (ctypes.c_double * 3)(*COEFFICIENTS), 1e-7, 1, p(u), 6, 24, p(room), size - 1,
                                _native.current_stream_ptr()) == _native.HB_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("shape", [(1, 20, 30), (3, 12, 70), (1, 100, 90), (2, 64, 200), (1, 300, 200), (2, 260, 300), (1, 900, 1000)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("more", [1, 6, 24])
def test_orthogonalize_rows_and_matrices_apart(shape, dtype, more):
    """Through the C interface: pitches and strides, of which nothing else is written to."""
    lib = _native.load()
    batch, rows, cols = shape
    update = _update(shape, sum(shape), dtype)
    kind = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    pitch, stride = cols + more, rows * (cols + more) + 3 * more
    source, out = (torch.full((batch * stride,), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    at = torch.arange(batch, device="cuda")[:, None, None] * stride + torch.arange(rows, device="cuda")[:, None] * pitch + torch.arange(cols, device="cuda")
    source[at] = update
    out.fill_(7.0)
    split = 0 if dtype == torch.bfloat16 else 1
    size = lib.hb_orthogonalize_workspace_bytes(batch, rows, cols, split)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    assert lib.hb_orthogonalize(p(source), kind, batch, rows, cols, pitch, stride, 5, (ctypes.c_double * 3)(*COEFFICIENTS), 1e-7, split, p(out), pitch, stride,
                                p(room), size, None) == 0
    torch.cuda.synchronize()
    dense.check_status()
    got = out[at]
    _check(update, got)
    out[at] = 7.0
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("m, n, k", [(3, 50, 64), (100, 70, 40), (600, 300, 100)])
@pytest.mark.parametrize("more", [1, 4, 8, 16])
def test_int8_matmul_rows_apart(m, n, k, more):
    lib = _native.load()
    arrays = _layer(m, n, k, m)
    q, s, w, ws, b = arrays
    wide_q, wide_w = np.full((m, k + more), 99, np.int8), np.full((n, k + more), -99, np.int8)
    wide_q[:, :k], wide_w[:, :k] = q, w
    dq, ds, dw, dws, db = _cuda(wide_q, s, wide_w, ws, b)
    want = torch.from_numpy(_product(*arrays, True))
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    size = lib.hb_int8_workspace_bytes(p(dq), k + more, p(dw), k + more, m, n, k, 0)
    room = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    for kind, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16)):
        out = torch.full((m, n + more), 7.0, dtype=dtype, device="cuda")
        assert lib.hb_int8_matmul(p(dq), k + more, p(ds), p(dw), k + more, p(dws), p(db), 1, m, n, k, p(out), kind, n + more, p(room), size, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(out[:, :n].cpu(), want.to(dtype)) and bool((out[:, n:] == 7.0).all())
