"""Refusals of the dense-layer operators: everything here ends before a GPU is touched."""
import ctypes

import pytest
import torch

from habitat_b200 import _native, dense

P = ctypes.c_void_p


def _matmul(M=4, N=4, K=16, q_pitch=16, w_pitch=16, q=16, out=16, out_type=0, out_pitch=4, ws=0, ws_bytes=0):
    return _native.load().hb_int8_matmul(P(q), q_pitch, P(16), P(16), w_pitch, P(16), None, 0, M, N, K, P(out), out_type, out_pitch,
                                         P(ws), ws_bytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(M=-1), _native.HB_ERR_INVALID_ARGUMENT), (dict(N=-1), _native.HB_ERR_INVALID_ARGUMENT),
    (dict(K=0), _native.HB_ERR_INVALID_ARGUMENT), (dict(q_pitch=15), _native.HB_ERR_INVALID_ARGUMENT),
    (dict(w_pitch=8), _native.HB_ERR_INVALID_ARGUMENT), (dict(q=0), _native.HB_ERR_INVALID_ARGUMENT),
    (dict(out=0), _native.HB_ERR_INVALID_ARGUMENT), (dict(out_type=3), _native.HB_ERR_INVALID_ARGUMENT),
    (dict(out_type=-1), _native.HB_ERR_INVALID_ARGUMENT), (dict(out_pitch=3), _native.HB_ERR_INVALID_ARGUMENT),
    (dict(K=131072, q_pitch=131072, w_pitch=131072), _native.HB_ERR_TOO_LARGE),
    (dict(M=1 << 31), _native.HB_ERR_TOO_LARGE),
])
def test_product_refuses(bad, status):
    assert _matmul(**bad) == status
    assert b"hb_int8_matmul" in _native.load().hb_last_error()


def test_quantized_product_refuses():
    lib = _native.load()

    def call(N=16, out=16, out_pitch=16):
        return lib.hb_int8_matmul_quantized(P(16), 16, P(16), P(16), 16, P(16), None, 0, 4, N, 16, P(out), out_pitch, P(16), None, 0, None)
    for bad in (dict(out=0), dict(out=24), dict(out_pitch=24, N=16), dict(out_pitch=0), dict(N=0)):
        assert call(**bad) == _native.HB_ERR_INVALID_ARGUMENT


def test_quantisation_refuses():
    lib = _native.load()

    def call(x=16, kind=0, rows=4, cols=16, pitch=16, q=16, q_pitch=16, scales=16):
        return lib.hb_quantize_rows(P(x), kind, rows, cols, pitch, P(q), q_pitch, P(scales), None)
    for bad in (dict(rows=-1), dict(cols=0), dict(pitch=15), dict(q_pitch=15), dict(kind=3), dict(x=0), dict(q=0), dict(scales=0)):
        assert call(**bad) == _native.HB_ERR_INVALID_ARGUMENT
    assert call(rows=1 << 31) == _native.HB_ERR_TOO_LARGE
    assert call(rows=0, x=0, q=0, scales=0) == _native.HB_OK      # nothing to do


def test_workspace_sizes():
    lib = _native.load()
    size = lib.hb_int8_workspace_bytes
    assert size(P(16), 16, P(16), 32, 4, 4, 16, 0) == 0                      # rows on 16-byte boundaries
    assert size(P(17), 16, P(16), 16, 4, 4, 16, 0) == 256                    # q is copied: 4 x 16 bytes, rounded up
    assert size(P(16), 17, P(16), 17, 40, 4, 17, 0) == 40 * 32 + 256         # both are
    assert size(P(16), 16, P(16), 16, 4, 1024, 16, 1) == 0
    assert size(P(16), 16, P(16), 16, 4, 1025, 16, 1) >= 4 * 1025 * 4        # wider rows go through memory
    assert size(P(16), 16, P(16), 16, -1, 4, 16, 0) == -1
    assert lib.hb_orthogonalize_workspace_bytes(1, -1, 2, 0) == -1
    one, two = (lib.hb_orthogonalize_workspace_bytes(3, 70, 50, s) for s in (0, 1))
    assert one >= 2 * 3 * 50 * 70 * 2 + 2 * 3 * 50 * 50 * 2
    assert two > one


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(rows=-1), dict(type=3), dict(pitch=3), dict(out_pitch=3), dict(steps=0), dict(steps=101),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(coefficients=(float("nan"), 0.0, 0.0)), dict(coefficients=(float("inf"), 0.0, 0.0)),
    dict(coefficients=(300.0, 0.0, 0.0)),                # the factor itself
    dict(coefficients=(3.0, 0.0, 0.0)),                  # 3^5
    dict(coefficients=(0.0, -1e30, 1e30)),
])
def test_orthogonalize_refuses(bad):
    a = dict(type=0, batch=1, rows=4, cols=4, pitch=4, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, out_pitch=4)
    a.update(bad)
    status = _native.load().hb_orthogonalize(P(16), a["type"], a["batch"], a["rows"], a["cols"], a["pitch"], 16, a["steps"],
                                             (ctypes.c_double * 3)(*a["coefficients"]), a["eps"], 1, P(16), a["out_pitch"], 16,
                                             None, 0, None)
    assert status == _native.HB_ERR_INVALID_ARGUMENT
    assert b"hb_orthogonalize" in _native.load().hb_last_error()


def test_misaligned_arguments_are_refused():
    lib = _native.load()
    assert _matmul(out=18) == _native.HB_ERR_INVALID_ARGUMENT                  # float32 on a 2-byte boundary
    assert _matmul(out=17, out_type=1) == _native.HB_ERR_INVALID_ARGUMENT
    for at in range(3):
        scales, w_scales, bias = (18 if i == at else 16 for i in range(3))
        assert lib.hb_int8_matmul(P(16), 16, P(scales), P(16), 16, P(w_scales), P(bias), 0, 4, 4, 16, P(16), 0, 4, None, 0,
                                  None) == _native.HB_ERR_INVALID_ARGUMENT
    assert lib.hb_quantize_rows(P(18), 0, 4, 16, 16, P(16), 16, P(16), None) == _native.HB_ERR_INVALID_ARGUMENT
    assert lib.hb_quantize_rows(P(16), 0, 4, 16, 16, P(16), 16, P(18), None) == _native.HB_ERR_INVALID_ARGUMENT
    for misplaced in ((P(17), P(16)), (P(16), P(17))):
        status = lib.hb_int8_mlp_output(misplaced[0], 16, P(16), P(16), P(16), 4, 16, misplaced[1], None)
        assert status == _native.HB_ERR_INVALID_ARGUMENT


def test_predictor_ends_refuse():
    lib = _native.load()

    def put_in(F=4, rows=6, width=64, q=16, pitch=64, Q=3):
        return lib.hb_int8_mlp_input(P(16), F, P(16), P(16), rows, P(16), P(16), P(16), P(16), Q, width, P(q), pitch, P(16), None)
    for bad in (dict(F=0), dict(F=9), dict(rows=0), dict(rows=257), dict(width=0), dict(width=1025), dict(Q=-1)):
        assert put_in(**bad) == _native.HB_ERR_UNSUPPORTED
    for bad in (dict(q=0), dict(q=24), dict(pitch=63), dict(pitch=72)):
        assert put_in(**bad) == _native.HB_ERR_INVALID_ARGUMENT
    assert put_in(Q=0, q=0) == _native.HB_OK


def test_host_tensors_are_refused():
    x = torch.zeros((4, 16))
    q, s = torch.zeros((4, 16), dtype=torch.int8), torch.zeros((4,))
    with pytest.raises(TypeError, match="CUDA"):
        dense.quantize_rows(x)
    with pytest.raises(TypeError, match="CUDA"):
        dense.int8_matmul(q, s, q, s)
    with pytest.raises(TypeError, match="CUDA"):
        dense.int8_matmul_quantized(q, s, q, s)
    with pytest.raises(TypeError, match="CUDA"):
        dense.orthogonalize(x)
