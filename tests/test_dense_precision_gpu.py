"""Orthogonalised updates against the formula in 64 bits, within what their operands' bits account for (tests/newton_schulz.py)."""
import ctypes

import pytest
import torch

from habitat_b200 import _native, dense
from tests import newton_schulz as ns

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# all ways an update can take: float64 matrices (a shorter side of up to 32), one cluster (up to 128), tiles, with K of few of them
# split over clusters and launches; batches, sides exchanged, sizes that end inside tiles
SHAPES = [(1, 9), (12, 1024), (1024, 12), (32, 33), (3, 20, 500), (33, 40), (64, 64), (128, 128), (63, 65), (128, 1024), (128, 6000), (9000, 100), (3, 40, 70),
          (2, 64, 200), (129, 200), (257, 255), (300, 1000), (777, 300), (777, 1000), (150, 8000), (1024, 1024), (8, 256, 512), (520, 2100)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_results_are_as_good_as_their_type(shape, dtype):
    update = ns.update(shape, sum(shape), dtype).cuda()
    got = dense.orthogonalize(update)
    dense.check_status()
    ns.check(got, update, 64 if min(shape[-2:]) <= 32 else 22)


@pytest.mark.parametrize("shape", SHAPES)
def test_bfloat16_results_of_fewer_operand_bits(shape):
    update = ns.update(shape, sum(shape), torch.bfloat16).cuda()
    got = dense.orthogonalize(update, operand_bits=11)
    dense.check_status()
    ns.check(got, update, 64 if min(shape[-2:]) <= 32 else 11)
    if min(shape[-2:]) > 32:
        assert not torch.equal(got, dense.orthogonalize(update))


def test_operand_bits_refused():
    for bad in (0, 16, None, "22"):
        with pytest.raises(ValueError, match="operand_bits"):
            dense.orthogonalize(torch.ones((40, 50), device="cuda"), operand_bits=bad)


# rows and columns that depend on each other, on each way an update can take
@pytest.mark.parametrize("shape, rank", [((12, 1024), 4), ((1024, 12), 4), ((32, 600), 9), ((20, 30), 7), ((2, 8, 50), 1), ((64, 500), 20), ((100, 100), 30), ((300, 260), 90)])
@pytest.mark.parametrize("steps", [5, 15, 30])
def test_dependent_rows(shape, rank, steps):
    """Where singular values are zero the formula leaves zeros, and arithmetic of finitely many bits what rounding makes of them, at
    most the coefficients' largest value (1.21) once it has grown; the others end in their band (0.67 to 1.21)."""
    update = ns.update(shape, steps, rank=rank).cuda()
    got = dense.orthogonalize(update, steps=steps)
    dense.check_status()
    if steps == 5:
        ns.check(got, update, 64 if min(shape[-2:]) <= 32 else 22)
    assert bool(torch.isfinite(got).all())
    assert float(torch.linalg.svdvals(got.double()).max()) < 1.25
    u, s, vt = torch.linalg.svd(update.double(), full_matrices=False)
    inside = torch.linalg.svdvals(u[..., :rank].mT @ got.double() @ vt[..., :rank, :].mT)
    if steps > 5:
        assert 0.6 < float(inside.min()) and float(inside.max()) < 1.25


@pytest.mark.parametrize("shape, rank", [((12, 1024), 4), ((400, 25), 6), ((64, 500), 20), ((200, 300), 50)])
def test_dependent_rows_and_steps_that_converge(shape, rank):
    """(3 x - x^3) / 2 goes to one and stays: U V^T of the update's directions, and at most one elsewhere.  What a step's operands
    (pairs: 2^-22 each, X and B) are off by is left of the last steps', towards one with the slope 0; between equal singular values nothing
    pulls back, so in those directions steps add up: 60 of them, in squares, with sums of 2^-22 as well."""
    update = ns.update(shape, 3, rank=rank).cuda()
    got = dense.orthogonalize(update, steps=60, coefficients=(1.5, -0.5, 0.0)).double()
    assert float(torch.linalg.svdvals(got).max()) < 1.0 + 1e-5
    u, s, vt = torch.linalg.svd(update.double(), full_matrices=False)
    u, vt = u[..., :rank], vt[..., :rank, :]
    inside = u.mT @ got @ vt.mT
    eye = torch.eye(rank, dtype=torch.float64, device="cuda")
    assert float((inside - eye).norm() / rank ** 0.5) < 60 ** 0.5 * 3 * 2.0 ** -22 * 4


@pytest.mark.parametrize("shape", [(12, 1024), (31, 31), (700, 20), (3, 24, 100)])
@pytest.mark.parametrize("steps", [1, 2, 6, 7, 8, 9, 14, 15, 16])
def test_steps_of_float64_matrices(shape, steps):
    update = ns.update(shape, steps).cuda()
    ns.check(dense.orthogonalize(update, steps=steps), update, 64, steps=steps)


@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5), (1.0, 0.0, 0.0), (0.5, 0.25, 0.0)])
@pytest.mark.parametrize("steps", [3, 40, 100])
def test_coefficients_of_float64_matrices(coefficients, steps):
    update = ns.update((16, 200), 5).cuda()
    got = dense.orthogonalize(update, steps=steps, coefficients=coefficients)
    want = ns.steps_of(update, steps, coefficients)
    # slopes of at most one in the end: what is off in the first steps (a^steps of 2^-52, until values are near one) is all there is
    assert float((got.double() - want).norm()) <= float((want.float().double() - want).norm()) * 1.01 + 1e-9 * float(want.norm())


@pytest.mark.parametrize("shape", [(33, 40), (64, 64), (3, 70, 50), (100, 90), (128, 1000), (2000, 120), (300, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_single_parts_of_wider_types(shape, dtype):
    """11 bits of what a float32 or float16 update has, not bfloat16's 8."""
    update = ns.update(shape, sum(shape), dtype).cuda()
    ns.check(dense.orthogonalize(update, operand_bits=11), update, 11)


def test_single_parts_of_the_largest_numbers():
    update = ns.update((60, 200), 6).double()
    update = (update * (0.99999 * torch.finfo(torch.float32).max / update.abs().max())).float().cuda()    # beyond bfloat16's largest when rounded to it
    ns.check(dense.orthogonalize(update, operand_bits=11), update, 11)


@pytest.mark.parametrize("rows, cols", [(64, 200), (100, 100), (300, 260)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_single_parts_through_the_c_interface(rows, cols, dtype):
    lib = _native.load()
    update = ns.update((rows, cols), rows, dtype).cuda()
    out = torch.empty_like(update)
    size = lib.hb_orthogonalize_workspace_bytes(1, rows, cols, 0)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    _native.check(lib.hb_orthogonalize(p(update), DTYPES.index(dtype), 1, rows, cols, cols, rows * cols, 5, (ctypes.c_double * 3)(*ns.COEFFICIENTS), 1e-7, 0, p(out),
                                       cols, rows * cols, p(room), size, _native.current_stream_ptr()))
    ns.check(out, update, 11)
    assert torch.equal(out, dense.orthogonalize(update, operand_bits=11))


def _float32_operations(g):
    a, b, c = ns.COEFFICIENTS
    flip = g.shape[-2] > g.shape[-1]
    x = g.mT if flip else g
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    for _ in range(5):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if flip else x


@pytest.mark.parametrize("shape", [(33, 40), (40, 500), (64, 64), (100, 100), (128, 128), (64, 1024), (128, 1024), (100, 4000), (700, 112), (3, 80, 300)])
def test_float32_results_are_near_what_float32_operations_give(shape):
    """Pairs round at 2^-23, twice float32's 2^-24, and their sums are cut where float32's are rounded, which doubles that error too."""
    update = ns.update(shape, 1).cuda()
    want = ns.steps_of(update)
    off = lambda x: float((x.double() - want).norm() / want.norm())
    here, plain = off(dense.orthogonalize(update)), off(_float32_operations(update))
    assert here <= 2 * plain, (here, plain)


# tiles with other numbers of steps (the buffers of X change places), K of all products split over clusters and over launches, batches
@pytest.mark.parametrize("shape", [(64, 500), (100, 180), (300, 260), (200, 200), (150, 8000), (300, 3000), (2, 650, 700), (12, 140, 150), (1200, 1100)])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 7])
def test_steps_of_larger_matrices(shape, steps):
    for dtype in (torch.float32, torch.bfloat16):
        update = ns.update(shape, steps, dtype).cuda()
        ns.check(dense.orthogonalize(update, steps=steps), update, 22, steps=steps)


def test_streams_and_graphs_share_nothing():
    """Updates whose shares lie in workspaces, on several streams and in two graphs at once."""
    updates = [ns.update(shape, 9).cuda() for shape in ((150, 8000), (150, 9000), (300, 3000), (12, 1000), (100, 2000))]
    run = lambda: [dense.orthogonalize(u) for u in updates] + [dense.orthogonalize(updates[3], steps=20)]
    want = run()
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(4):
        torch.cuda.synchronize()
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


@pytest.mark.parametrize("shape", [(20, 30), (64, 200), (200, 100), (300, 260), (260, 300)])
@pytest.mark.parametrize("largest", [1e-32, 1e-36, 1e-38, 1e-41, 3e38])
def test_updates_next_to_the_ends_of_float32(shape, largest):
    update = ns.update(shape, 4).double()
    update = (update * (largest / update.abs().max())).float().cuda()
    for eps in (0.0, 1e-30 if largest < 1 else 1e30):
        want = ns.steps_of(update, eps=eps)
        if float(want.abs().max()) > 1e-3:                # else there is little left beside 2^-32
            ns.check(dense.orthogonalize(update, eps=eps), update, 64 if min(shape) <= 32 else 22, eps=eps)
