"""That the tolerances of orthogonalised updates let no fault through: results with one are made here, on the CPU."""
import pytest
import torch

from habitat_b200 import _native
from tests import newton_schulz as ns

SHAPES = [(12, 1024), (64, 200), (128, 700), (300, 260), (2, 150, 180)]


def _operands(shape):
    return 64 if min(shape[-2:]) <= 32 else 22


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_right_results_pass(shape, dtype):
    g = ns.update(shape, 1, dtype)
    ns.check(ns.steps_of(g).to(dtype), g, _operands(shape))
    ns.check(ns.steps_of(g, bits=22).to(dtype), g, 22)
    ns.check(ns.steps_of(g, bits=11).to(dtype), g, 11)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_faults_do_not(shape, dtype):
    g = ns.update(shape, 1, dtype)
    want, rest = ns.steps_of(g), ns.steps_of(g, bits=11)
    lost = rest.clone()
    lost[..., : min(32, shape[-2]), 32:64] = 0                         # a block that was not stored
    mirrored = rest.clone()
    k = min(32, shape[-2])
    mirrored[..., :k, :k] = rest[..., :k, :k].mT                       # or stored the wrong way round
    for x in (lost, mirrored, ns.steps_of(g, steps=4), ns.steps_of(g, bits=6), ns.steps_of(g, bits=8)):
        with pytest.raises(AssertionError):
            ns.check(x.to(dtype), g, 11)
    # fewer bits than were asked for (results of 8 and 11 bits show no more than that)
    for bits in (11, 16) if dtype == torch.float32 else (11,):
        with pytest.raises(AssertionError):
            ns.check(ns.steps_of(g, bits=bits).to(dtype), g, _operands(shape))
    assert float((want - lost).norm() / want.norm()) < 0.5             # (no gross ones)


def test_workspaces_have_room_for_shares_only_where_there_are_some():
    """Symmetric products of few tiles and a long K leave shares of 256 x 128 float32 in memory; nothing else does."""
    size = _native.load().hb_orthogonalize_workspace_bytes
    for batch, rows, cols in ((1, 1, 1), (1, 1024, 12), (1, 64, 64), (1, 128, 300), (3, 100, 90), (1, 200, 200)):
        for split in (0, 1):
            s, l = min(rows, cols), max(rows, cols)
            up = lambda x, m: (x + m - 1) // m * m
            planes = 2 * batch * (1 + split) * 2 * s * (up(l, 64) + up(s, 64)) + 4 * batch * 257 * 2
            assert planes <= size(batch, rows, cols, split) <= planes + 6 * 256
    assert size(1, 150, 8000, 1) >= 2 * 2 * 2 * 150 * 8000 + 2 * 25 * 256 * 128 * 4
