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
