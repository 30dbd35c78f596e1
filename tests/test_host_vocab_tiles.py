"""That the cases of tests/vocab_cases.py take the ways that they are there for.  No device call is made."""

import pytest
import torch

from boundflow_amd import _lib
from tests import vocab_cases as vc

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built (run python -m boundflow_amd.build)")


@pytest.mark.parametrize("dtype", list(vc.ELEM))
@pytest.mark.parametrize("case,narrow,wide", vc.CASES)
def test_cases_take_the_ways_that_they_are_there_for(case, narrow, wide, dtype):
    want = wide if dtype == torch.float32 else narrow
    if want is None:
        pytest.skip("for 16-bit types")
    pieces, logits, grads, *_ = vc.plan(*case, dtype)
    assert (logits, grads, pieces > 1) == want


def test_every_tile_is_taken_both_ways():
    """Logits formed once and formed again, in each tile that there is for a type."""
    for dtype in vc.ELEM:
        ways = set()
        for case, narrow, wide in vc.CASES:
            if (wide if dtype == torch.float32 else narrow) is not None:
                ways |= vc.kernels(case, dtype, True) | vc.kernels(case, dtype, False)
        tiles = ("large", "deep", "registers") if dtype == torch.float32 else ("large", "mid", "deep", "slim", "thin")
        for tile in tiles:
            assert {mode for what, mode, _, t in ways if what == "logits" and t == tile} >= {0, 1}, (dtype, tile)
            assert any(what == "grads" and t == tile for what, _, _, t in ways), (dtype, tile)


def test_the_plan_refuses_what_the_call_refuses():
    lib = _lib.load()
    assert lib.bf_vocab_loss_plan(0, 4, 4, 0, 0, 4, 1, 0, 0, None) == 1
    assert lib.bf_vocab_loss_plan(4, 4, 4, 0, 0, 4, 1, 0, 0, None) == 1
    out = torch.zeros(6, dtype=torch.int64)
    assert lib.bf_vocab_loss_plan(1 << 24, 4, 4, 0, 0, 4, 1, 0, 0, out.data_ptr()) == 3
    assert lib.bf_vocab_loss_plan(4, 4, 4, 0, 0, 4, 1, 0, 0, out.data_ptr()) == 0
