"""That the cases of tests/vocab_cases.py take the ways that they are there for.  No device call is made."""

import collections
import re
import subprocess

import pytest
import torch

from boundflow_amd import _lib
from tests import vocab_cases as vc

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built (run python -m boundflow_amd.build)")


@pytest.mark.parametrize("case,dtype,want", vc.RUNS)
def test_cases_take_the_ways_that_they_are_there_for(case, dtype, want):
    pieces, logits, grads, *_ = vc.plan(*case, dtype)
    assert (logits, grads, pieces > 1) == want


def test_every_tile_is_taken_both_ways():
    """Logits formed once and formed again, in each tile that there is for a type."""
    for dtype in vc.ELEM:
        ways = set()
        for case, of, _ in vc.RUNS:
            if of == dtype:
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


def test_no_kernel_is_compiled_that_no_call_reaches():
    """The products' kernels in the library, by what they do, G's parts and the type, against those that the cases launch."""
    names = subprocess.run(["nm", str(_lib.LIB_PATH)], capture_output=True, text=True, check=True).stdout
    built = collections.Counter()
    # bf::__device_stub__vocab_logits_kernel<VocabTile<eight numbers>, MODE, E, GP, S>: E is DF16b (bf16) or DF16_ (fp16)
    for mode, e, parts in re.findall(r"__device_stub__vocab_logits_kernelINS_9VocabTileI(?:Li\d+E){8}EELi(\d)E(DF16[b_])Li(\d)E", names):
        built[("logits", int(mode), int(parts), e)] += 1
    for e, parts in re.findall(r"__device_stub__vocab_grads_kernelINS_9VocabTileI(?:Li\d+E){8}EE(?:NS1_I(?:Li\d+E){8}EE|S2_)(DF16[b_])Li(\d)E",
                               names):
        built[("grads", None, int(parts), e)] += 1
    for e, parts in re.findall(r"__device_stub__vocab_softmax_columns_kernelI(DF16[b_])Li(\d)EE", names):
        built[("columns", None, int(parts), e)] += 1
    assert sum(built.values()) == len(set(re.findall(
        r"\S*__device_stub__vocab_(?:logits|grads|softmax_columns)_kernel\S*", names))), "a name that was not understood"
    reached = set()
    for case, dtype, _ in vc.RUNS:
        e = "DF16_" if dtype == torch.float16 else "DF16b"
        ways = vc.kernels(case, dtype, True) | vc.kernels(case, dtype, False)
        reached |= {(what, mode, parts, e, tile) for what, mode, parts, tile in ways}
        *_, parts, _, columns = vc.plan(*case, dtype)
        reached |= {("columns", None, parts, e, None)} if columns else set()
    assert collections.Counter(w[:4] for w in reached) == built
