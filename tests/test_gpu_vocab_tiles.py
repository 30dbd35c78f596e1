"""The vocabulary loss through every tile of its products, with several stages of k each, the logits formed once and formed
again: against float64, with the tolerances of tests/test_gpu_supervised.py."""

import pytest
import torch

from tests import vocab_cases as vc
from tests.gpu_util import device
from tests.test_gpu_supervised import check, head
from tests.test_gpu_training import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case,dtype,_ways", vc.RUNS)
def test_vocabulary_loss_through_every_tile(case, dtype, _ways):
    N, D, V, gap, with_bias, room = case
    hidden, weight, tokens, bias = head(N, D, V, dtype, N + D + V)
    mask = torch.rand(N, generator=gen(1)) < 0.9
    mask[0] = True
    on = {}
    if gap:
        whole = torch.full((V, D + gap), float("nan"), dtype=dtype)
        whole[:, :D] = weight
        on["weight"] = whole.to(device())[:, :D]
    check(hidden, weight, tokens, bias=bias if with_bias else None, mask=mask, room=room, on=on)
