"""Edges of the training operators' calls: other default types, numbers at the ends of their range, layouts,
limits.  Tolerances as in test_gpu_training.py."""

import pytest
import torch

from boundflow_amd import training
from boundflow_amd._lib import HipError
from tests.gpu_util import device
from tests.test_gpu_training import gen, policy_inputs, preference_inputs

pytestmark = pytest.mark.gpu


def to(dev, s):
    return {k: v.to(dev) if v is not None else None for k, v in s.items()}


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
def test_results_do_not_depend_on_the_default_type(default):
    """A program for 16-bit networks sets its default type: buffers that kernels fill with fp32 stay fp32."""
    dev = device()
    tokens = torch.randint(0, 90, (3000,), generator=gen(1)).to(dev)
    rows = torch.randn(3000, 40, generator=gen(2)).bfloat16().to(dev)
    calls = [(to(dev, policy_inputs(*shape, torch.bfloat16, 3, True, "some")),
              to(dev, preference_inputs(lengths, shape[-1], torch.bfloat16, 4)))
             for shape, lengths in (((2, 5, 7), [3, 4]), ((3, 7, 4099), [5, 2, 9, 1]), ((2, 300, 2050), [150, 200]))]
    weights = torch.randn(1000, generator=gen(5)).to(dev)

    def everything():
        out = [training.embed_tokens_grad(rows, tokens, 90)]
        for s, q in calls:
            a, b = training.policy_loss(**s, kl_weight=0.1), training.preference_loss(**q)
            out += [a.stats, a.logp, a.grad_logits, b.loss, b.rewards, b.logp, b.grad_logits]
        for bits in (32, 8):
            p = weights.clone()
            opt = training.AdamW([p], bits=bits, master=True)
            opt.step([weights])
            out += [p, *(t.view(torch.uint8) for t in opt.moments if t is not None)]
        return out

    want = everything()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = everything()
    finally:
        torch.set_default_dtype(before)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_adamw_refuses_tied_weights():
    dev = device()
    w = torch.ones(300, device=dev)
    opt = training.AdamW([w, torch.ones(5, device=dev), w])
    with pytest.raises(HipError, match="share memory"):
        opt.step([torch.ones(300, device=dev), torch.ones(5, device=dev), torch.ones(300, device=dev)])
    assert torch.equal(w, torch.ones(300, device=dev)) and not opt.moments.m.any() and opt.t == 0
