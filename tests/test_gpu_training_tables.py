"""The table's gradient of more than 2048 tokens (sort, sums, join) and preference losses of many rows, at the sizes where
their kernels change what they do; oracle and tolerances as in test_gpu_training.py."""

import pytest
import torch

from boundflow_amd import training
from oracle import training_ref as ref
from tests.gpu_util import announce, device
from tests.test_gpu_training import TYPES, close, gen, logp_tol, preference_inputs, rounded
from tests.test_gpu_training import test_embed_tokens_grad as check_embed_grad
from tests.test_gpu_training import test_preference_loss as check_preference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,count,vocab,dim", [
    # no more tokens than values: the table is cleared during the sort, and its bytes are no multiple of 16
    ("spread", 3000, 5001, 37), ("outside", 2049, 2049, 1), ("hot", 2500, 70001, 3),
    # rows of several whole chunks, pairs of them, and a rest; several column groups of the join
    ("spread", 2500, 4000, 1100), ("hot", 4000, 900, 4200), ("hot", 4000, 6000, 4200), ("outside", 2300, 300, 2057),
    # tokens read a second time (more than 16384), one value that holds all of them
    ("hot", 20_000, 1500, 40), ("one", 17_000, 3, 16), ("outside", 16_385, 200, 9), ("spread", 16_384, 20_000, 12),
    # more values than 256 workgroups take of 512
    ("spread", 2100, 140_001, 6), ("outside", 18_000, 131_073, 5),
    # few values
    ("spread", 2049, 1, 33), ("hot", 5000, 2, 1031), ("spread", 9000, 9, 8)])
def test_table_gradient_of_a_batch(dtype, kind, count, vocab, dim):
    check_embed_grad(dtype, kind, count, vocab, dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [500, 5000])
def test_table_gradient_of_tokens_that_are_all_outside(dtype, vocab):
    dev = device()
    rows = torch.randn(3000, 50, generator=gen(1)).to(dtype).to(dev)
    tokens = torch.where(torch.arange(3000, device=dev) % 2 == 0, -1, vocab)
    assert not training.embed_tokens_grad(rows, tokens, vocab).any()
    running = torch.randn(vocab, 50, generator=gen(2)).to(dev)
    start = running.clone()
    training.embed_tokens_grad(rows, tokens, vocab, accumulate_into=running)
    assert torch.equal(running, start)


@pytest.mark.parametrize("vocab,dim", [(700, 300), (4000, 1100)])
def test_table_gradient_of_a_batch_of_views(vocab, dim):
    """Rows with a stride that start at odd elements; tokens of a transposed array."""
    dev = device()
    g = gen(vocab)
    whole = torch.randn(60, 60, dim + 5, generator=g).bfloat16().to(dev)
    rows = whole[:, :, 3:3 + dim]
    tokens = torch.randint(-1, vocab + 1, (60, 60), generator=g).t()
    want, size, n = ref.embed_tokens_grad(rows.cpu(), tokens, vocab, 2.0)
    got = training.embed_tokens_grad(rows, tokens.to(dev), vocab, scale=2.0)
    close(got, want, rounded(want, torch.bfloat16) + size * n * 2.0 ** -23, "gradient of views")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,V", [
    # 2048 rows and more are in one part: a wave each up to four vectors a lane, then four waves
    ([1500, 700, 3, 0], 100), ([900, 1200], 1024), ([900, 1200], 1027), ([40, 2100], 2048), ([1100, 1000], 2051),
    ([700, 20, 900, 600], 2600), ([2048, 1], 4099), ([1, 2047], 1), ([1024, 1024, 5, 5], 17),
    # one row fewer comes in two
    ([1000, 1047], 2051), ([1000, 1045, 0, 2], 4099)])
def test_preference_loss_of_many_rows(dtype, lengths, V):
    check_preference(dtype, lengths, V)


@pytest.mark.parametrize("dtype", TYPES)
def test_preference_loss_of_many_pairs_in_one_part(dtype):
    """Pairs of a few rows each, padding tokens, rows of no response on both sides, rows at odd elements."""
    dev = device()
    g = gen(7)
    lengths = torch.randint(0, 9, (600,), generator=g).tolist()
    for V in (301, 2053):
        announce(f"{sum(lengths)} rows of {V}")
        s = preference_inputs(lengths, V, dtype, 5, 4, 6)
        s["tokens"][::13] = -1
        r = ref.preference_loss(**s, label_smoothing=0.1)
        whole = torch.zeros(s["logits"].shape[0], V + 2, dtype=dtype)
        whole[:, 1:-1] = s["logits"]
        on = {k: v.to(dev) for k, v in s.items()}
        on["logits"] = whole.to(dev)[:, 1:-1]
        got = training.preference_loss(**on, label_smoothing=0.1)
        tol = logp_tol(s["logits"], V)
        close(got.logp, r["logp"], tol + 2.0 ** -24 * r["logp"].abs(), "logp")
        bounds = s["offsets"].tolist()
        size = (r["logp"] - s["ref_logp"].double()).abs()
        moved = torch.stack([0.1 * (tol[a:b].sum() + (b - a + 8) * 2.0 ** -23 * size[a:b].sum())
                             for a, b in zip(bounds, bounds[1:])])
        close(got.rewards, r["rewards"], moved + 2.0 ** -22 * r["rewards"].abs(), "rewards")
        # |d loss / d h| <= 1, and each pair has a share of 1 / 300
        close(got.loss, r["loss"], float(moved.sum()) / 300 + 2.0 ** -19 * float(r["loss"]) + 2.0 ** -22, "loss")
        # the coefficient is at most beta / pairs, off by a quarter of what h is off by; the softmax by its row's tolerance
        pairs, worst = len(lengths) // 2, float(2 * moved.max())
        allowed = 0.1 / pairs * (worst / 4 + 2.0 ** -20 + tol[:, None] * 2)
        close(got.grad_logits, r["grad"], allowed + rounded(r["grad"], dtype), "gradient")
