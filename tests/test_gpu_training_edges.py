"""Edges of the training operators' calls: other default types, numbers at the ends of their range, layouts,
limits.  Tolerances as in test_gpu_training.py."""

import math

import pytest
import torch

from boundflow_amd import training
from boundflow_amd._lib import HipError
from oracle import training_ref as ref
from tests.gpu_util import announce, device
from tests.test_gpu_training import check_policy, close, gen, logp_tol, policy_inputs, preference_inputs

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,rows", [(5, 6), (301, 6), (4099, 6), (2050, 300)])
def test_losses_at_tokens_that_a_mask_took_out(dtype, V, rows):
    """A token whose logit is a mask's value, the type's lowest: its log-probability is about that number, and where
    the old and the reference policy say the same, the ratio is 1, the KL term 0 and the loss finite."""
    dev = device()
    s = policy_inputs(1, rows, V, dtype, 7, True, "none")
    z, lowest = s["logits"].clone(), torch.finfo(dtype).min
    picked = torch.arange(0, rows, 2)
    z[0, picked, s["tokens"][0, picked]] = lowest
    s["logits"] = z
    lp = torch.log_softmax(z.double(), -1).gather(-1, s["tokens"][..., None])[..., 0]
    s["old_logp"], s["ref_logp"] = lp.float(), lp.float()
    got = check_policy(s, dev, what=f"tokens at the lowest value, {rows} x {V}")
    assert torch.isfinite(got.logp).all() and torch.isfinite(got.stats).all()
    q = dict(logits=z[0], tokens=s["tokens"][0], ref_logp=s["ref_logp"][0], offsets=torch.tensor([0, 2, rows]))
    r = ref.preference_loss(**q)
    got = training.preference_loss(**to(dev, q))
    tol = logp_tol(z[0], V) + 2.0 ** -23 * r["logp"].abs()
    close(got.logp, r["logp"], tol, "preference logp")
    # rows at a mask's value differ from the reference's by what both are rounded by, 2^-24 of it each
    moved = 0.1 * tol.sum()
    close(got.rewards, r["rewards"], moved.expand(2), "preference rewards")
    assert torch.isfinite(got.loss)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("smoothing,out", [(0.0, 1), (1.0, 0), (0.1, 1)])
def test_preference_loss_of_a_response_that_cannot_be(dtype, smoothing, out):
    """A token at -inf: its response has reward -inf.  Rejected (out = 1), h = inf and -log sigma(h) = 0; the term whose
    weight is 0 is not there, so the batch's loss is that of the other pair.  With both weights the loss is infinite."""
    dev = device()
    s = preference_inputs([3, 2, 2, 4], 40, dtype, 6)
    want = ref.preference_loss(**s, label_smoothing=smoothing)
    h = float(want["rewards"][0] - want["rewards"][2])
    other = math.log1p(math.exp(-h)) if smoothing == 0.0 else math.log1p(math.exp(h))
    row = {1: 8, 0: 3}[out]     # in the second pair: of its rejected response, or of its chosen one
    s["logits"][row, s["tokens"][row]] = float("-inf")
    got = training.preference_loss(**to(dev, s), label_smoothing=smoothing)
    assert float(got.rewards[1 + 2 * out]) == float("-inf")
    if smoothing in (0.0, 1.0):
        # the pair's loss is 0 and so is its gradient
        assert abs(float(got.loss) - other / 2) < 2.0 ** -18 * (abs(h) + 1)
        assert not got.grad_logits[[3, 4, 7, 8, 9, 10]].any() and torch.isfinite(got.grad_logits).all()
    else:
        assert float(got.loss) == float("inf")
        # d loss / d h of the second pair is -(0.9 * 0 - 0.1 * 1) = 0.1 for the rejected response at -inf
        assert got.grad_logits[[3, 4]].any()


def test_embed_tokens_from_a_table_of_one_row():
    dev = device()
    table = torch.randn(6, 1, generator=gen(1)).to(dev).t()
    tokens = torch.tensor([0, -1, 0, 1], device=dev)
    got = training.embed_tokens(table, tokens)
    assert torch.equal(got[0], table[0]) and torch.equal(got[2], table[0])
    assert not got[1].any() and torch.isnan(got[3]).all()


def test_embed_tokens_of_more_rows_than_a_launch_takes():
    """2^23 + 11 rows of 4096 bf16 columns, 64 GiB: 2^32 vectors of 16 bytes and some."""
    dev = device()
    count, dim = (1 << 23) + 11, 4096
    announce("embedding of 64 GiB")
    table = torch.randn(50, dim, generator=gen(1)).bfloat16().to(dev)
    tokens = torch.randint(0, 50, (count,), generator=gen(2)).to(dev)
    got = training.embed_tokens(table, tokens)
    for rows in (slice(0, 300), slice(count // 2, count // 2 + 300), slice(count - 300, count)):
        assert torch.equal(got[rows], table[tokens[rows]])
    # every row's first and last element
    for d in (0, dim - 1):
        assert torch.equal(got[:, d], table[tokens, d])


def test_preference_loss_of_more_pairs_than_a_launch_has_workgroups():
    """Answers of one token, 2^22 + 3 pairs: a workgroup takes several."""
    dev = device()
    pairs, V = (1 << 22) + 3, 3
    N = 2 * pairs
    announce(f"{pairs} pairs")
    z = torch.randn(N, V, generator=gen(3))
    tokens = torch.randint(0, V, (N,), generator=gen(4))
    ref_logp = -torch.rand(N, generator=gen(5))
    got = training.preference_loss(z.to(dev), tokens.to(dev), ref_logp.to(dev), torch.arange(N + 1, device=dev), beta=0.5,
                                   grad_scale=float(pairs))
    logsm = torch.log_softmax(z.double(), -1)
    logp = logsm.gather(-1, tokens[:, None])[:, 0]
    rewards = 0.5 * (logp - ref_logp.double())
    h = rewards[:pairs] - rewards[pairs:]
    tol = logp_tol(z, V)
    close(got.logp, logp, tol + 2.0 ** -24 * logp.abs(), "logp")
    close(got.rewards, rewards, 0.5 * tol + 2.0 ** -22 * rewards.abs(), "rewards")
    # 1024 threads sum some 4096 terms each, and then one another's: 4106 roundings at most
    loss = torch.nn.functional.softplus(-h).mean()
    close(got.loss, loss, 4200 * 2.0 ** -24 * float(loss) + float(tol.max()), "loss")
    g = -torch.sigmoid(-h) * 0.5
    want = torch.cat([g, -g])[:, None] * (torch.nn.functional.one_hot(tokens, V) - logsm.exp())
    close(got.grad_logits, want, 2.0 ** -20 + 2.0 ** -20 * want.abs(), "gradient")


@pytest.mark.parametrize("bits,master", [(32, False), (8, True)])
def test_adamw_goes_on_from_its_saved_state(bits, master, tmp_path):
    dev = device()
    g = gen(9)
    first = [torch.randn(n, generator=g).bfloat16().to(dev) for n in (1000, 7)]
    grads = [[torch.randn(n, generator=g).bfloat16().to(dev) for n in (1000, 7)] for _ in range(6)]
    straight = [p.clone() for p in first]
    opt = training.AdamW(straight, bits=bits, master=master)
    for k in grads:
        opt.step(k)
    broken = [p.clone() for p in first]
    opt = training.AdamW(broken, bits=bits, master=master)
    for k in grads[:3]:
        opt.step(k)
    torch.save({"params": broken, "moments": tuple(opt.moments), "t": opt.t}, tmp_path / "state.pt")
    kept = torch.load(tmp_path / "state.pt", weights_only=True)
    again = training.AdamW(kept["params"], bits=bits, master=master)
    again.moments, again.t = training.AdamWMoments(*kept["moments"]), kept["t"]
    for k in grads[3:]:
        again.step(k)
    assert all(torch.equal(a, b) for a, b in zip(kept["params"], straight))


@pytest.mark.parametrize("B,T,V", [(1, 6, 5), (2, 40, 300), (2, 5, 4099), (2, 200, 2050)])
def test_policy_loss_with_a_kl_weight_of_0_at_rows_far_from_the_reference(B, T, V):
    """exp(ref - p) passes the largest fp32 (the reference has the token 95 and 300 nats above): the KL statistic is inf,
    and a term of weight 0 is not in the loss or its gradient."""
    dev = device()
    s = policy_inputs(B, T, V, torch.float32, 3, True, "none")
    s["ref_logp"][0, 1] += 95.0
    s["ref_logp"][-1, 4] += 300.0
    want = training.policy_loss(**{**to(dev, s), "ref_logp": None})
    got = training.policy_loss(**to(dev, s), kl_weight=0.0)
    assert float(got.stats[2]) == float("inf")
    for k in (0, 1, 3):
        assert float(got.stats[k]) == float(want.stats[k])
    assert torch.equal(got.grad_logits, want.grad_logits) and torch.equal(got.logp, want.logp)
    r = ref.policy_loss(**s)
    # terms of a few units, each off by some 2^-22 of its row's spread of 30 (logp_tol) and summed in fp32
    assert abs(float(got.loss) - float(r["stats"][0])) < 1e-4 * (1 + abs(float(r["stats"][0])))


@pytest.mark.parametrize("B,T,V", [(1, 6, 5), (2, 40, 300), (2, 5, 4099), (2, 200, 2050)])
def test_policy_loss_of_rows_without_an_advantage_far_from_the_old_policy(B, T, V):
    """exp(p - old) passes the largest fp32 at rows whose advantage is 0: the term is 0, as exp(95) * 0 is."""
    dev = device()
    s = policy_inputs(B, T, V, torch.float32, 5, False, "none")
    s["advantages"][0, 1] = s["advantages"][-1, 4] = 0.0
    near = ref.policy_loss(**s)
    s["old_logp"][0, 1] -= 95.0
    s["old_logp"][-1, 4] -= 300.0
    r = ref.policy_loss(**s)
    assert torch.equal(r["stats"], near["stats"])
    got = training.policy_loss(**to(dev, s))
    # terms of a few units, each off by some 2^-22 of its row's spread of 30 (logp_tol) and summed in fp32
    close(got.stats, r["stats"], 1e-4 * (1 + r["stats"].abs()), "stats")
    assert torch.isfinite(got.grad_logits).all()
    assert not got.grad_logits[0, 1].any() and not got.grad_logits[-1, 4].any()
