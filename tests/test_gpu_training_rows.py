"""Policy losses of large batches: rows that a workgroup holds in registers one after another, short rows in turns, rows
past what a workgroup holds.  The float64 restatement (oracle/training_ref.py) runs on the device here, where its
elementary operations take milliseconds; tolerances are those of test_gpu_training.py."""

import math

import pytest
import torch

from boundflow_amd import training
from oracle import training_ref as ref
from tests.gpu_util import announce, device
from tests.test_gpu_training import TINY, TYPES, close, grad_tol, logp_tol

pytestmark = pytest.mark.gpu

BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


def inputs(dev, B, T, V, dtype, *, start=0, temperature=1.0, kl=True, seed=0):
    """Logits from element `start` of a buffer, a row of NaN after every sequence; masked runs of rows, whole sequences
    of them, negative tokens; tokens at a row's ends."""
    g = torch.Generator(device=dev).manual_seed(seed + B + T + V)
    rand = lambda *shape: torch.rand(*shape, device=dev, generator=g)  # noqa: E731
    randn = lambda *shape: torch.randn(*shape, device=dev, generator=g)  # noqa: E731
    whole = (randn(start + B * (T + 1) * V) * 3).to(dtype)
    padded = whole[start:].view(B, T + 1, V)
    padded[:, T] = float("nan")
    logits = padded[:, :T]
    tokens = torch.randint(0, V, (B, T), device=dev, generator=g)
    flat = tokens.view(-1)
    for k, t in enumerate((0, V - 1, min(1, V - 1), max(V - 8, 0), max(V - 9, 0))):
        flat[k::11] = t
    lp = torch.log_softmax(logits.double() / temperature, -1).gather(-1, tokens[..., None])[..., 0]
    drift = randn(B, T) * 0.2
    for limit in (math.log(0.8), math.log(1.28)):     # no ratio so near a limit that rounding decides
        drift = torch.where((drift - limit).abs() < 5e-3, limit + 0.01, drift)
    mask = rand(B, T) < 0.8
    mask.view(-1)[5:40] = True       # a run of live rows, and one of masked ones
    mask.view(-1)[50:70] = False
    if B > 3:
        mask[1] = False
        mask[-1] = False
    flat[::17] = -1
    return dict(logits=logits, tokens=tokens, old_logp=(lp - drift).float(), advantages=randn(B, T),
                ref_logp=(lp + randn(B, T) * 0.4).float() if kl else None, mask=mask)


def check(s, what, *, temperature=1.0, reduction="token", kl_weight=0.05, grad_scale=1.0):
    announce(what)
    kw = dict(clip_low=0.2, clip_high=0.28, kl_weight=kl_weight, temperature=temperature, reduction=reduction,
              grad_scale=grad_scale)
    got = training.policy_loss(**s, **kw)
    r = ref.policy_loss(**s, **kw)
    dtype, V, N = s["logits"].dtype, s["logits"].shape[-1], r["g"].numel()
    tol_lp = torch.where(r["live"], logp_tol(s["logits"] / temperature, V), 0.0)
    r["token"] = s["tokens"].clamp(min=0)
    extra = r["slope"] * (tol_lp + 2.0 ** -22)
    tol = grad_scale * grad_tol(r["grad"] / grad_scale, r, extra, tol_lp, 1 / temperature, dtype) + TINY[dtype]
    # compared on the device: the gradients are large
    for name, a, want, allowed in (("logp", got.logp, r["logp"], tol_lp + 2.0 ** -24 * r["logp"].abs()),
                                   ("gradient", got.grad_logits, r["grad"], tol)):
        d = (a.double() - want).abs()
        bad = int((~(d <= allowed)).sum())     # a NaN is outside
        announce(f"  {name}: max abs err {float(d.max()):.2e}, outside {bad}/{d.numel()}")
        assert bad == 0, f"{what}, {name}: {bad} elements outside their tolerance"
    slack = float((r["slope"] * tol_lp).sum()) + (N / 256 + 32) * 2.0 ** -23 * float((r["slope"] + r["g"].abs()).sum() + 1)
    close(got.stats, r["stats"].cpu(), slack, f"{what} stats")
    alone = training.policy_loss(**s, **kw, with_grad=False)
    assert alone.grad_logits is None and torch.equal(alone.stats, got.stats) and torch.equal(alone.logp, got.logp)
    again = training.policy_loss(**s, **kw)
    assert torch.equal(again.grad_logits, got.grad_logits) and torch.equal(again.stats, got.stats)


# (threads, vectors a thread, vectors of the shape before): a row's vectors decide the shape that holds it
SHAPES = [(64, 1, 63), (64, 2, 64), (64, 4, 128), (256, 2, 256), (256, 4, 512), (512, 3, 1024), (512, 4, 1536),
          (512, 6, 2048), (512, 8, 3072), (1024, 6, 4096), (1024, 8, 6144), (1024, 10, 8192), (1024, 12, 10240),
          (1024, 14, 12288), (1024, 16, 14336)]
GROUPS = {64: 4096, 256: 1536, 512: 512, 1024: 256}     # workgroups of a launch


@pytest.mark.parametrize("threads,each,before", SHAPES)
def test_rows_held_one_after_another(threads, each, before):
    """More than twice as many rows as workgroups, so each goes from live row to live row, masked ones between
    them; the shortest and the longest rows of every shape.  Rows of 16 bits that start at odd elements, from the
    buffer's start or from every other row's, have a vector less than their length says."""
    dev = device()
    B, T = 8, GROUPS[threads] * 9 // 32       # 2.25 rows a workgroup
    for k, (dtype, vectors, rest, start) in enumerate([(BF16, threads * each, 7, 0), (BF16, before + 1, 0, 1),
                                                       (F16, before + 1, 1, 0), (F32, threads * each, 3, 1),
                                                       (F32, before + 1, 0, 0)]):
        size = 4 if dtype == F32 else 8
        V = vectors * size + rest
        if V <= (256 if dtype == F32 else 512):
            V = 257 if dtype == F32 else 513      # shorter rows are not held
        warm = (1.0, 0.8)[k % 2]
        check(inputs(dev, B, T, V, dtype, start=start, temperature=warm, kl=k != 2),
              f"{dtype} {B * T} x {V} in {threads} x {each}", temperature=warm,
              reduction=("token", "sequence")[(k + each) % 2], grad_scale=(1.0, 64.0)[k % 2])


@pytest.mark.parametrize("dtype,V", [(BF16, 131072), (BF16, 131079), (BF16, 131080), (F16, 131081), (F32, 65536),
                                     (F32, 65539), (F32, 65540), (F32, 70001)])
@pytest.mark.parametrize("B,T", [(5, 60), (3, 86), (8, 260)])
def test_rows_at_the_longest_that_a_workgroup_holds(dtype, V, B, T):
    """16384 vectors and what is left of one more are held; longer rows are read twice, in several parts or (from
    2048 rows on) in one."""
    dev = device()
    for start in (0, 1):
        check(inputs(dev, B, T, V, dtype, start=start), f"{dtype} {B * T} x {V} from {start}",
              reduction=("token", "sequence")[start])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,V", [(70, 70, 5), (1, 5000, 16), (600_000, 1, 3), (30, 300, 17), (4, 10_001, 100),
                                   (50, 90, 256), (41, 211, 255)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_short_rows_in_turns(dtype, B, T, V, reduction):
    """Batches past the one workgroup that takes small ones, up to more rows than lanes of the grid."""
    check(inputs(device(), B, T, V, dtype, start=1), f"{dtype} {B} x {T} x {V}", reduction=reduction)


@pytest.mark.parametrize("B,T,V", [(2500, 3, 700), (150_000, 1, 5), (70_000, 2, 4), (1, 6000, 600), (3000, 1, 520),
                                   (20_000, 3, 6)])
def test_sequences_counted_by_several_workgroups(B, T, V):
    """Each counts a share of the sequences, more than are held at a time among them."""
    check(inputs(device(), B, T, V, BF16), f"{B} sequences of {T}", reduction="sequence")


@pytest.mark.parametrize("B,T,V", [(8, 600, 700), (4, 200, 5000), (9, 100, 100), (2, 150, 70001)])
def test_large_batches_without_a_live_row(B, T, V):
    dev = device()
    s = inputs(dev, B, T, V, BF16)
    for change in (dict(mask=torch.zeros(B, T, dtype=torch.bool, device=dev)), dict(tokens=torch.full_like(s["tokens"], -3))):
        for reduction in ("token", "sequence"):
            got = training.policy_loss(**{**s, **change}, reduction=reduction, kl_weight=0.1)
            assert not got.stats.any() and not got.logp.any() and not got.grad_logits.any()


def test_a_row_that_is_not_a_number_among_held_rows():
    """NaN and inf in live rows show there; the rows that the workgroup holds before and after are as without them."""
    dev = device()
    s = inputs(dev, 8, 1200, 1500, BF16)
    s["mask"][:] = True
    s["tokens"].clamp_(min=0)
    want = training.policy_loss(**s, kl_weight=0.05)
    s["logits"][2, 100:103, 7] = torch.tensor([float("nan"), float("inf"), float("nan")], device=dev)
    s["tokens"][5, 5] = 1500
    got = training.policy_loss(**s, kl_weight=0.05)
    odd = torch.zeros(8, 1200, dtype=torch.bool, device=dev)
    odd[2, 100:103] = odd[5, 5] = True
    assert torch.isnan(got.logp[odd]).all() and torch.isnan(got.loss)
    assert torch.isnan(got.grad_logits[odd]).all()
    assert torch.equal(got.logp[~odd], want.logp[~odd]) and torch.equal(got.grad_logits[~odd], want.grad_logits[~odd])
