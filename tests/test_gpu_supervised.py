"""The operators of a supervised step, ``vocabulary_loss`` and ``dropout``, against plain float64 restatements
(oracle/training_ref.py).

Tolerances are those of the arithmetic.  A logit is a sum of D exact products in fp32 (fp32 inputs: of six part
products each, what they leave out below 2^-22 of a product): off by at most (6 D + 8) 2^-24 of the sum of their
magnitudes, as is a gradient's sum over its rows or its vocabulary.  A log-probability is off by what the logits, the exponents' roundings and the sum
leave.  The softmax's gradient is rounded to the inputs' type between the products (fp32: to three bf16 parts, 2^-24),
and results are rounded once."""

import copy
import importlib.util
import math
import os

import pytest
import torch

from boundflow_amd import training
from boundflow_amd._lib import HipError
from oracle import training_ref as ref
from tests import vocab_cases
from tests.gpu_util import announce, device
from tests.test_gpu_training import TINY, TYPES, U, close, gen, logp_tol, rounded

pytestmark = pytest.mark.gpu


def head(N, D, V, dtype, seed, *, bias=True, spread=2.0):
    """Hidden rows, a head and tokens, the tokens' logits raised by different amounts."""
    g = gen(seed)
    weight = (torch.randn(V, D, generator=g) * spread / math.sqrt(D)).to(dtype)
    tokens = torch.randint(0, V, (N,), generator=g)
    lift = torch.rand(N, 1, generator=g) * (math.log(V) + 2) / spread ** 2
    hidden = (torch.randn(N, D, generator=g) + lift * weight[tokens].float()).to(dtype)
    return hidden, weight, tokens, (torch.randn(V, generator=g) * 0.5).to(dtype) if bias else None


def tolerances(r, dtype, temperature, V, D):
    """(of logp per live row, of G per live row and entry)"""
    count = 6 * D + 8 if dtype == torch.float32 else D + 8
    dz = (count * 2.0 ** -24 * r["size"]).amax(1) / temperature + 2.0 ** -22 * r["size"].amax(1) * (
        dtype == torch.float32)
    tol_lp = 2 * dz + logp_tol(r["z"] / temperature, V)
    # What is below a type's normal numbers: fp16 holds 2^14 G in steps of 2^-24, so G to 2^-39, and 2^15 times the exponentials
    # of 16-bit types, so these to 2^-40.  In fp32 a probability below 2^-126 is 0, and so is each of three bf16 parts (the
    # matrix cores read subnormal bf16 as 0): 4 * 2^-126 in all.
    extra = 2.0 ** -124 if dtype == torch.float32 else 2.0 ** -38
    # exponentials are rounded to 11 bits before they are scaled (but for the token's; fp32 not at all), G to its type after it
    early = 0.0 if dtype == torch.float32 else 2.0 ** -11
    return tol_lp, r["p"] * (tol_lp + 2.0 ** -21 + early)[:, None] + r["g"].abs() * (U[dtype] + 2.0 ** -23) + extra


def check(hidden, weight, tokens, *, bias=None, mask=None, temperature=1.0, grad_scale=1.0, wide=None, room=2 << 30, on=None,
          what=""):
    """`on`: the device tensors where their layout is not that of the others."""
    dev = device()
    dtype, (V, D) = weight.dtype, weight.shape
    r = ref.vocabulary_loss(hidden, weight, tokens, bias=bias, mask=mask, temperature=temperature, grad_scale=grad_scale)
    args = {"hidden": hidden, "weight": weight, "tokens": tokens, "bias": bias, "mask": mask}
    args = {k: None if v is None else v.to(dev) for k, v in args.items()}
    args.update(on or {})
    kw = dict(temperature=temperature, grad_scale=grad_scale, room=room)
    what = f"{what or tuple(hidden.shape)} x {V} {dtype}"
    got = training.vocabulary_loss(**args, **kw, weight_grad_dtype=wide)
    tol_lp, tol_g = tolerances(r, dtype, temperature, V, D)
    flat = torch.zeros(tokens.numel(), dtype=torch.float64)
    flat[r["at"]] = tol_lp
    close(got.logp, r["logp"], flat.view(tokens.shape) + 2.0 ** -23 * r["logp"].abs(), f"logp {what}")
    n = max(r["at"].numel(), 1)
    close(got.loss, r["loss"], float(tol_lp.sum()) / n + (n / 256 + 16) * 2.0 ** -23 * float(r["logp"].abs().sum()) / n,
          f"loss {what}")
    f, g = r["factor"], r["g"].abs()
    many = 6 if dtype == torch.float32 else 1
    tol = torch.zeros(tokens.numel(), D, dtype=torch.float64)
    tol[r["at"]] = f * (torch.mm(tol_g, r["w"].abs()) + (many * V + 8) * 2.0 ** -24 * torch.mm(g, r["w"].abs()))
    assert got.grad_hidden.dtype == dtype and got.grad_hidden.is_contiguous()
    close(got.grad_hidden, r["hidden"], tol.view(hidden.shape) + rounded(r["hidden"], dtype), f"grad hidden {what}")
    tol = f * (torch.mm(tol_g.t(), r["x"].abs()) + (many * n + 8) * 2.0 ** -24 * torch.mm(g.t(), r["x"].abs()))
    assert got.grad_weight.dtype == (wide or dtype)
    close(got.grad_weight, r["weight"], tol + rounded(r["weight"], wide or dtype), f"grad weight {what}")
    if bias is None:
        assert got.grad_bias is None
    else:
        tol = f * (tol_g.sum(0) + (many * n + 8) * 2.0 ** -24 * g.sum(0))
        close(got.grad_bias, r["bias"], tol + rounded(r["bias"], dtype), f"grad bias {what}")
    alone = training.vocabulary_loss(**args, **kw, with_grad=False)
    assert alone[2:] == (None, None, None)
    assert torch.equal(alone.logp, got.logp) and torch.equal(alone.loss, got.loss), "other bits without gradients"
    return got


SIZES = [(1, 1, 1), (1, 8, 5), (2, 7, 130), (3, 64, 257), (7, 192, 1003), (8, 129, 97), (9, 128, 128), (16, 65, 256),
         (17, 320, 300), (33, 64, 4099), (64, 256, 129), (65, 1025, 200), (130, 96, 2), (257, 128, 515), (300, 63, 1003)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", SIZES)
def test_vocabulary_loss(dtype, N, D, V):
    hidden, weight, tokens, bias = head(N, D, V, dtype, N + D + V)
    check(hidden, weight, tokens)
    check(hidden, weight, tokens, bias=bias, temperature=0.7, grad_scale=100.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(3, 4090, 600), (190, 2552, 904), (1, 2048, 8192), (70, 1024, 8193), (2000, 520, 7)])
def test_vocabulary_loss_of_long_rows(dtype, N, D, V):
    """Few tiles, whose sums are cut along the width (up to 8192 tokens)."""
    hidden, weight, tokens, bias = head(N, D, V, dtype, N + D)
    mask = torch.rand(N, generator=gen(1)) < 0.8
    mask[0] = True
    bias[V // 2:V // 2 + 2] = float("-inf")
    tokens = torch.where((tokens >= V // 2) & (tokens < V // 2 + 2), 0, tokens)
    check(hidden, weight, tokens, bias=bias, mask=mask, temperature=1.2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(700, 192, 1500), (1500, 64, 700), (40, 64, 9000), (513, 1100, 520)])
def test_vocabulary_loss_of_many_tiles(dtype, N, D, V):
    hidden, weight, tokens, bias = head(N, D, V, dtype, N + D)
    mask = torch.rand(N, generator=gen(1)) < 0.8
    check(hidden, weight, tokens, bias=bias, mask=mask, wide=torch.float32)


@pytest.mark.parametrize("N,D,V,dtype", [(1025, 24, 60, torch.float32), (5000, 40, 9, torch.bfloat16), (66_000, 16, 530, torch.bfloat16),
                                         (70_000, 8, 5, torch.float32)])
def test_rows_that_are_counted_by_many(N, D, V, dtype):
    """More rows than one workgroup counts, and than many do, of 32-bit tokens, long stretches of them not counting."""
    hidden, weight, tokens, bias = head(N, D, V, dtype, 3)
    mask = torch.rand(N, generator=gen(6)) < 0.7
    mask[: N // 9] = False
    mask[N // 3: N // 2] = False
    check(hidden, weight, tokens, bias=bias, mask=mask, on={"tokens": tokens.int().to(device())})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["some", "sequence", "first", "empty", "negative"])
@pytest.mark.parametrize("B,T", [(3, 2), (5, 77)])
def test_rows_that_do_not_count(dtype, kind, B, T):
    """Masked rows and rows of a negative token may hold anything, are not read, and get zeros."""
    dev = device()
    N, D, V = B * T, 96, 333
    hidden, weight, tokens, bias = head(N, D, V, dtype, 5)
    hidden, tokens = hidden.view(B, T, D).clone(), tokens.view(B, T).clone()
    mask = torch.ones(B, T, dtype=torch.bool)
    if kind == "some":
        mask = torch.rand(B, T, generator=gen(2)) < 0.5
    elif kind == "sequence":
        mask[0] = False
    elif kind == "first":
        mask[:] = False
        mask[-1, -1] = True
    elif kind == "empty":
        mask[:] = False
    else:
        tokens[torch.rand(B, T, generator=gen(3)) < 0.4] = -100
    live = mask & (tokens >= 0)
    hidden[~live] = float("nan")
    got = check(hidden, weight, tokens, bias=bias, mask=None if kind == "negative" else mask, what=kind)
    assert not bool(got.logp.cpu()[~live].any()) and not bool(got.grad_hidden.cpu()[~live].any())
    if kind == "empty":
        assert float(got.loss) == 0.0 and not bool(got.grad_weight.any()) and not bool(got.grad_bias.any())
    small = training.vocabulary_loss(hidden.to(dev), weight.to(dev), tokens.int().to(dev), bias=bias.to(dev),
                                     mask=None if kind == "negative" else mask.to(dev))
    for a, b in zip(small, got):
        assert torch.equal(a, b), "32-bit tokens, other bits"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [6, 100])
def test_views_are_read_in_place(dtype, N):
    dev = device()
    D, V = 72, 140
    hidden, weight, tokens, bias = head(N, D, V, dtype, 8)
    whole = torch.full((2, N // 2 + 1, D + 5), float("nan"), dtype=dtype)
    whole[:, :-1, 3:-2] = hidden.view(2, N // 2, D)
    table = torch.full((V + 2, D + 9), float("nan"), dtype=dtype)
    table[1:-1, 7:-2] = weight
    on = {"hidden": whole.to(dev)[:, :-1, 3:-2], "weight": table.to(dev)[1:-1, 7:-2]}
    on["bias"] = torch.stack([bias, bias], 1).to(dev)[:, 0]
    on["tokens"] = torch.stack([tokens, tokens]).t().contiguous().to(dev)[:, 0].view(2, N // 2)
    check(hidden.view(2, N // 2, D), weight, tokens.view(2, N // 2), bias=bias, on=on, what="views")
    wide = torch.zeros(V, 2 * 128, dtype=dtype)       # a weight that can be read as it lies, with gaps
    wide[:, :64] = weight[:, :64]
    check(hidden[:, :64], weight[:, :64], tokens, on={"weight": wide.to(dev)[:, :64]}, what="rows with gaps")
    # one hidden row for all, by a stride of 0
    same = hidden[:1].expand(N, D)
    check(same, weight, tokens, on={"hidden": hidden[:1].to(dev).expand(N, D)}, what="a repeated row")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [5, 70])
def test_masked_vocabulary(dtype, N):
    """-inf and the type's lowest value in the bias take entries out: no probability, no gradient."""
    hidden, weight, tokens, bias = head(N, 64, 300, dtype, 12)
    bias[40:170] = float("-inf")
    bias[200:] = torch.finfo(dtype).min
    bias[41] = 0.25
    tokens = torch.where((tokens >= 40) & (tokens < 170) | (tokens >= 200), 41, tokens)
    got = check(hidden, weight, tokens, bias=bias, what="masked vocabulary")
    assert not bool(got.grad_weight[42:170].any()) and not bool(got.grad_weight[200:].any())
    assert not bool(got.grad_bias[42:170].any())
    bias[:] = torch.finfo(torch.float32).min if dtype == torch.float32 else torch.finfo(dtype).min
    if dtype != torch.float16:      # 65504 leaves fp32 logits their digits; these leave none, so all are alike
        dev = device()
        got = training.vocabulary_loss(hidden.to(dev), weight.to(dev), tokens.to(dev), bias=bias.to(dev))
        close(got.logp, torch.full((N,), -math.log(300), dtype=torch.float64), 2.0 ** -20, "nothing but the lowest value")


@pytest.mark.parametrize("N", [4, 40])
def test_what_is_not_a_number_shows(N):
    dev = device()
    hidden, weight, tokens, bias = (t.to(dev) for t in head(N, 64, 40, torch.float32, 9))
    late = tokens.clone()
    late[1] = 40
    got = training.vocabulary_loss(hidden, weight, late)
    assert torch.isnan(got.logp[1]) and torch.isnan(got.loss) and torch.isnan(got.grad_hidden[1]).all()
    assert int(torch.isnan(got.logp).sum()) == 1 and torch.isnan(got.grad_weight).all()
    late = tokens.clone()
    late[1] = 1 << 40
    assert torch.isnan(training.vocabulary_loss(hidden, weight, late).logp[1])
    for value in (float("nan"), float("inf")):
        odd = hidden.clone()
        odd[2, 5] = value
        got = training.vocabulary_loss(odd, weight, tokens)
        assert torch.isnan(got.logp[2]) and torch.isnan(got.loss) and torch.isnan(got.grad_hidden[2]).any()
        assert int(torch.isnan(got.logp).sum()) == 1
        odd = bias.clone()
        odd[3] = value
        got = training.vocabulary_loss(hidden, weight, tokens, bias=odd)
        assert torch.isnan(got.logp).all()
    got = training.vocabulary_loss(hidden, weight, tokens, bias=torch.full_like(bias, float("-inf")))
    assert torch.isnan(got.logp).all()


def test_no_rows():
    dev = device()
    weight, bias = torch.randn(9, 16, device=dev), torch.randn(9, device=dev)
    for shape in ((0,), (0, 5), (3, 0)):
        got = training.vocabulary_loss(torch.zeros(*shape, 16, device=dev), weight,
                                       torch.zeros(shape, dtype=torch.int64, device=dev), bias=bias)
        assert float(got.loss) == 0.0 and got.logp.shape == shape and got.grad_hidden.shape == (*shape, 16)
        assert not bool(got.grad_weight.any()) and not bool(got.grad_bias.any())
        assert float(training.vocabulary_loss(torch.zeros(*shape, 16, device=dev), weight, torch.zeros(
            shape, dtype=torch.int64, device=dev), with_grad=False).loss) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,scale", [(5, 30.0), (90, 30.0)])
def test_sure_and_far_logits(dtype, N, scale):
    """Logits of hundreds: probabilities of 1 and of 0."""
    hidden, weight, tokens, bias = head(N, 64, 500, dtype, 4)
    check((hidden.float() * scale).to(dtype), weight, tokens, bias=bias, what="far logits")


def test_gradients_against_differences():
    """Along a direction the loss moves as the gradients say: central differences of the oracle-free fp32 loss, whose own
    error is that of two losses over the step."""
    dev = device()
    hidden, weight, tokens, bias = (t.to(dev) for t in head(37, 96, 211, torch.float32, 3))
    got = training.vocabulary_loss(hidden, weight, tokens, bias=bias, temperature=1.3)
    loss = lambda h, w, b: float(training.vocabulary_loss(h, w, tokens, bias=b, temperature=1.3,  # noqa: E731
                                                          with_grad=False).loss)
    g = torch.Generator(device=dev).manual_seed(1)
    step = 2.0 ** -6
    for name, at, grad in (("hidden", 0, got.grad_hidden), ("weight", 1, got.grad_weight), ("bias", 2, got.grad_bias)):
        d = torch.randn(grad.shape, device=dev, generator=g) * (0.3 if name == "weight" else 1.0)
        moved = [[t + s * step * d if k == at else t for k, t in enumerate((hidden, weight, bias))] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        want = float((grad.double() * d.double()).sum())
        # third derivatives of a mean log-softmax along d are below 2 |dz|^3, dz the logits' own change
        if name == "hidden":
            dz = float((d @ weight.t()).abs().max())
        elif name == "weight":
            dz = float((hidden @ d.t()).abs().max())
        else:
            dz = float(d.abs().max())
        tol = step ** 2 / 6 * 2 * (2 * dz / 1.3) ** 3 + 2.0 ** -18 / step
        announce(f"difference along {name}: {slope:.6f} against {want:.6f}, tolerance {tol:.2e}")
        assert abs(slope - want) <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(5, 64, 700), (70, 40, 1003), (300, 192, 513), (90, 65, 2000), (90, 520, 700), (6, 1000, 2051)])
@pytest.mark.parametrize("room", [0, 300_000])
def test_pieces(dtype, N, D, V, room):
    """No room, or a little: pieces of 256 tokens or some more, the logits of all but the first formed again."""
    hidden, weight, tokens, bias = head(N, D, V, dtype, 17)
    mask = torch.rand(N, generator=gen(5)) < 0.9
    check(hidden, weight, tokens, bias=bias, mask=mask, room=room, wide=torch.float32)


def test_room_that_is_the_products_alone():
    """The first piece's gradient comes from rounded exponentials, the others' from logits formed again: both as close."""
    for dtype in TYPES:
        hidden, weight, tokens, bias = head(40, 128, 1024, dtype, 23)
        whole = check(hidden, weight, tokens, bias=bias)
        cut = check(hidden, weight, tokens, bias=bias, room=0)
        assert torch.equal(whole.logp, cut.logp) and torch.equal(whole.loss, cut.loss)


def test_many_pieces_of_a_large_vocabulary():
    dev = device()
    N, D, V = 1024, 40, 170_001
    hidden, weight, tokens, bias = head(N, D, V, torch.float32, 6)
    mask = torch.rand(N, generator=gen(4)) < 0.6
    got = training.vocabulary_loss(hidden.to(dev), weight.to(dev), tokens.to(dev), bias=bias.to(dev), mask=mask.to(dev),
                                   room=400 << 20)
    at = mask.nonzero()[:, 0]
    n = at.numel()
    x, w = hidden[at].double().to(dev), weight.double().to(dev)
    q = torch.log_softmax(torch.mm(x, w.t()) + bias.double().to(dev), 1)
    rows, y = torch.arange(n, device=dev), tokens[at].to(dev)
    logp = q[rows, y]
    g = q.exp_()
    g[rows, y] -= 1.0
    size = float(torch.mm(x.abs()[:64], w.abs().t()).max() * 1.5)
    rel = 2 * ((6 * D + 8) * 2.0 ** -24 + 2.0 ** -22) * size + 2.0 ** -22 * 40 + (V / 256 + 64) * 2.0 ** -24
    close(got.logp.cpu()[at], logp.cpu(), rel, "logp of pieces")
    for name, have, want, bound in (
            ("hidden", got.grad_hidden[at.to(dev)], torch.mm(g, w) / n, torch.mm(g.abs(), w.abs()) / n),
            ("weight", got.grad_weight, torch.mm(g.t(), x) / n, torch.mm(g.abs().t(), x.abs()) / n),
            ("bias", got.grad_bias, g.sum(0) / n, g.abs().sum(0) / n)):
        # sums of up to V terms in fp32: 512 part sums of at most 6 * 512 terms each would be their worst order; 2^-15 holds
        # (6 V 2^-24 = 2^-4 is the bound of one sum, which the random signs of its roundings stay far below)
        close(have.cpu(), want.cpu(), (rel + 2.0 ** -15) * bound.cpu() + rounded(want.cpu(), torch.float32), f"grad {name}")
    assert not bool(got.grad_hidden.cpu()[~mask].any())


def test_refusals():
    dev = device()
    hidden, weight, tokens, bias = (t.to(dev) for t in head(6, 8, 10, torch.bfloat16, 1))
    call = training.vocabulary_loss
    for error, match, args, kw in (
            (HipError, "weight must be", (hidden, weight.float(), tokens), {}),
            (ValueError, "weight must be", (hidden, weight[:, :7], tokens), {}),
            (ValueError, "V >= 1", (hidden, weight[:0], tokens), {}),
            (HipError, "contiguous rows", (hidden, weight.t().contiguous().t(), tokens), {}),
            (HipError, "contiguous rows", (hidden, weight[:1].expand(10, 8), tokens), {}),
            (HipError, "contiguous last axis", (hidden.t().contiguous().t(), weight, tokens), {}),
            (ValueError, "hidden must be", (hidden[0], weight, tokens[0]), {}),
            (ValueError, "tokens of shape", (hidden, weight, tokens[:5]), {}),
            (HipError, "tokens must be", (hidden, weight, tokens.float()), {}),
            (HipError, "bias must be", (hidden, weight, tokens), {"bias": bias.float()}),
            (ValueError, "bias of shape", (hidden, weight, tokens), {"bias": bias[:9]}),
            (HipError, "mask must be", (hidden, weight, tokens), {"mask": tokens}),
            (ValueError, "mask of shape", (hidden, weight, tokens), {"mask": tokens[:5] > 0}),
            (ValueError, "temperature", (hidden, weight, tokens), {"temperature": 0.0}),
            (ValueError, "room must be", (hidden, weight, tokens), {"room": -1}),
            (ValueError, "weight_grad_dtype", (hidden, weight, tokens), {"weight_grad_dtype": torch.float16}),
            (HipError, "device tensor", (hidden, weight.cpu(), tokens), {}),
            (HipError, "must be float32", (hidden.double(), weight, tokens), {})):
        with pytest.raises(error, match=match):
            call(*args, **kw)


# ---------------------------------------------------------------------------
# dropout

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (), (7,), (8,), (3, 5), (33, 8), (5, 129), (2, 3, 50), (64, 160)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(dtype, shape, p):
    dev = device()
    g = gen(len(shape) + 3)
    x, r = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    seed, counter = 0xFEDCBA9876543210, (3 << 33) + 5
    want, kept = ref.dropout(x, p, seed, counter)
    got = training.dropout(x.to(dev), p, seed=seed, counter=counter)
    assert got.dtype == dtype and got.shape == x.shape
    close(got, want, rounded(want, dtype), f"dropout {shape} {p}")
    assert torch.equal(got.cpu() != 0, kept & (x != 0))
    assert torch.equal(training.dropout_grad(x.to(dev), p, seed=seed, counter=counter), got)
    on_device = torch.tensor(counter, device=dev)
    assert torch.equal(training.dropout(x.to(dev), p, seed=seed, counter=on_device), got)
    want, _ = ref.dropout(x, p, seed, counter, residual=r)
    both = training.dropout(x.to(dev), p, seed=seed, counter=counter, residual=r.to(dev))
    # the sum's rounding in fp32, before that to the type, is of a term that may be larger than the sum
    close(both, want, rounded(want, dtype) + 2.0 ** -22 * (x.abs().double() / max(1 - p, 0.5) + r.abs().double()),
          f"dropout and residual {shape} {p}")


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_of_views(dtype):
    """The mask follows an element's place in x, not in memory."""
    dev = device()
    whole = torch.randn(20, 41, generator=gen(2)).to(dtype).to(dev)
    kw = dict(seed=5, counter=1)
    for view in (whole[:, :40], whole[:, 3:], whole[::2], whole.t(), whole[:, ::3], whole[4], whole[:, 7],
                 whole[:1].expand(9, 41), whole.view(4, 5, 41)[:, 1:, 2:]):
        want = training.dropout(view.contiguous(), 0.3, **kw)
        assert torch.equal(training.dropout(view, 0.3, **kw), want)
        assert torch.equal(training.dropout(view.contiguous(), 0.3, residual=view, **kw),
                           training.dropout(view, 0.3, residual=view.contiguous(), **kw))
    assert torch.equal(training.dropout(whole[:0], 0.3, **kw), whole[:0])


def test_masks_of_counters_and_seeds():
    """Shares of kept elements within six standard deviations, of one mask and of both of two."""
    dev = device()
    n = 1 << 20
    x = torch.ones(n, device=dev)
    masks = [training.dropout(x, 0.25, seed=s, counter=c) != 0 for s, c in ((1, 0), (1, 1), (2, 0), (1, 1 << 32),
                                                                        (1 << 32, 0))]
    for i, a in enumerate(masks):
        share = float(a.float().mean())
        assert abs(share - 0.75) < 6 * math.sqrt(0.75 * 0.25 / n), share
        assert abs(float((a[1:] & a[:-1]).float().mean()) - 0.75 ** 2) < 6 * math.sqrt(0.25 / n)
        for b in masks[:i]:
            assert abs(float((a & b).float().mean()) - 0.75 ** 2) < 6 * math.sqrt(0.25 / n)


def test_dropped_places_may_hold_anything():
    dev = device()
    x = torch.randn(4096, generator=gen(3)).to(dev)
    kept = training.dropout(torch.ones_like(x), 0.5, seed=9) != 0
    odd = torch.where(kept, x, torch.tensor([float("nan"), float("inf")], device=dev).repeat(2048))
    assert torch.equal(training.dropout(odd, 0.5, seed=9), training.dropout(x, 0.5, seed=9))
    assert torch.equal(training.dropout(odd, 1.0, seed=9), torch.zeros_like(x))


def test_dropout_of_a_large_tensor():
    """Past 2^32 elements: the last ones against the oracle."""
    dev = device()
    n = (1 << 32) + 1000 * 8 + 3
    x = torch.ones(n, device=dev, dtype=torch.bfloat16)
    got = training.dropout(x, 0.5, seed=11, counter=2)
    for first in (0, (1 << 31) - 64, (1 << 32) - 64, (1 << 32) + 7936):
        part = got[first:first + 256].cpu()
        want, _ = ref.dropout(torch.ones(part.numel()), 0.5, 11, 2, first=first)
        assert torch.equal(part.double(), want), first


def test_dropout_refusals():
    dev = device()
    x = torch.ones(4, 6, device=dev)
    for error, match, args, kw in (
            (ValueError, "p must be", (x, 1.5), {"seed": 1}), (ValueError, "p must be", (x, float("nan")), {"seed": 1}),
            (ValueError, "seed must be", (x, 0.5), {"seed": -1}), (ValueError, "seed must be", (x, 0.5), {"seed": 1 << 64}),
            (ValueError, "counter must be", (x, 0.5), {"seed": 1, "counter": -1}),
            (HipError, "counter must be", (x, 0.5), {"seed": 1, "counter": torch.ones(1, device=dev)}),
            (HipError, "device tensor", (x, 0.5), {"seed": 1, "counter": torch.ones(1, dtype=torch.int64)}),
            (ValueError, "residual must be", (x, 0.5), {"seed": 1, "residual": x.half()}),
            (ValueError, "residual must be", (x, 0.5), {"seed": 1, "residual": x[:3]}),
            (HipError, "dropout_grad", (x.clone().requires_grad_(True), 0.5), {"seed": 1}),
            (HipError, "residual requires grad", (x, 0.5), {"seed": 1, "residual": x.clone().requires_grad_(True)}),
            (HipError, "must be float32", (x.double(), 0.5), {"seed": 1})):
        with pytest.raises(error, match=match):
            training.dropout(*args, **kw)


# ---------------------------------------------------------------------------
# streams, graphs, both together

def test_on_another_stream_and_in_a_graph():
    """A captured step, replayed with other tokens and a raised counter, between eager work: every replay as the eager
    call."""
    dev = device()
    hidden, weight, tokens, bias = (t.to(dev) for t in head(150, 128, 700, torch.bfloat16, 2))
    counter = torch.zeros((), dtype=torch.int64, device=dev)

    def step():
        x = training.dropout(hidden, 0.2, seed=3, counter=counter)
        r = training.vocabulary_loss(x, weight, tokens, bias=bias)
        return [*r, training.dropout_grad(r.grad_hidden, 0.2, seed=3, counter=counter)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(there, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    seen = []
    for turn in range(4):
        counter.fill_(turn)
        tokens.copy_(torch.randint(-1, 700, (150,), generator=gen(turn)))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), turn
        seen.append(captured[2].clone())
    assert not torch.equal(seen[0], seen[1])


def test_two_graphs():
    """Two captured calls of different sizes, replayed in turn beside eager ones: neither's workspace is the other's."""
    dev = device()
    cases = [[t.to(dev) for t in head(n, 128, v, dtype, n)] for n, v, dtype in
             ((150, 2000, torch.bfloat16), (7, 9000, torch.bfloat16), (100, 40, torch.float32))]
    run = lambda c: training.vocabulary_loss(c[0], c[1], c[2], bias=c[3], room=1 << 20)  # noqa: E731
    for c in cases:
        run(c)
    graphs, results = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(run(c))
    for turn in range(3):
        for c in cases:
            c[0].copy_(torch.randn(c[0].shape, generator=gen(turn)))
        for k in (0, 1, 2, 1, 0):
            graphs[k].replay()
        want = [run(c) for c in cases]
        torch.cuda.synchronize()
        for a, b in zip(results, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y), turn


def test_scores_feed_the_other_losses():
    """log-probabilities without gradients are those that the losses on logits compute."""
    dev = device()
    hidden, weight, tokens, bias = (t.to(dev) for t in head(44, 128, 301, torch.float32, 7))
    scored = training.vocabulary_loss(hidden, weight, tokens, bias=bias, with_grad=False).logp
    logits = torch.addmm(bias, hidden, weight.t())
    offsets = torch.tensor([0, 9, 20, 33, 44], device=dev)
    r = training.preference_loss(logits, tokens, scored, offsets)
    tol = (2 * 128 * 2.0 ** -24 * float((hidden.abs() @ weight.abs().t()).max() + 3) * 2 + 2.0 ** -17)
    assert float((r.logp - scored).abs().max()) < tol
    assert abs(float(r.loss) - math.log(2)) < 0.1 * 24 * tol


def test_calls_on_two_streams():
    """Two calls under way at once, and the same call twice: the bits of calls one after another."""
    dev = device()
    cases = [tuple(t.to(dev) for t in head(n, 256, 9000, torch.bfloat16, n)) for n in (300, 50)]
    run = lambda c: training.vocabulary_loss(c[0], c[1], c[2], bias=c[3])  # noqa: E731
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(c))
    torch.cuda.synchronize()
    for k, r in enumerate(got):
        for a, b in zip(r, want[k % 2]):
            assert torch.equal(a, b), k


def test_more_than_four_gigabytes():
    """A weight of 4.6 GB, and a softmax gradient of 8.7 GB where there is room: offsets past 32 bits."""
    dev = device()
    g = torch.Generator(device=dev).manual_seed(3)

    def check_rows(hidden, weight, tokens, got, rows, words, dtype):
        n = tokens.numel()
        size, tops = 0.0, []
        for i in rows:
            z = torch.mv(weight.float(), hidden[i].float()).double()      # fp32 sums of D products
            q = torch.log_softmax(z, 0)
            D = hidden.shape[1]
            size = (D + 8) * 2.0 ** -23 * float(torch.mv(weight.float().abs(), hidden[i].float().abs()).max())
            assert abs(float(got.logp[i]) - float(q[tokens[i]])) <= 4 * size + 2.0 ** -20 * (40 + z.numel() / 4096), i
            p = q.exp()
            p[tokens[i]] -= 1.0
            want = torch.mv(weight.t().float(), p.float()).double() / n
            bound = torch.mv(weight.t().float().abs(), p.float().abs()).double() / n
            tops.append((i, got.grad_hidden[i].double(), want, bound * (2 * U[dtype] + 4 * size + 2.0 ** -16)))
        for i, have, want, tol in tops:
            close(have.cpu(), want.cpu(), (tol + rounded(want, dtype)).cpu(), f"grad hidden of row {i}")
        # the weight's rows that are asked for, from all rows' probabilities of those tokens
        for v in words:
            z = torch.mv(hidden.float(), weight[v].float()).double()
            # the row's normaliser from its own token
            own = torch.stack([torch.dot(hidden[i].float(), weight[tokens[i]].float()) for i in range(n)]).double() \
                if n <= 100 else (hidden.float() * weight[tokens].float()).sum(1).double()
            p = torch.exp(z - (own - got.logp.double())) - (tokens == v).double()
            want = torch.mv(hidden.t().double(), p) / n
            bound = torch.mv(hidden.t().double().abs(), p.abs()) / n
            close(got.grad_weight[v].cpu(), want.cpu(), (bound * (2 * U[dtype] + 2.0 ** -12) + rounded(want, dtype)).cpu(),
                  f"grad weight of token {v}")

    V, D = 140_000, 16_384
    weight = torch.empty(V, D, device=dev, dtype=torch.bfloat16).normal_(0.0, 2.0 / math.sqrt(D), generator=g)
    tokens = torch.tensor([0, V - 1, 131_071, 131_073, 5], device=dev)
    hidden = torch.randn(5, D, device=dev, generator=g).bfloat16()
    got = training.vocabulary_loss(hidden, weight, tokens)
    check_rows(hidden, weight, tokens, got, range(5), (0, V - 1, 131_072, 131_073), torch.bfloat16)
    del weight, got
    N, V, D = 33_000, 131_072, 64
    weight = torch.empty(V, D, device=dev, dtype=torch.bfloat16).normal_(0.0, 0.25, generator=g)
    hidden = torch.randn(N, D, device=dev, generator=g).bfloat16()
    tokens = torch.randint(0, V, (N,), device=dev, generator=g)
    got = training.vocabulary_loss(hidden, weight, tokens, room=16 << 30)
    check_rows(hidden, weight, tokens, got, (0, 1, 32_767, 32_768, N - 1), (0, 65_536, V - 1, int(tokens[-1])), torch.bfloat16)


# ---------------------------------------------------------------------------
# the example

def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_and_verify.py")
    spec = importlib.util.spec_from_file_location("train_and_verify", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_supervised_step_against_autograd():
    """The step's gradients, chained through lookup, layers, dropout and loss, against float64 autograd with the oracle's
    mask.  fp32 throughout: products of up to 160 terms, a mean over 64 rows."""
    dev = device()
    ex = example()
    contexts = torch.randint(0, ex.VOCAB, (64, ex.CONTEXT), generator=gen(1)).to(dev)
    policy = ex.Policy(dev, seed=3)
    label = ex.right_action(contexts)
    params = [p.detach().double().cpu().requires_grad_(True) for p in policy.params]
    result, grads = policy.imitate(contexts, label, 0.25)
    net = copy.deepcopy(policy.net).double().cpu()
    table, w0, b0, w1, b1 = params
    x = (table[contexts.cpu()] * ex.SCALE).flatten(1)
    hidden = torch.relu(torch.nn.functional.linear(x, w0, b0))
    _, kept = ref.dropout(hidden.detach(), 0.25, 7, 0)
    logits = torch.nn.functional.linear(torch.where(kept, hidden / 0.75, 0.0), w1, b1)
    loss = torch.nn.functional.cross_entropy(logits, label.cpu())
    want = torch.autograd.grad(loss, params)
    assert len(list(net.parameters())) == 4
    # hidden and logits are sums of up to 160 products in fp32, off by 168 2^-24 of their magnitudes, some 1e-5 of
    # the values; gradients are means of 64 such terms, whose magnitudes are some ten times their sum
    assert abs(float(result.loss) - float(loss.detach())) < 2.0 ** -15
    for name, a, b in zip(("table", "w0", "b0", "w1", "b1"), grads, want):
        err = float((a.double().cpu() - b).abs().max())
        announce(f"supervised step: gradient of {name} off by {err:.2e} of {float(b.abs().max()):.2e}")
        assert err <= 2.0 ** -13 * float(b.abs().max()), name


def test_example_with_a_supervised_stage():
    got = example().main(["--steps", "2", "--contexts", "64", "--eps", "0.02", "--imitate", "5"])
    assert len(got["imitated"]) == 5 and all(math.isfinite(x) for x in (*got["imitated"], *got["losses"]))
    assert 0.0 <= got["after"][1] <= got["after"][0] <= 1.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V", [(6, 130), (6, 33_001), (100, 130), (100, 8300)])
def test_far_temperatures(dtype, N, V):
    """The largest temperature leaves all tokens alike, the least the largest logit alone; padded entries stay out of both."""
    dev = device()
    hidden, weight, tokens, bias = (t.to(dev) for t in head(N, 64, V, dtype, 2))
    bias[1] = float("-inf")
    tokens = torch.where(tokens == 1, 2, tokens)
    got = training.vocabulary_loss(hidden, weight, tokens, bias=bias, temperature=2.0 ** 120)
    # a sum of V - 1 equal terms in fp32, V / 256 of them one after another, and its logarithm
    tol = (V / 256 + 16) * 2.0 ** -24 + 2.0 ** -23 * math.log(V)
    close(got.logp, torch.full((N,), -math.log(V - 1), dtype=torch.float64), tol, "all alike")
    assert all(bool(torch.isfinite(t).all()) for t in got)
    z = torch.mm(hidden.float(), weight.float().t()) + bias.float()
    top = z.argmax(1)
    got = training.vocabulary_loss(hidden, weight, top, bias=bias, temperature=2.0 ** -120)
    assert not bool(got.logp.any()), "the largest logit has all the probability"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V", [(128, 9000), (200, 9000), (600, 10_001), (600, 20_001)])
def test_bias_gradient_of_every_piece_is_summed_before_rounding(dtype, N, V):
    """Rows that answer tokens as often as their probabilities say: a token's column of G cancels to what the bias's rounding
    leaves, and G's own rounding, the same in all rows, would be as large as that.  So it has no place in the tolerance: the
    exponentials of the first piece are rounded to 11 bits in 16-bit types, what follows is formed in fp32."""
    dev = device()
    D = 72
    ids = torch.tensor([3, 70, 255, 256, 700, 2049, 4100, 4101, 5000, 8000, V - 257, V - 1])
    share = torch.rand(len(ids), generator=gen(3)) + 0.2
    tokens = ids[torch.multinomial(share, N, replacement=True, generator=gen(4))]
    often = torch.bincount(tokens, minlength=V).double() / N
    bias = often.log().to(dtype)
    weight = torch.randn(V, D, generator=gen(5)).to(dtype)
    hidden = torch.zeros(N, D, dtype=dtype)
    r = ref.vocabulary_loss(hidden, weight, tokens, bias=bias)
    got = training.vocabulary_loss(hidden.to(dev), weight.to(dev), tokens.to(dev), bias=bias.to(dev), room=0)
    tol_lp = 2.0 ** -23 * float(r["size"].max()) + logp_tol(r["z"], V)
    tol_g = r["p"] * (tol_lp + 2.0 ** -21)[:, None] + r["g"].abs() * 2.0 ** -23
    if dtype != torch.float32:
        tol_g[:, :256] += r["p"][:, :256] * 2.0 ** -11       # the first piece: what is left of no room
    tol = r["factor"] * (tol_g.sum(0) + (N + 8) * 2.0 ** -24 * r["g"].abs().sum(0))
    close(got.grad_bias, r["bias"], tol + rounded(r["bias"], dtype), f"grad bias of pieces {N} x {V} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_exponentials_kept_and_logits_formed_again(dtype):
    """G in one part.  Where the exponentials are kept, in the first piece, they have 11 bits before G is rounded; in the others,
    whose logits are formed again, G is rounded alone: the weight's gradient there is held to the lesser error."""
    dev = device()
    N, D, V = 100, 128, 9000
    for room, border in ((2 << 30, V), (0, 256)):
        pieces, _, _, parts, summed, _ = vocab_cases.plan(N, D, V, 0, True, room, dtype)
        assert (pieces > 1, parts, summed) == (border < V, 1, 0)
    hidden, weight, tokens, bias = head(N, D, V, dtype, 23)
    r = ref.vocabulary_loss(hidden, weight, tokens, bias=bias)
    whole = check(hidden, weight, tokens, bias=bias)
    cut = check(hidden, weight, tokens, bias=bias, room=0)
    assert torch.equal(whole.logp, cut.logp) and torch.equal(whole.loss, cut.loss)
    assert torch.equal(whole.grad_weight[:256], cut.grad_weight[:256]) and torch.equal(whole.grad_bias[:256], cut.grad_bias[:256])
    _, tol_g = tolerances(r, dtype, 1.0, V, D)
    tol_g = tol_g - r["p"] * 2.0 ** -11
    g, x = r["g"].abs(), r["x"].abs()
    tol = r["factor"] * (torch.mm(tol_g.t(), x) + (N + 8) * 2.0 ** -24 * torch.mm(g.t(), x)) + rounded(r["weight"], dtype)
    close(cut.grad_weight[256:], r["weight"][256:], tol[256:], f"grad weight past the first piece {dtype}")


@pytest.mark.parametrize("N,V", [(5, 300), (5, 40_001), (200, 300), (200, 9000)])
def test_the_largest_fp32_values(N, V):
    """Finite values past the largest bf16, 3.39e38, whose first of three bf16 parts would round to infinity: in a hidden row
    and in a weight's, against 2^-100, at a temperature that brings their logits down to a few."""
    hidden, weight, tokens, bias = head(N, 72, V, torch.float32, 15)
    most = torch.finfo(torch.float32).max
    weight[:, 3] = torch.randn(V, generator=gen(1)) * 2.0 ** -100
    hidden[:, 5] = torch.randn(N, generator=gen(2)) * 2.0 ** -100
    hidden[1, 3], hidden[2, 3] = most, -3.395e38
    weight[7, 5], weight[V - 1, 5] = -most, 3.4e38
    dev, T, dtype = device(), 2.0 ** 26, torch.float32
    r = ref.vocabulary_loss(hidden, weight, tokens, bias=bias, temperature=T)
    got = training.vocabulary_loss(*(t.to(dev) for t in (hidden, weight, tokens)), bias=bias.to(dev), temperature=T)
    tol_lp, tol_g = tolerances(r, dtype, T, V, 72)
    close(got.logp, r["logp"], tol_lp + 2.0 ** -23 * r["logp"].abs(), f"logp of the largest values {N} x {V}")
    g = r["g"].abs()

    def held(have, want, a, b, terms, name):
        """A gradient's sum is multiplied by 1 / (T N) at its end.  No partial sum is past the sum of the magnitudes and the
        roundings, terms 2^-24 of it, so below 2^128 (1 - 2^-9) of that nothing is infinite; of the few entries beyond, two
        rows or tokens of 2^128 in one sum, nothing is said."""
        size = torch.mm(a.abs(), b.abs())
        tol = r["factor"] * (torch.mm(tol_g if a is g else tol_g.t(), b.abs()) + terms * 2.0 ** -24 * size)
        beyond = size * (1 + terms * 2.0 ** -24) > most * (1 - 2.0 ** -9)
        assert int(beyond.sum()) <= max(N, V) // 4, "the test has nothing to look at"
        close(torch.where(beyond.to(dev), 0.0, have), torch.where(beyond, 0.0, want), tol + rounded(want, dtype), name)

    held(got.grad_hidden, r["hidden"], g, r["w"], 6 * V + 8, f"grad hidden of the largest values {N} x {V}")
    held(got.grad_weight, r["weight"], g.t(), r["x"], 6 * N + 8, f"grad weight of the largest values {N} x {V}")
    close(got.grad_bias, r["bias"], r["factor"] * (tol_g.sum(0) + (6 * N + 8) * 2.0 ** -24 * g.sum(0)) + rounded(r["bias"], dtype),
          f"grad bias of the largest values {N} x {V}")


@pytest.mark.parametrize("N,dtype", [(300, torch.bfloat16), (600, torch.float32)])
def test_a_captured_call_past_the_room(N, dtype):
    """Pieces of the vocabulary with the bias's columns summed in each: replays between eager calls, other inputs each time."""
    dev = device()
    V = 9000
    inputs = [t.to(dev) for t in head(N, 72, V, dtype, 21)]
    call = lambda: training.vocabulary_loss(*inputs[:3], bias=inputs[3], room=1 << 20)  # noqa: E731
    pieces, _, _, _, _, columns = vocab_cases.plan(N, 72, V, 0, True, 1 << 20, dtype)
    assert pieces > 1 and columns
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for turn in range(3):
        for t, other in zip(inputs, head(N, 72, V, dtype, turn)):
            t.copy_(other)
        inputs[2][turn::5] = -1
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), turn
        again = call()
        for a, b in zip(again, want):
            assert torch.equal(a, b), turn
