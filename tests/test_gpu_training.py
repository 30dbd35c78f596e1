"""The training operators against plain float64 restatements (oracle/training_ref.py).

Tolerances are those of the arithmetic: u is the unit roundoff of a type (half the spacing at 1),
results are rounded once to their type, sums are fp32 in an order of the kernel's choosing, and
a log-probability is off by what its exponent's rounding, the sum and the logarithm leave."""

import math

import pytest
import torch

from boundflow_amd import training
from boundflow_amd._lib import HipError
from oracle import training_ref as ref
from tests.gpu_util import announce, device

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} vs {tuple(want.shape)}"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    d = (got - want).abs()
    bad = (d > tol) & ~torch.isnan(want) & (got != want)
    announce(f"{what}: max abs err {float(d[~torch.isnan(d)].max()) if d.numel() else 0.0:.2e}, "
             f"outside {int(bad.sum())}/{d.numel()}")
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} elements outside their tolerance"


def rounded(want, dtype):
    return want.abs() * (U[dtype] + 2.0 ** -22) + TINY[dtype]


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------
# embedding

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,vocab,dim", [((0,), 5, 8), ((1,), 1, 1), ((7,), 9, 5), ((3, 4), 17, 8),
                                             ((300,), 50, 33), ((2, 65), 1000, 130), ((9,), 11, 257), ((5,), 6, 4096)])
def test_embed_tokens(dtype, shape, vocab, dim):
    dev = device()
    g = gen(dim)
    table = torch.randn(vocab, dim, generator=g).to(dtype)
    tokens = torch.randint(-1, vocab + 1, shape, generator=g)     # padding and tokens past the table among them
    want = ref.embed_tokens(table, tokens, 3.5)
    got = training.embed_tokens(table.to(dev), tokens.to(dev), scale=3.5)
    assert got.dtype == dtype
    close(got, want, rounded(want, dtype), f"embed {shape} x {dim} {dtype}")
    assert torch.equal(training.embed_tokens(table.to(dev), tokens.int().to(dev), scale=3.5).nan_to_num(7.0),
                       got.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_embed_tokens_reads_views_in_place(dtype):
    dev = device()
    g = gen(1)
    whole = torch.randn(40, 71, generator=g).to(dtype).to(dev)
    table = whole[:, 1:66]                                          # rows at odd addresses, a stride of its own
    tokens = torch.randint(0, 40, (20, 3), generator=g).to(dev)[:, ::2]
    want = ref.embed_tokens(table.cpu(), tokens.cpu(), 1.0)
    close(training.embed_tokens(table, tokens), want, rounded(want, dtype), "embed of a view")


def grad_case(kind, count, vocab, g):
    if kind == "spread":
        return torch.randint(0, vocab, (count,), generator=g)
    if kind == "one":
        return torch.full((count,), vocab - 1)
    if kind == "hot":       # two values hold most of the batch, the others are rare
        t = torch.randint(0, vocab, (count,), generator=g)
        pick = torch.rand(count, generator=g)
        return torch.where(pick < 0.5, vocab // 2, torch.where(pick < 0.8, 0, t))
    return torch.randint(-2, vocab + 2, (count,), generator=g)       # "outside": some take no part


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,count,vocab,dim", [
    ("spread", 0, 3, 8), ("spread", 1, 1, 1), ("one", 64, 5, 9), ("one", 65, 5, 9), ("one", 700, 3, 40),
    ("hot", 900, 1003, 129), ("hot", 129, 300, 8), ("outside", 333, 31, 65), ("spread", 500, 70001, 6),
    ("hot", 5000, 513, 36), ("outside", 64, 1, 300), ("hot", 1100, 40, 2050)])
def test_embed_tokens_grad(dtype, kind, count, vocab, dim):
    dev = device()
    g = gen(count + dim)
    tokens = grad_case(kind, count, vocab, g)
    rows = torch.randn(count, dim, generator=g).to(dtype)
    want, size, n = ref.embed_tokens_grad(rows, tokens, vocab, 0.7)
    for out_type in {dtype, torch.float32}:
        got = training.embed_tokens_grad(rows.to(dev), tokens.to(dev), vocab, scale=0.7, dtype=out_type)
        assert got.dtype == out_type
        close(got, want, rounded(want, out_type) + size * n * 2.0 ** -23, f"embed grad {kind} {count} {out_type}")
        again = training.embed_tokens_grad(rows.to(dev), tokens.int().to(dev), vocab, scale=0.7, dtype=out_type)
        assert torch.equal(got, again), "another call, other bits"
    start = torch.randn(vocab, dim, generator=g)
    running = start.to(dev)
    version = running._version
    got = training.embed_tokens_grad(rows.to(dev), tokens.to(dev), vocab, scale=0.7, accumulate_into=running)
    assert got is running and running._version > version
    close(got, start.double() + want, (start.double().abs() + size) * (n + 2) * 2.0 ** -23, "embed grad, added")
    untouched = (n[:, 0] == 0)
    assert torch.equal(running.cpu()[untouched], start[untouched])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,count,vocab,dim", [
    ("hot", 900, 1003, 1601), ("hot", 2048, 9000, 1100), ("outside", 777, 5000, 1537), ("spread", 800, 70001, 771)])
def test_embed_tokens_grad_of_few_tokens_in_wide_rows(dtype, kind, count, vocab, dim):
    test_embed_tokens_grad(dtype, kind, count, vocab, dim)


def test_embed_tokens_grad_of_views():
    dev = device()
    g = gen(5)
    whole = torch.randn(6, 10, 37, generator=g).bfloat16().to(dev)
    rows, tokens = whole[:, 1:, 2:35], torch.randint(0, 12, (6, 9), generator=g)
    want, size, n = ref.embed_tokens_grad(rows.cpu(), tokens, 12, 1.0)
    close(training.embed_tokens_grad(rows, tokens.to(dev), 12), want,
          rounded(want, torch.bfloat16) + size * n * 2.0 ** -23, "embed grad of a view")
    flat = whole.view(60, 37)[:, 3:20]
    want, size, n = ref.embed_tokens_grad(flat.cpu(), tokens.new_ones(60), 2, 1.0)
    close(training.embed_tokens_grad(flat, torch.ones(60, dtype=torch.int64, device=dev), 2), want,
          rounded(want, torch.bfloat16) + size * n * 2.0 ** -23, "embed grad of rows with a stride")


# ---------------------------------------------------------------------------
# losses

def logp_tol(z, V):
    """What a log-probability may be off: the exponents' roundings and that of log2(e) / T (2^-23 of the
    row's spread), those of the sum (a thread's terms one after another, then trees), the logarithm."""
    finite = torch.where(torch.isfinite(z) & (z.abs() < 1e30), z, torch.zeros((), dtype=z.dtype)).double()
    spread = finite.amax(-1) - finite.amin(-1)
    return 2.0 ** -22 * (spread + math.log(V) + 2) + (V / 256 + 64) * 2.0 ** -24


def grad_tol(want, r, extra, tol_lp, inv_t, dtype):
    """|error| of g / T (onehot - softmax): g off by `extra`, the softmax by its log-probabilities' tolerance."""
    part = r["p"] + 0.0
    part.scatter_add_(-1, r["token"][..., None], torch.ones_like(r["p"][..., :1]))
    return 2 * inv_t * (extra + r["g"].abs() * (tol_lp + 2.0 ** -22))[..., None] * part + rounded(want, dtype)


def policy_inputs(B, T, V, dtype, seed, kl, mask_kind):
    g = gen(seed)
    logits = (torch.randn(B, T + 1, V, generator=g) * 3).to(dtype)[:, :-1]
    tokens = torch.randint(0, V, (B, T), generator=g)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, tokens[..., None])[..., 0]
    drift = torch.randn(B, T, generator=g) * 0.2
    for limit in (math.log(0.8), math.log(1.28)):     # no ratio so near a limit that rounding decides
        drift = torch.where((drift - limit).abs() < 5e-3, limit + 0.01, drift)
    s = dict(logits=logits, tokens=tokens, old_logp=(lp - drift).float(), advantages=torch.randn(B, T, generator=g),
             ref_logp=(lp + torch.randn(B, T, generator=g) * 0.4).float() if kl else None, mask=None)
    if mask_kind != "none":
        s["mask"] = torch.rand(B, T, generator=g) < 0.7
        if mask_kind == "empty":
            s["mask"][:] = False
        elif mask_kind == "sequence":
            s["mask"][0] = False
    return s


def check_policy(s, dev, *, temperature=1.0, reduction="token", kl_weight=0.05, grad_scale=1.0, what=""):
    kw = dict(clip_low=0.2, clip_high=0.28, kl_weight=kl_weight, temperature=temperature, reduction=reduction,
              grad_scale=grad_scale)
    shift = {}
    if temperature != 1.0:   # sampled at that temperature: ratios keep their distance from the limits
        t = s["tokens"].clamp(min=0)[..., None]
        plain = torch.log_softmax(s["logits"].double(), -1).gather(-1, t)[..., 0]
        warm = torch.log_softmax(s["logits"].double() / temperature, -1).gather(-1, t)[..., 0]
        shift = {k: (s[k].double() - plain + warm).float() for k in ("old_logp", "ref_logp") if s[k] is not None}
    s = {**s, **shift}
    r = ref.policy_loss(**s, **kw)
    whole = torch.empty(s["logits"].shape[0], s["logits"].shape[1] + 1, s["logits"].shape[2], dtype=s["logits"].dtype)
    whole[:, :-1] = s["logits"]
    whole[:, -1] = float("nan")
    on = {k: v.to(dev) if v is not None else None for k, v in s.items()}
    on["logits"] = whole.to(dev)[:, :-1]           # read in place, a row of NaN after every sequence
    got = training.policy_loss(**on, **kw)
    dtype = s["logits"].dtype
    V = s["logits"].shape[-1]
    tol_lp = torch.where(r["live"], logp_tol(s["logits"] / temperature, V), torch.zeros((), dtype=torch.float64))
    close(got.logp, r["logp"], tol_lp + 2.0 ** -24 * r["logp"].abs(), f"policy logp {what}")
    N = r["g"].numel()
    r["token"] = s["tokens"].clamp(min=0)
    extra = r["slope"] * (tol_lp + 2.0 ** -22)
    want = r["grad"]
    close(got.grad_logits, want, grad_scale * grad_tol(want / grad_scale, r, extra, tol_lp, 1 / temperature, dtype)
          + TINY[dtype], f"policy grad {what}")
    # every term moves by at most its slope, and is summed in fp32
    slack = float((r["slope"] * tol_lp).sum()) + (N / 256 + 32) * 2.0 ** -23 * float((r["slope"] + r["g"].abs()).sum() + 1)
    close(got.stats, r["stats"], slack, f"policy stats {what}")
    assert float(got.loss) == float(got.stats[0])
    alone = training.policy_loss(**on, **kw, with_grad=False)
    assert alone.grad_logits is None and torch.equal(alone.stats, got.stats) and torch.equal(alone.logp, got.logp)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (2, 3, 5), (3, 7, 129), (1, 2, 4097), (4, 33, 1000), (1, 1, 70001),
                                   (2, 5, 32771), (70, 9, 64), (1, 700, 2050)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss(dtype, B, T, V, reduction):
    dev = device()
    for k, (kl, mask) in enumerate([(True, "none"), (False, "some"), (True, "sequence"), (True, "empty")]):
        s = policy_inputs(B, T, V, dtype, 100 * B + T + k, kl, mask)
        check_policy(s, dev, reduction=reduction, temperature=[1.0, 0.8, 1.0, 1.7][k],
                     grad_scale=[1.0, 64.0, 0.5, 1.0][k], what=f"{B}x{T}x{V} {mask}")


@pytest.mark.parametrize("dtype", TYPES)
def test_policy_loss_of_masked_vocabulary_and_odd_rows(dtype):
    """-inf and the type's lowest value in masked entries; rows that hold nothing but the lowest value (uniform)
    or very small logits; a padded row of NaN; negative tokens."""
    dev = device()
    s = policy_inputs(3, 6, 301, dtype, 3, True, "some")
    lowest = torch.finfo(dtype).min
    z = s["logits"].clone()
    z[0, 0, 50:] = float("-inf")
    s["tokens"][0, 0] = 7
    z[0, 1, :290] = lowest
    s["tokens"][0, 1] = 295
    z[0, 2] = lowest
    z[0, 3, 8:] = -300.0
    z[0, 3, :8] = float("-inf")
    s["tokens"][0, 3] = 100
    z[0, 4] = lowest
    z[0, 4, ::3] = float("-inf")
    s["tokens"][0, 4] = 1
    s["mask"][0, :5] = True
    s["tokens"][1, 2] = -1
    s["mask"][1, 2] = True
    s["mask"][2, 3] = False
    lp = torch.log_softmax(z.double(), -1).gather(-1, s["tokens"].clamp(min=0)[..., None])[..., 0]
    s["old_logp"], s["ref_logp"] = (lp - 0.03).float(), (lp + 0.1).float()
    z[2, 3] = float("nan")
    s["logits"] = z
    check_policy(s, dev, what="odd rows")


def test_policy_loss_shows_what_is_not_a_number():
    dev = device()
    s = policy_inputs(1, 4, 40, torch.float32, 9, True, "none")
    s["logits"] = s["logits"].clone()
    s["logits"][0, 0, 3] = float("nan")
    s["logits"][0, 1, 3] = float("inf")
    s["logits"][0, 2] = float("-inf")
    s["tokens"][0, 3] = 40
    got = training.policy_loss(**{k: v.to(dev) if v is not None else None for k, v in s.items()}, kl_weight=0.05)
    assert torch.isnan(got.logp).all() and torch.isnan(got.loss)
    assert torch.isnan(got.grad_logits[0, :3]).all()


def test_policy_loss_of_flat_rows_and_broadcast_advantages():
    dev = device()
    s = policy_inputs(5, 4, 77, torch.bfloat16, 21, True, "some")
    one = torch.randn(5, generator=gen(2))
    s["advantages"] = one[:, None].expand(5, 4)
    want = check_policy(s, dev, what="expanded advantages")
    on = {k: v.to(dev) if v is not None else None for k, v in s.items()}
    kw = dict(clip_low=0.2, clip_high=0.28, kl_weight=0.05)
    got = training.policy_loss(**{**on, "advantages": one.to(dev)}, **kw)
    assert torch.equal(got.grad_logits, want.grad_logits)
    flat = {k: v.reshape(20, *v.shape[2:]) if v is not None else None for k, v in on.items()}
    got = training.policy_loss(**flat, **kw)
    assert got.logp.shape == (20,)
    close(got.grad_logits.view(5, 4, 77), want.grad_logits.double().cpu(),
          2.0 ** -20 * want.grad_logits.double().cpu().abs() + rounded(want.grad_logits.double().cpu(), torch.bfloat16) * 2,
          "flat rows")


def test_policy_gradient_against_differences():
    """Central differences of the float64 loss: the gradient is the formula's, and the formula is the loss's."""
    dev = device()
    s = policy_inputs(2, 3, 7, torch.float32, 31, True, "some")
    kw = dict(clip_low=0.2, clip_high=0.28, kl_weight=0.3, temperature=1.0, reduction="sequence")
    got = training.policy_loss(**{k: v.to(dev) if v is not None else None for k, v in s.items()}, **kw)
    z, h = s["logits"].double(), 1e-5
    want = torch.zeros_like(z)
    for i in range(z.numel()):
        e = torch.zeros(z.numel(), dtype=torch.float64)
        e[i] = h
        up, down = (ref.policy_loss(**{**s, "logits": z + d * e.view(z.shape)}, **kw)["stats"][0] for d in (1, -1))
        want.view(-1)[i] = (up - down) / (2 * h)
    # the differences' own error is h^2 times the third derivative (below 10 here)
    close(got.grad_logits, want, 2e-6 * want.abs().max() + 10 * h * h, "policy gradient against differences")


def preference_inputs(lengths, V, dtype, seed, before=0, after=0):
    g = gen(seed)
    N = before + sum(lengths) + after
    logits = (torch.randn(N, V, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, V, (N,), generator=g)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, tokens[:, None])[:, 0] if N else torch.zeros(0)
    offsets = torch.tensor([before] + lengths).cumsum(0)
    return dict(logits=logits, tokens=tokens, ref_logp=(lp + torch.randn(N, generator=g) * 0.5).float(), offsets=offsets)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,V", [([1, 1], 1), ([3, 2], 5), ([0, 4, 2, 0], 130), ([300, 1, 7, 40], 1000),
                                       ([2, 3], 70001), ([5, 0, 1, 9, 2, 600], 2049), ([0, 0], 9)])
def test_preference_loss(dtype, lengths, V):
    dev = device()
    for beta, smoothing, scale, before, after in ((0.1, 0.0, 1.0, 0, 0), (0.5, 0.1, 8.0, 2, 3)):
        s = preference_inputs(lengths, V, dtype, V + len(lengths), before, after)
        if len(lengths) == 6:
            s["tokens"][before + 2] = -1
        kw = dict(beta=beta, label_smoothing=smoothing, grad_scale=scale)
        r = ref.preference_loss(**s, **kw)
        got = training.preference_loss(**{k: v.to(dev) for k, v in s.items()}, **kw)
        tol_lp = logp_tol(s["logits"], V) if len(s["tokens"]) else torch.zeros(0)
        close(got.logp, r["logp"], tol_lp + 2.0 ** -24 * r["logp"].abs(), "preference logp")
        # a response's sum moves by its rows' tolerances, and is summed in fp32
        bounds = s["offsets"].tolist()
        moved = torch.stack([beta * (tol_lp[a:b].sum() + (b - a + 8) * 2.0 ** -23
                                     * (r["logp"] - s["ref_logp"].double())[a:b].abs().sum())
                             for a, b in zip(bounds, bounds[1:])])
        close(got.rewards, r["rewards"], moved + 2.0 ** -22 * r["rewards"].abs(), "preference rewards")
        pairs = len(lengths) // 2
        apart = moved[:pairs] + moved[pairs:] + 2.0 ** -22 * (r["rewards"][:pairs].abs() + r["rewards"][pairs:].abs())
        close(got.loss, r["loss"], float(apart.mean()) + 2.0 ** -20 * float(r["loss"]) + 2.0 ** -22, "preference loss")
        # |dg| <= beta |dh| / 4 per pair (sigma' <= 1/4), and sigma's own rounding
        owner = torch.zeros(len(s["tokens"]), dtype=torch.long)
        for k, (a, b) in enumerate(zip(bounds, bounds[1:])):
            owner[a:b] = k % pairs
        h = r["rewards"][:pairs] - r["rewards"][pairs:]
        g = -((1 - smoothing) * torch.sigmoid(-h) - smoothing * torch.sigmoid(h)) * beta / pairs
        extra = (beta / pairs * (apart / 4 + 2.0 ** -21 * (torch.sigmoid(-h) + smoothing)))[owner]
        live = r["live"].double()
        r["g"], r["token"] = g[owner] * live, s["tokens"].clamp(min=0)
        close(got.grad_logits, r["grad"], scale * grad_tol(r["grad"] / scale, r, extra * live, tol_lp, 1.0, dtype)
              + TINY[dtype], "preference grad")
        alone = training.preference_loss(**{k: v.to(dev) for k, v in s.items()}, **kw, with_grad=False)
        assert alone.grad_logits is None and torch.equal(alone.loss, got.loss)


@pytest.mark.parametrize("dtype,V", [(torch.float32, 4097), (torch.bfloat16, 8192), (torch.bfloat16, 16391),
                                     (torch.float16, 33001), (torch.float32, 20003)])
def test_preference_loss_of_many_long_rows(dtype, V):
    """Batches of many long rows: responses of very different lengths, empty ones, a pair without a row, rows of no
    response, padding tokens, and rows that start at odd elements."""
    for lengths in ([260, 0, 1, 40, 90, 0, 131, 7], [600, 3], [0] * 30 + [5, 250] * 3 + [0] * 30 + [80, 1] * 3):
        test_preference_loss(dtype, lengths, V)
        dev = device()
        s = preference_inputs(lengths, V, dtype, 77, 1, 2)
        s["tokens"][::7] = -1
        on = {k: v.to(dev) for k, v in s.items()}
        r = ref.preference_loss(**s)
        got = training.preference_loss(**on)
        tol_lp = logp_tol(s["logits"], V)
        close(got.logp, r["logp"], tol_lp + 2.0 ** -24 * r["logp"].abs(), "preference logp with padding")
        assert not got.grad_logits[::7].any() and not got.grad_logits[-2:].any()
        again = training.preference_loss(**on)
        assert torch.equal(got.grad_logits, again.grad_logits) and torch.equal(got.rewards, again.rewards)
        alone = training.preference_loss(**on, with_grad=False)
        close(alone.rewards, got.rewards.double().cpu(), 0.1 * float(tol_lp.sum()) + 2.0 ** -20, "rewards alone")


def test_preference_loss_without_pairs_and_with_offsets_out_of_range():
    dev = device()
    s = preference_inputs([4, 3], 20, torch.float32, 4)
    on = {k: v.to(dev) for k, v in s.items()}
    got = training.preference_loss(**{**on, "offsets": torch.zeros(1, dtype=torch.int64, device=dev)})
    assert float(got.loss) == 0.0 and not got.grad_logits.any() and got.rewards.numel() == 0
    # rows that are not there are not read
    wide = training.preference_loss(**{**on, "offsets": torch.tensor([-5, 4, 900], device=dev)})
    want = training.preference_loss(**on)
    assert torch.equal(wide.loss, want.loss) and torch.equal(wide.grad_logits, want.grad_logits)


def test_preference_gradient_against_differences():
    dev = device()
    s = preference_inputs([2, 1, 1, 2], 5, torch.float32, 8)
    kw = dict(beta=0.7, label_smoothing=0.2)
    got = training.preference_loss(**{k: v.to(dev) for k, v in s.items()}, **kw)
    z, h = s["logits"].double(), 1e-5
    want = torch.zeros_like(z)
    for i in range(z.numel()):
        e = torch.zeros(z.numel(), dtype=torch.float64)
        e[i] = h
        up, down = (ref.preference_loss(**{**s, "logits": z + d * e.view(z.shape)}, **kw)["loss"] for d in (1, -1))
        want.view(-1)[i] = (up - down) / (2 * h)
    close(got.grad_logits, want, 2e-6 * want.abs().max() + 10 * h * h, "preference gradient against differences")


# ---------------------------------------------------------------------------
# AdamW

HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def adamw_params(sizes, dtype, dev, seed, odd):
    """Weights as views of one buffer; with `odd` they start at any element."""
    g = gen(seed)
    gap = 1 if odd else 64
    flat = torch.randn(sum(sizes) + gap * (len(sizes) + 1), generator=g).to(dtype).to(dev)
    out, at = [], gap
    for n in sizes:
        out.append(flat[at:at + n])
        at += n + gap if odd else -(-(n + gap) // 64) * 64
        if not odd and at + max(sizes, default=0) > flat.numel():
            flat = torch.randn(flat.numel() * 2 + max(sizes), generator=g).to(dtype).to(dev)
            at = gap
    return out


@pytest.mark.parametrize("p_type", TYPES)
@pytest.mark.parametrize("g_type", TYPES)
@pytest.mark.parametrize("master", [False, True])
def test_adamw_in_32_bits(p_type, g_type, master):
    dev = device()
    for sizes, odd in (([1], False), ([127, 128, 129, 0, 5], True), ([5000, 3, 2048, 2049], False), ([7] * 130, True)):
        params = adamw_params(sizes, p_type, dev, 1, odd)
        opt = training.AdamW(params, **HYPER, master=master)
        w = [p.double().cpu() for p in params]
        m, v = ([torch.zeros(n, dtype=torch.float64) for n in sizes] for _ in range(2))
        for step in (1, 2, 3):
            grads = [g * 1e-2 for g in adamw_params(sizes, g_type, dev, 10 + step, odd)]
            factor = torch.tensor(0.6, device=dev) if step == 2 else 0.5
            before = [p.double().cpu() for p in params]
            versions = [p._version for p in params]
            opt.step(grads, grad_scale=factor)
            assert all(p._version > a for p, a in zip(params, versions))
            for k in range(len(sizes)):
                base = w[k] if master else before[k]
                g = grads[k].double().cpu() * float(factor)
                w[k], m[k], v[k] = ref.adamw(base, g, m[k], v[k], step=step, **HYPER)
                gm, gv = opt.moment(k)
                # three roundings a step of a sum of like terms, and of the constants
                close(gm, m[k], step * 2.0 ** -21 * (m[k].abs() + g.abs() + 1e-2), f"m {k} step {step}")
                close(gv, v[k], step * 2.0 ** -21 * (v[k] + g * g + 1e-4), f"v {k} step {step}")
                # an update is at most lr / (1 - b1) large; m off by its tolerance moves it by lr times that over sqrt(v)
                tol = 2.0 ** -22 * base.abs() + HYPER["lr"] * 1e-4 + TINY[p_type]
                if master:
                    at = training.moment_offsets(sizes)[k]
                    close(opt.moments.master[at:at + sizes[k]], w[k], step * tol, f"master {k} step {step}")
                close(params[k], w[k], step * tol + U[p_type] * w[k].abs(), f"w {k} step {step}")


@pytest.mark.parametrize("p_type,g_type,master", [(torch.float32, torch.float32, False),
                                                  (torch.bfloat16, torch.bfloat16, False),
                                                  (torch.bfloat16, torch.float32, True),
                                                  (torch.float16, torch.float16, True)])
def test_adamw_in_8_bits(p_type, g_type, master):
    """One step from what the moments stand for: the weights as in 32 bits, the new moments the numbers that the
    rounding names (where a magnitude lies within its own rounding error of the cut, the one beside it)."""
    dev = device()
    for sizes, odd in (([1], False), ([127, 128, 129, 0, 5], True), ([5000, 3, 2048], False), ([9] * 100, True)):
        params = adamw_params(sizes, p_type, dev, 2, odd)
        opt = training.AdamW(params, **HYPER, bits=8, master=master)
        at = training.moment_offsets(sizes)
        for step in (1, 2, 3, 4):
            grads = [g * 1e-2 for g in adamw_params(sizes, g_type, dev, 20 + step, odd)]
            w = [p.double().cpu() for p in params]
            if master:
                w = [opt.moments.master[a:a + n].double().cpu() for a, n in zip(at, sizes)]
            old = [opt.moment(k) for k in range(len(sizes))]
            opt.step(grads)
            new_m, new_r = (torch.zeros(at[-1], dtype=torch.float64) for _ in range(2))
            for k, n in enumerate(sizes):
                m0, v0 = (x.double().cpu() for x in old[k])
                want, m, v = ref.adamw(w[k], grads[k].double().cpu(), m0, v0, step=step, **HYPER)
                new_m[at[k]:at[k] + n], new_r[at[k]:at[k] + n] = m, v.sqrt()
                close(params[k], want, 2.0 ** -21 * w[k].abs() + HYPER["lr"] * 1e-4 + U[p_type] * want.abs() + TINY[p_type],
                      f"w {k} step {step}")
            phase = ref.phases(at[-1], step)
            for name, x, root in (("m", new_m, False), ("v", new_r, True)):
                count, spacing, scale = ref.hold(x, phase, root)
                held = getattr(opt.moments, name).float().cpu().double()
                got_scale = getattr(opt.moments, name + "_scale").double().cpu()
                close(got_scale, scale, 2.0 ** -20 * scale, f"{name} scale")
                got = held.abs() / spacing
                # the magnitude carries 2^-21 of rounding, so its count of spacings (16 at most) 2^-17
                near = (count - count.round()).abs() < 2.0 ** -16
                beside = (got - count.floor()).abs() <= 1.0001
                ok = torch.where(near, beside, got == count.floor()) | (held.abs() == 448)
                assert bool(ok.all()), f"{name}: {int((~ok).sum())} of {ok.numel()} held as another number"
                assert bool((torch.sign(held) * torch.sign(x) >= 0).all())
                if root:
                    assert bool((held[x > 0] > 0).all()), "a root held as zero"


def test_adamw_in_8_bits_follows_a_slow_average():
    """400 steps at beta2 = 0.99 of steady gradients, one of a block with a burst of 100 at step 20, whose decay the
    block's scale follows: sqrt(v) of the others stays the steady one within two spacings, 25 per cent, where
    nearest rounding would let them fall with the scale (test_host_training.py)."""
    dev = device()
    n = 1024
    p = torch.zeros(n, device=dev)
    opt = training.AdamW([p], lr=1e-3, betas=(0.9, 0.99), bits=8)
    level = (torch.rand(n, generator=gen(3)) * 0.9 + 0.1).to(dev)
    burst = torch.zeros(n, device=dev)
    burst[5::128] = 100.0
    v = torch.zeros(n, dtype=torch.float64, device=dev)
    for step in range(1, 401):
        g = (level + (burst if step == 20 else 0.0)) * (1.0 if step % 2 else -1.0)
        v = 0.99 * v + 0.01 * g.double().square()
        opt.step([g])
    ratio = (opt.moment(0)[1].double() / v).sqrt()
    announce(f"8-bit root of v over the exact one: {float(ratio.min()):.3f} to {float(ratio.max()):.3f}")
    assert float(ratio.min()) > 0.75 and float(ratio.max()) < 1.25


def test_adamw_in_8_bits_of_zeros_and_of_what_is_not_finite():
    dev = device()
    p = torch.ones(256, device=dev)
    g = torch.zeros(256, device=dev)
    g[128:] = torch.linspace(-1, 1, 128, device=dev)
    g[130], g[140] = float("inf"), float("nan")
    opt = training.AdamW([p], lr=1e-2, weight_decay=0.0, bits=8)
    opt.step([g])
    assert torch.equal(p[:128], torch.ones(128, device=dev)), "a zero gradient moves nothing"
    m, v = opt.moment(0)
    bad = torch.zeros(256, dtype=torch.bool, device=dev)
    bad[130] = bad[140] = True
    assert not m[:128].any() and not v[:128].any()
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
    assert torch.isfinite(p[~bad]).all()


def test_adamw_equals_the_formula_of_torch():
    dev = device()
    g = gen(6)
    a = [torch.randn(50, 3, generator=g).to(dev), torch.randn(7, generator=g).to(dev)]
    b = [t.clone().requires_grad_(True) for t in a]
    ours = training.AdamW(a, lr=1e-2, weight_decay=0.05)
    theirs = torch.optim.AdamW(b, lr=1e-2, weight_decay=0.05)
    for _ in range(5):
        grads = [torch.randn(t.shape, generator=g).to(dev) for t in a]
        for t, x in zip(b, grads):
            t.grad = x
        ours.step(grads)
        theirs.step()
    for x, y in zip(a, b):
        close(x, y.detach().double().cpu(), 1e-6, "five steps against torch.optim.AdamW")


def test_adamw_step_is_seen_by_bound_queries():
    """What a bound query keeps of a weight (its transpose, its packed parts) is remade after a step."""
    from boundflow_amd import crown, workloads as wl
    dev = device()
    w = wl.to_device(wl.subset(wl.make_c1(eps=0.01, label_mode="predicted"), 4), dev)
    crown.run_crown_ibp_mlp(w.module, w.spec, linear_spec_C=w.C)
    names = [k for k, t in w.module.params.items() if t.is_floating_point()]
    params = [w.module.params[k] for k in names]
    training.AdamW(params, lr=1e-2).step([torch.randn(p.shape, generator=gen(5)).to(dev) for p in params])
    got = crown.run_crown_ibp_mlp(w.module, w.spec, linear_spec_C=w.C)
    for k in names:
        w.module.params[k] = w.module.params[k].clone()
    want = crown.run_crown_ibp_mlp(w.module, w.spec, linear_spec_C=w.C)
    assert torch.equal(got.lower, want.lower) and torch.equal(got.upper, want.upper)


# ---------------------------------------------------------------------------
# streams, graphs, long offsets

def test_on_another_stream_and_in_a_graph():
    dev = device()
    g = gen(12)
    table = torch.randn(500, 96, generator=g).bfloat16().to(dev)
    tokens = torch.randint(0, 500, (4, 200), generator=g).to(dev)
    s = {k: v.to(dev) if v is not None else None
         for k, v in policy_inputs(4, 200, 500, torch.bfloat16, 13, True, "some").items()}
    q = {k: v.to(dev) for k, v in preference_inputs([200, 300, 150, 150], 500, torch.bfloat16, 14).items()}
    p = torch.randn(500, 96, generator=g).to(dev)
    moments = training.adamw_moments([p], bits=8)
    x = torch.empty(4, 200, 96, dtype=torch.bfloat16, device=dev)

    def step():
        x.copy_(training.embed_tokens(table, tokens, scale=2.0))
        a = training.policy_loss(**s, kl_weight=0.1)
        b = training.preference_loss(**q)
        c = training.embed_tokens_grad(x, tokens, 500, dtype=torch.float32)
        training.adamw_step([p], [c], moments, step=5)
        return a.stats, a.logp, a.grad_logits, b.loss, b.rewards, b.grad_logits, c, p, *moments[:4]

    def reset(kept=(p.clone(), *(t.clone() for t in moments[:4]))):
        for t, k in zip((p, *moments[:4]), kept):
            t.view(torch.uint8).copy_(k.view(torch.uint8))

    want = [t.clone() for t in step()]
    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    same = lambda a, b: all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))  # noqa: E731
    flat = lambda ts: [t.contiguous().reshape(-1) for t in ts]  # noqa: E731
    assert same(flat(got), flat(want)), "another stream, other bits"
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert same(flat(out), flat(want)), "a replay differs"
        torch.randn(1000, device=dev).sum().item()


def test_offsets_past_32_bits():
    dev = device()
    # a table and a gradient of more than 2^31 elements
    vocab, dim = 600_000, 4096
    announce("embedding of 2.4 G elements")
    table = torch.zeros(vocab, dim, dtype=torch.bfloat16, device=dev)
    table[-1] = 1.5
    table[3] = 2.0
    tokens = torch.tensor([vocab - 1, 3, vocab - 1], device=dev)
    out = training.embed_tokens(table, tokens, scale=2.0)
    assert torch.equal(out[:, 0].float().cpu(), torch.tensor([3.0, 4.0, 3.0])) and torch.equal(out[:, 0], out[:, -1])
    del table
    got = training.embed_tokens_grad(out, tokens, vocab)
    assert float(got[-1, -1]) == 6.0 and float(got[3, 0]) == 4.0 and int(torch.count_nonzero(got[4:-1])) == 0
    del got
    # logits of more than 2^31 elements: the last rows are those of a small call
    announce("losses over 2.3 G logits")
    N, V = 18_000, 128_000
    logits = torch.zeros(N, V, dtype=torch.bfloat16, device=dev)
    tail = torch.randn(3, V, generator=gen(1)).bfloat16().to(dev)
    logits[-3:] = tail
    tokens = torch.full((N,), -1, dtype=torch.int64, device=dev)
    tokens[-3:] = torch.tensor([5, V - 1, 77], device=dev)
    old = torch.full((N,), -11.0, device=dev)
    adv = torch.ones(N, device=dev)
    a = training.policy_loss(logits, tokens, old, adv)
    b = training.policy_loss(tail, tokens[-3:], old[-3:], adv[-3:])
    close(a.logp[-3:], b.logp.double().cpu(), 1e-4, "logp of the last rows")
    close(a.grad_logits[-3:], b.grad_logits.double().cpu(), 2.0 ** -7 * b.grad_logits.double().cpu().abs() + 1e-30,
          "gradient of the last rows")
    assert int(torch.count_nonzero(a.grad_logits[:-3])) == 0
    del a
    q = training.preference_loss(logits, tokens, old, torch.tensor([N - 3, N - 1, N], device=dev))
    assert float(q.grad_logits[-3].float().abs().sum()) > 0 and int(torch.count_nonzero(q.grad_logits[:-3])) == 0
    del q, logits
    announce("AdamW over 2.2 G elements")
    n = 2_200_000_000
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device=dev) for _ in range(2))
    p[-1], g[-1], g[-300] = 1.0, 0.5, -2.0
    moments = training.adamw_moments([p], bits=8)
    training.adamw_step([p], [g], moments, step=1, lr=0.25, weight_decay=0.0)
    assert float(p[-1]) == 0.75 and float(p[-300]) == 0.25 and int(torch.count_nonzero(p)) == 2


# ---------------------------------------------------------------------------
# refusals

def test_refusals():
    dev = device()
    t = torch.zeros(4, 6, device=dev)
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    with pytest.raises(HipError, match="device tensor"):
        training.embed_tokens(t.cpu(), ids)
    with pytest.raises(HipError, match="float32, bfloat16 or float16"):
        training.embed_tokens(t.double(), ids)
    with pytest.raises(HipError, match="int32 or int64"):
        training.embed_tokens(t, ids.float())
    with pytest.raises(HipError, match="contiguous rows"):
        training.embed_tokens(t.t(), ids)
    with pytest.raises(ValueError, match="tokens of shape"):
        training.embed_tokens_grad(t, ids, 9)
    with pytest.raises(ValueError, match="dtype must be"):
        training.embed_tokens_grad(t[:3], ids, 9, dtype=torch.float16)
    with pytest.raises(ValueError, match="accumulate_into of shape"):
        training.embed_tokens_grad(t[:3], ids, 9, accumulate_into=t)
    with pytest.raises(HipError, match="accumulate_into must be float32"):
        training.embed_tokens_grad(t[:3], ids, 4, accumulate_into=t.half())
    s = {k: v.to(dev) if v is not None else None
         for k, v in policy_inputs(2, 3, 5, torch.float32, 1, True, "some").items()}
    for change, error, match in (
            (dict(logits=s["logits"].transpose(1, 2).contiguous().transpose(1, 2)), HipError, "contiguous last axis"),
            (dict(tokens=s["tokens"][:, :1]), ValueError, "tokens of shape"),
            (dict(logits=s["logits"][0, 0]), ValueError, "must be"),
            (dict(mask=s["mask"].float()), HipError, "mask must be bool"),
            (dict(mask=s["mask"][:1]), ValueError, "mask of shape"),
            (dict(advantages=s["advantages"][:, :1]), ValueError, "advantages of shape"),
            (dict(old_logp=s["old_logp"].half()), HipError, "old_logp must be float32"),
            (dict(temperature=0.0), ValueError, "temperature"),
            (dict(clip_low=-0.1), ValueError, "clip limits"),
            (dict(reduction="sum"), ValueError, "unknown reduction")):
        with pytest.raises(error, match=match):
            training.policy_loss(**{**s, **change})
    q = {k: v.to(dev) for k, v in preference_inputs([2, 3], 5, torch.float32, 1).items()}
    for change, error, match in ((dict(offsets=q["offsets"][:2]), ValueError, "offsets must be"),
                                 (dict(offsets=q["offsets"].int()), HipError, "offsets must be int64"),
                                 (dict(label_smoothing=1.5), ValueError, "label_smoothing"),
                                 (dict(ref_logp=q["ref_logp"][:2]), ValueError, "ref_logp of shape")):
        with pytest.raises(error, match=match):
            training.preference_loss(**{**q, **change})
    p = [torch.zeros(5, device=dev), torch.zeros(6, device=dev)]
    g = [torch.zeros_like(x) for x in p]
    moments = training.adamw_moments(p)
    for args, kw, error, match in (
            ((p, g[:1], moments), dict(step=1), ValueError, "2 parameters, 1 gradients"),
            ((p, g, moments), dict(step=0), ValueError, "step counts from 1"),
            ((p, [g[0], g[1][:5]], moments), dict(step=1), ValueError, "of shape"),
            ((p, [g[0], g[1].half()], moments), dict(step=1), HipError, "as the first are"),
            ((p[:1], g[:1], moments), dict(step=1), ValueError, "flat of"),
            ((p, g, moments._replace(v_scale=moments.m)), dict(step=1), HipError, "must be torch.float8_e4m3fn"),
            ((p, g, moments), dict(step=1, betas=(1.0, 0.9)), ValueError, "betas"),
            ((p, g, moments), dict(step=1, grad_scale=torch.zeros(2, device=dev)), HipError, "scalar")):
        with pytest.raises(error, match=match):
            training.adamw_step(*args, **kw)
    with pytest.raises(ValueError, match="32 or 8"):
        training.adamw_moments(p, bits=16)
    with pytest.raises(ValueError, match="no gradient"):
        training.AdamW(p).step()
