"""The training operators whose time is measured: what stands at both ends of a token network's
training step and updates its weights, for networks that are then handed to the bound queries.

A case is a dict of plain values.  ``op`` names what is called:

* ``embed``       ``embed_tokens``: rows of a table by token, scaled
* ``embed_grad``  ``embed_tokens_grad``: the table's gradient, every token's rows summed in fp32,
                  written whole or added to a running fp32 gradient
* ``policy``      ``policy_loss``: the clipped policy objective with a KL term against a reference,
                  and its gradient with respect to the logits
* ``preference``  ``preference_loss``: the paired log-ratio loss of chosen and rejected responses,
                  and its gradient with respect to the logits
* ``adamw``       ``adamw_step``: one AdamW step over many tensors, moments in 32 or in 8 bits

``run`` computes an operator in its plain form, elementary tensor operations in fp32 rounded once
at the end, or, where ``own`` is set, calls the package.
"""

from __future__ import annotations

import math
import random
from typing import List

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}

BLOCK = 128                  # elements of an 8-bit moment that share a scale; tensors start at multiples of it
LARGEST = 448.0              # the largest value of float8_e4m3fn
LEAST_TOP = 2.0 ** -100      # a block whose largest moment is below this is held as zeros
PHASE_STEP, PHASE_ELEMENT = 0x9E3779B9, 0x6A09E667   # golden ratio and sqrt(2), fractions of 2^32

CLIP_LOW, CLIP_HIGH = 0.2, 0.28
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1


def listed() -> List[dict]:
    return [
        # the next token of eight requests: a few rows, latency alone
        {"name": "embed_next", "op": "embed", "tokens": 8, "vocab": 32000, "dim": 2048, "dtype": "bfloat16",
         "scale": 45.25},
        # a training batch's whole input
        {"name": "embed_batch", "op": "embed", "tokens": 16384, "vocab": 64000, "dim": 4096, "dtype": "bfloat16",
         "scale": 64.0},
        # the table of a small token policy: odd sizes, fp32
        {"name": "embed_grad_policy", "op": "embed_grad", "tokens": 600, "vocab": 1003, "dim": 129,
         "dtype": "float32", "accumulate": False, "scale": 1.0},
        # a training batch: the dense gradient of a large table
        {"name": "embed_grad_batch", "op": "embed_grad", "tokens": 16384, "vocab": 32000, "dim": 4096,
         "dtype": "bfloat16", "accumulate": False, "scale": 64.0},
        # a minibatch of a controller with five actions: many rows of a very short axis
        {"name": "policy_actions", "op": "policy", "sequences": 64, "length": 16, "vocab": 5, "dtype": "float32",
         "kl": True, "reduction": "token", "temperature": 1.0},
        # a minibatch of sampled responses, padded to a common length
        {"name": "policy_responses", "op": "policy", "sequences": 8, "length": 511, "vocab": 32000,
         "dtype": "bfloat16", "kl": True, "reduction": "token", "temperature": 0.8},
        # the largest: long responses over a large vocabulary
        {"name": "policy_long", "op": "policy", "sequences": 8, "length": 1023, "vocab": 128000,
         "dtype": "bfloat16", "kl": True, "reduction": "sequence", "temperature": 1.0},
        # two short pairs, so few rows that each has to be split to fill the device
        {"name": "preference_few", "op": "preference", "pairs": 2, "rows": 45, "vocab": 50001, "dtype": "float32",
         "smoothing": 0.0},
        # an ordinary batch of pairs of very different lengths, rows of an odd length
        {"name": "preference_batch", "op": "preference", "pairs": 16, "rows": 9001, "vocab": 50001,
         "dtype": "bfloat16", "smoothing": 0.1},
        # the weights of an image-sized MLP (784-256-256-10): six tensors
        {"name": "adamw_mlp", "op": "adamw", "tensors": 6, "elements": 269322, "dtype": "float32", "bits": 32,
         "master": False},
        # bf16 weights with fp32 master copies and fp32 moments
        {"name": "adamw_master", "op": "adamw", "tensors": 150, "elements": 150_000_000, "dtype": "bfloat16",
         "bits": 32, "master": True},
        # bf16 weights, moments in 8 bits
        {"name": "adamw_eight", "op": "adamw", "tensors": 200, "elements": 300_000_000, "dtype": "bfloat16",
         "bits": 8, "master": False},
    ]


def _size(rng, lo: int, hi: int) -> int:
    """A size spread over the logarithm of its range; half of them a multiple of 8, as widths often are."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 8:
        n = n // 8 * 8
    return max(lo, min(hi, n))


def draw(rng) -> dict:
    op = rng.choice(["embed", "embed_grad", "policy", "preference", "adamw"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    if op == "embed":
        return {"op": op, "tokens": _size(rng, 1, 16384), "vocab": _size(rng, 300, 128000),
                "dim": _size(rng, 16, 4096), "dtype": dtype, "scale": round(rng.uniform(0.5, 64.0), 2)}
    if op == "embed_grad":
        return {"op": op, "tokens": _size(rng, 1, 16384), "vocab": _size(rng, 300, 64000),
                "dim": _size(rng, 16, 4096), "dtype": dtype, "accumulate": rng.random() < 0.4,
                "scale": round(rng.uniform(0.5, 64.0), 2)}
    if op in ("policy", "preference"):
        rows = _size(rng, 2, 8184)
        vocab = _size(rng, 4, min(128000, max(4, 500_000_000 // rows)))
        if op == "preference":
            pairs = _size(rng, max(1, rows // 600), max(1, min(64, rows // 2)))
            return {"op": op, "pairs": pairs, "rows": rows, "vocab": vocab, "dtype": dtype,
                    "smoothing": rng.choice([0.0, 0.1])}
        sequences = _size(rng, 1, max(1, min(64, rows)))
        return {"op": op, "sequences": sequences, "length": max(1, rows // sequences), "vocab": vocab,
                "dtype": dtype, "kl": rng.random() < 0.7, "reduction": rng.choice(["token", "sequence"]),
                "temperature": rng.choice([1.0, 1.0, 0.7, 1.3])}
    tensors = _size(rng, 1, 300)
    return {"op": op, "tensors": tensors, "elements": max(tensors, _size(rng, 1000, 150_000_000)), "dtype": dtype,
            "bits": rng.choice([32, 8]), "master": dtype != "float32" and rng.random() < 0.5}


# ---------------------------------------------------------------------------
# sizes that follow from a case alone

def _lengths(case) -> np.ndarray:
    """Response lengths of a padded batch: between 60 and 100 per cent of the padded length."""
    r = random.Random(f"lengths {case['sequences']} {case['length']}")
    return np.array([max(1, round(case["length"] * r.uniform(0.6, 1.0))) for _ in range(case["sequences"])])


def _sizes(case) -> List[int]:
    """Elements of every weight: sizes spread over their logarithm, as a network's matrices and vectors are."""
    if (case["tensors"], case["elements"]) == (6, 784 * 256 + 256 + 256 * 256 + 256 + 256 * 10 + 10):
        return [784 * 256, 256, 256 * 256, 256, 256 * 10, 10]
    r = random.Random(f"sizes {case['tensors']} {case['elements']}")
    parts = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    room, total = case["elements"] - case["tensors"], sum(parts)
    sizes = [1 + int(room * p / total) for p in parts]
    sizes[-1] += case["elements"] - sum(sizes)
    return sizes


def _starts(sizes) -> List[int]:
    """First element of every tensor in the flat buffers, and their length."""
    return [0] + np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes]).tolist()


def _token_shares(vocab: int) -> np.ndarray:
    edges = (np.arange(vocab + 1) / vocab) ** (1.0 / 3.0)
    return np.diff(edges)


def _distinct(tokens: int, vocab: int) -> float:
    """Expected number of different tokens of ``_tokens``."""
    return float(np.sum(-np.expm1(tokens * np.log1p(-_token_shares(vocab)))))


def work(case) -> dict:
    op, size = case["op"], SIZES[case["dtype"]]
    if op == "embed":
        n, d = case["tokens"], case["dim"]
        return {"bytes": 8 * n + size * d * (n + _distinct(n, case["vocab"])), "flops": n * d}
    if op == "embed_grad":
        n, d = case["tokens"], case["dim"]
        # added to: the rows that occur are read and written; made: every row is written
        out = 8 * _distinct(n, case["vocab"]) if case["accumulate"] else size * case["vocab"]
        return {"bytes": 8 * n + d * (size * n + out), "flops": 2 * n * d}
    if op == "policy":
        n, v = case["sequences"] * case["length"], case["vocab"]
        live = int(_lengths(case).sum())
        return {"bytes": size * v * (live + n) + n * (8 + 1 + 4 + 4 + 4 * case["kl"]) + 4 * case["sequences"],
                "flops": 8 * live * v}
    if op == "preference":
        n, v = case["rows"], case["vocab"]
        return {"bytes": 2 * size * v * n + n * (8 + 4 + 4), "flops": 8 * n * v}
    n = case["elements"]
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (2 * size + (4 + 4 + moments - size if case["master"] else moments) + size),
            "flops": 15 * n}


# ---------------------------------------------------------------------------
# inputs

def _tokens(n: int, vocab: int, gen) -> torch.Tensor:
    """Tokens in order of falling frequency, as a vocabulary is: the share of the first v is (v / vocab)^(1/3)."""
    u = torch.rand(n, device="cuda", generator=gen)
    return (u * u * u * vocab).long().clamp_(max=vocab - 1)


def _logits(rows: int, vocab: int, dtype, gen):
    """Logits of a partly trained network and the tokens that it sampled, their log-probabilities in fp32."""
    logits = torch.empty(rows, vocab, device="cuda", dtype=dtype).normal_(0.0, 2.0, generator=gen)
    tokens = _tokens(rows, vocab, gen)
    lift = torch.rand(rows, 1, device="cuda", generator=gen) * (math.log(vocab) + 4.0)
    at = tokens.unsqueeze(1)
    logits.scatter_(1, at, (logits.gather(1, at).float() + lift).to(dtype))
    return logits, tokens


def _chosen_logp(logits: torch.Tensor, tokens: torch.Tensor, inv_t: float) -> torch.Tensor:
    z = logits.float() * inv_t
    return z.gather(1, tokens[:, None])[:, 0] - torch.logsumexp(z, 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if case["op"] == "embed":
        s["table"] = (normal(case["vocab"], case["dim"]) * 0.02).to(dtype)
        s["ids"] = _tokens(case["tokens"], case["vocab"], gen)
    elif case["op"] == "embed_grad":
        s["ids"] = _tokens(case["tokens"], case["vocab"], gen)
        s["grad"] = (normal(case["tokens"], case["dim"]) * 1e-2).to(dtype)
        s["running"] = normal(case["vocab"], case["dim"]) * 1e-2 if case["accumulate"] else None
    elif case["op"] == "policy":
        B, T, V = case["sequences"], case["length"], case["vocab"]
        # the network answers for T + 1 positions; the last predicts nothing that was sampled
        logits, tokens = _logits(B * (T + 1), V, dtype, gen)
        logp = _chosen_logp(logits, tokens, 1.0 / case["temperature"]).view(B, T + 1)[:, :T]
        s["logits"] = logits.view(B, T + 1, V)[:, :T]
        s["ids"] = tokens.view(B, T + 1)[:, :T].contiguous()
        # ratios of an update's later passes; none so near a clip limit that rounding decides its side
        drift = normal(B, T) * 0.15
        for limit in (math.log(1.0 - CLIP_LOW), math.log(1.0 + CLIP_HIGH)):
            drift = torch.where((drift - limit).abs() < 2e-3, torch.full_like(drift, limit + 5e-3), drift)
        s["old_logp"] = (logp - drift).contiguous()
        s["ref_logp"] = (logp + normal(B, T) * 0.3).contiguous() if case["kl"] else None
        s["advantages"] = normal(B, 1).expand(B, T)     # one for a whole response
        lengths = torch.from_numpy(_lengths(case)).cuda()
        s["mask"] = torch.arange(T, device="cuda")[None, :] < lengths[:, None]
    elif case["op"] == "preference":
        n, pairs = case["rows"], case["pairs"]
        s["logits"], s["ids"] = _logits(n, case["vocab"], dtype, gen)
        cuts = torch.sort(torch.randint(0, n + 1, (2 * pairs - 1,), device="cuda", generator=gen))[0]
        s["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)])
        # every response has become more or less likely than it was to the reference, by 10 to 30 nats in all
        moved = torch.rand(2 * pairs, device="cuda", generator=gen) * 40.0 - 20.0
        moved = moved + 10.0 * torch.where(moved < 0, -1.0, 1.0)
        lengths = torch.diff(s["offsets"])
        moved = torch.repeat_interleave(moved / lengths.clamp(min=1), lengths)
        s["ref_logp"] = _chosen_logp(s["logits"], s["ids"], 1.0) - moved + normal(n) * 0.1
    else:
        sizes = _sizes(case)
        starts = _starts(sizes)
        total = starts[-1]
        where = list(zip(starts, sizes))
        live = torch.zeros(total, device="cuda", dtype=torch.bool)
        for at, k in where:
            live[at:at + k] = True
        flat = lambda scale: torch.where(live, normal(total) * scale, 0.0)  # noqa: E731
        weight = flat(0.05)
        s["flat"], s["flat_grad"] = weight.to(dtype), flat(1e-3).to(dtype)
        s["params"] = [s["flat"][at:at + k] for at, k in where]
        s["grads"] = [s["flat_grad"][at:at + k] for at, k in where]
        s["master_copy"] = s["flat"].float() if case["master"] else None
        m, root = flat(3e-4), flat(1e-3).abs() + 1e-4 * live
        s["m_scale"] = s["v_scale"] = None
        if case["bits"] == 32:
            s["m"], s["v"] = m, root * root
        else:
            for name, x in (("m", m), ("v", root)):
                x = x.view(-1, BLOCK)
                top = x.abs().amax(1, keepdim=True)
                held = (x * torch.where(top > 0, LARGEST / top, top)).clamp_(-LARGEST, LARGEST)
                s[name] = held.to(torch.float8_e4m3fn).view(-1)
                s[name + "_scale"] = (top / LARGEST).view(-1)
        s["step"] = 100
        s["clip"] = torch.full((), 0.75, device="cuda")     # the factor of a clipped gradient norm
    return s


# ---------------------------------------------------------------------------
# one pass

def run(s):
    if own:
        return _call(s)
    return {"embed": _embed, "embed_grad": _embed_grad, "policy": _policy, "preference": _preference,
            "adamw": _adamw}[s["op"]](s)


def _call(s):
    from boundflow_amd import training

    op = s["op"]
    if op == "embed":
        return training.embed_tokens(s["table"], s["ids"], scale=s["scale"])
    if op == "embed_grad":
        return training.embed_tokens_grad(s["grad"], s["ids"], s["vocab"], scale=s["scale"],
                                          accumulate_into=s["running"])
    if op == "policy":
        r = training.policy_loss(s["logits"], s["ids"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                                 mask=s["mask"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_weight=0.05,
                                 temperature=s["temperature"], reduction=s["reduction"])
        return {"stats": r.stats, "logp": r.logp, "grad": r.grad_logits}
    if op == "preference":
        r = training.preference_loss(s["logits"], s["ids"], s["ref_logp"], s["offsets"], beta=0.1,
                                     label_smoothing=s["smoothing"])
        return {"loss": r.loss, "rewards": r.rewards, "logp": r.logp, "grad": r.grad_logits}
    s["step"] += 1
    moments = training.AdamWMoments(s["m"], s["v"], s["m_scale"], s["v_scale"], s["master_copy"])
    training.adamw_step(s["params"], s["grads"], moments, step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                        weight_decay=DECAY, grad_scale=s["clip"])
    return _updated(s)


def _updated(s):
    return {"params": s["flat"], "master": s["master_copy"], "m": s["m"], "v": s["v"], "m_scale": s["m_scale"],
            "v_scale": s["v_scale"]}


def _embed(s):
    return (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)


def _embed_grad(s):
    scaled = s["grad"].float() * s["scale"]
    if s["running"] is not None:
        return s["running"].index_add_(0, s["ids"], scaled)
    out = torch.zeros(s["vocab"], s["dim"], device=scaled.device)
    return out.index_add_(0, s["ids"], scaled).to(s["grad"].dtype)


def _token_logp(logits, ids, inv_t: float):
    """(log-probabilities of the tokens, softmax) over the last axis."""
    z = logits.float() * inv_t
    z -= z.amax(-1, keepdim=True)
    chosen = z.gather(-1, ids.unsqueeze(-1)).squeeze(-1)
    p = z.exp_()
    total = p.sum(-1, keepdim=True)
    return chosen - total.squeeze(-1).log(), p.div_(total)


def _logit_grad(p, ids, g, dtype):
    """g (onehot - softmax), in place of the softmax."""
    p.mul_(-g.unsqueeze(-1))
    p.scatter_add_(-1, ids.unsqueeze(-1), g.unsqueeze(-1))
    return p.to(dtype)


def _policy(s):
    inv_t, mask = 1.0 / s["temperature"], s["mask"]
    logp, p = _token_logp(s["logits"], s["ids"], inv_t)
    live = mask.float()
    if s["reduction"] == "token":
        weight = live / live.sum()
    else:
        counts = live.sum(1, keepdim=True)
        weight = live / counts.clamp_min(1.0) / (counts > 0).sum()
    a = s["advantages"]
    ratio = (logp - s["old_logp"]).exp()
    plain, clipped = ratio * a, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * a
    outside = clipped < plain
    policy = -torch.minimum(plain, clipped)
    g = torch.where(outside, 0.0, -plain)
    kl = torch.zeros_like(logp)
    if s["ref_logp"] is not None:
        apart = s["ref_logp"] - logp
        kl = apart.exp() - apart - 1.0
        g = g + 0.05 * (1.0 - apart.exp())
    stats = torch.stack([(weight * x).sum() for x in (policy + 0.05 * kl, policy, kl, outside)])
    grad = _logit_grad(p, s["ids"], weight * g * inv_t, s["logits"].dtype)
    return {"stats": stats, "logp": torch.where(mask, logp, 0.0), "grad": grad}


def _preference(s):
    logp, p = _token_logp(s["logits"], s["ids"], 1.0)
    pairs = s["pairs"]
    rows = torch.arange(s["rows"], device=logp.device)
    owner = (rows[:, None] >= s["offsets"][None, 1:-1]).sum(1)      # the response that a row belongs to
    of = owner[None, :] == torch.arange(2 * pairs, device=logp.device)[:, None]
    rewards = 0.1 * torch.where(of, logp - s["ref_logp"], 0.0).sum(1)
    h = rewards[:pairs] - rewards[pairs:]
    ls = s["smoothing"]
    # log sigma(x) = min(x, 0) - log(1 + exp(-|x|))
    tail = (1.0 + (-h.abs()).exp()).log()
    loss = -((1.0 - ls) * (h.clamp(max=0.0) - tail) + ls * ((-h).clamp(max=0.0) - tail)).mean()
    dh = -((1.0 - ls) / (1.0 + h.exp()) - ls / (1.0 + (-h).exp())) * 0.1 / pairs
    g = torch.cat([dh, -dh])[owner]
    return {"loss": loss, "rewards": rewards, "logp": logp, "grad": _logit_grad(p, s["ids"], g, s["logits"].dtype)}


def _taken(held, scale):
    return (held.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _held(x, phase, positive: bool):
    """fp32 moments as float8_e4m3fn and the scale of each block: the magnitude over its spacing, cut to
    20 bits below it, plus the element's 20-bit phase, and then down to a whole number of spacings."""
    x = x.view(-1, BLOCK)
    size = x.abs()
    top = size.amax(1, keepdim=True)
    used = top >= LEAST_TOP
    scale, inverse = torch.where(used, top / LARGEST, 0.0), torch.where(used, LARGEST / top, 0.0)
    y = (size * inverse).clamp_(max=LARGEST)
    exponent = ((y.view(torch.int32) >> 23) - 127).clamp_(min=-6)
    spacing = ((exponent - 3 + 127) << 23).view(torch.float32)
    count = ((y / spacing * 2.0 ** 20).int() + phase.view(-1, BLOCK)) >> 20
    if positive:
        count = torch.where((y > 0) & (count < 1), 1, count)
    value = count * spacing
    if not positive:
        value = torch.where(x < 0, -value, value)
    return value.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _adamw(s):
    s["step"] += 1
    t = s["step"]
    g = s["flat_grad"].float() * s["clip"]
    eight = s["m_scale"] is not None
    m = _taken(s["m"], s["m_scale"]) if eight else s["m"]
    if eight:
        root = _taken(s["v"], s["v_scale"])
        v = root * root
    else:
        v = s["v"]
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + g * g * (1.0 - BETA2)
    root = v.sqrt()
    w = s["flat"].float() if s["master_copy"] is None else s["master_copy"]
    rate = LR / (1.0 - BETA1 ** t)
    w = w * (1.0 - LR * DECAY) - m / (root / math.sqrt(1.0 - BETA2 ** t) + EPS) * rate
    s["flat"].copy_(w)
    if s["master_copy"] is not None:
        s["master_copy"].copy_(w)
    if eight:
        at = torch.arange(m.numel(), device=m.device)
        phase = (((at * PHASE_ELEMENT + t * PHASE_STEP) & 0xFFFFFFFF) >> 12).int()
        for name, x, positive in (("m", m, False), ("v", root, True)):
            held, scale = _held(x, phase, positive)
            s[name].copy_(held)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _updated(s)


# ---------------------------------------------------------------------------
# the same results in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        return torch.nn.functional.embedding(s["ids"], s["table"].double()) * case["scale"]
    if op == "embed_grad":
        table = torch.zeros(case["vocab"], case["dim"], device="cuda", dtype=torch.float64)
        table.index_put_((s["ids"],), s["grad"].double() * case["scale"], accumulate=True)
        return table if s["running"] is None else table + s["running"].double()
    if op == "policy":
        z = s["logits"].double().requires_grad_(True)
        logp = torch.log_softmax(z / case["temperature"], -1).gather(-1, s["ids"][..., None])[..., 0]
        counts = s["mask"].sum(1)
        if case["reduction"] == "token":
            mean = lambda x: x[s["mask"]].mean()  # noqa: E731
        else:
            mean = lambda x: torch.stack([row[:k].mean() for row, k in zip(x, counts.tolist()) if k]).mean()  # noqa: E731
        a = s["advantages"].double()
        ratio = torch.exp(logp - s["old_logp"].double())
        kept = torch.minimum(ratio * a, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * a)
        share = (kept < ratio * a).double()
        kl = torch.zeros_like(logp)
        if s["ref_logp"] is not None:
            apart = s["ref_logp"].double() - logp
            kl = torch.expm1(apart) - apart
        terms = torch.stack([mean(-kept), mean(kl), mean(share)])
        loss = terms[0] + 0.05 * terms[1]
        loss.backward()
        return {"stats": torch.cat([loss[None], terms]), "logp": logp * s["mask"], "grad": z.grad}
    if op == "preference":
        z = s["logits"].double().requires_grad_(True)
        logp = torch.log_softmax(z, -1).gather(-1, s["ids"][:, None])[:, 0]
        bounds = s["offsets"].tolist()
        sums = torch.stack([(logp - s["ref_logp"].double())[a:b].sum() for a, b in zip(bounds, bounds[1:])])
        chosen, rejected = (0.1 * sums).view(2, -1)
        good = torch.nn.functional.logsigmoid(chosen - rejected)
        bad = torch.nn.functional.logsigmoid(rejected - chosen)
        loss = -((1.0 - case["smoothing"]) * good + case["smoothing"] * bad).mean()
        loss.backward()
        return {"loss": loss, "rewards": torch.cat([chosen, rejected]), "logp": logp, "grad": z.grad}
    return _exact_adamw(s)


def _exact_adamw(s):
    t = s["step"] + 1
    g = s["flat_grad"].double() * 0.75
    if s["m_scale"] is None:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (s["v"].double() * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = torch.lerp(m, g, 1.0 - BETA1)
    v = torch.lerp(v, g.square(), 1.0 - BETA2)
    w = (s["flat"] if s["master_copy"] is None else s["master_copy"]).double()
    w = w - LR * DECAY * w - LR * (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)).sqrt() + EPS)
    out = {"params": w, "master": None if s["master_copy"] is None else w, "m": m, "v": v, "m_scale": None,
           "v_scale": None}
    if s["m_scale"] is None:
        return out
    at = torch.arange(m.numel(), device="cuda")
    # the phase of an element, as a share of a spacing
    phase = (((at * PHASE_ELEMENT + t * PHASE_STEP) % 2 ** 32) // 2 ** 12).double() / 2 ** 20
    for name, x in (("m", m), ("v", v.sqrt())):
        blocks = x.view(-1, BLOCK)
        scale = blocks.abs().amax(1) / LARGEST
        y = blocks / torch.where(scale > 0, scale, 1.0)[:, None]
        spacing = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        whole = torch.floor(y.abs() / spacing + phase.view(-1, BLOCK))
        if name == "v":
            whole = torch.where(y > 0, whole.clamp(min=1.0), whole)
        out[name] = (torch.sign(y) * whole * spacing).clamp(-LARGEST, LARGEST).view(-1)
        out[name + "_scale"] = scale
    return out
