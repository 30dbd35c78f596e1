"""Plain restatement, in float64 on the CPU, of the training operators: the formulas as they are
written, with autograd for the losses' gradients.  The reference has no counterpart."""

from __future__ import annotations

import torch

BLOCK = 128


def embed_tokens(table, tokens, scale):
    t = tokens.reshape(-1)
    out = torch.zeros(t.numel(), table.shape[1], dtype=torch.float64)
    for i, v in enumerate(t.tolist()):
        if v >= table.shape[0]:
            out[i] = float("nan")
        elif v >= 0:
            out[i] = table[v].double() * scale
    return out.view(*tokens.shape, table.shape[1])


def embed_tokens_grad(grad, tokens, vocab, scale):
    """(the gradient, the sum of the magnitudes that make it, how many)."""
    g = grad.double().reshape(-1, grad.shape[-1]) * scale
    out, size = (torch.zeros(vocab, grad.shape[-1], dtype=torch.float64) for _ in range(2))
    count = torch.zeros(vocab, 1, dtype=torch.float64)
    for i, v in enumerate(tokens.reshape(-1).tolist()):
        if 0 <= v < vocab:
            out[v] += g[i]
            size[v] += g[i].abs()
            count[v] += 1
    return out, size, count


def policy_loss(logits, tokens, old_logp, advantages, *, ref_logp=None, mask=None, clip_low=0.2, clip_high=0.2,
                kl_weight=0.0, temperature=1.0, reduction="token", grad_scale=1.0):
    """dict of stats, logp, grad, and what a tolerance needs: p (softmax), g (the loss's derivative by a
    row's log-probability) and slope (how much |g| moves with it)."""
    lead = tokens.shape
    live = tokens >= 0
    if mask is not None:
        live = live & mask
    z = logits.detach().double().requires_grad_(True)
    # rows that take no part may hold anything
    x = torch.where(live[..., None], z, torch.zeros((), dtype=torch.float64)) / temperature
    logsm = torch.log_softmax(x, -1)
    logp = logsm.gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    A = advantages.double()
    A = A if A.shape == lead else A.view(-1, *[1] * (len(lead) - 1)).expand(lead)
    ratio = torch.exp(logp - old_logp.double())
    kept = torch.minimum(ratio * A, ratio.clamp(1 - clip_low, 1 + clip_high) * A)
    outside = (kept < ratio * A).double()
    kl = torch.zeros_like(logp)
    slope = ratio * A.abs()
    if ref_logp is not None:
        d = ref_logp.double() - logp
        kl = torch.exp(d) - d - 1
        slope = slope + kl_weight * torch.exp(d)
    rows = live.double() if len(lead) == 2 else live.double()[:, None]
    counts = rows.sum(1)
    if reduction == "token":
        weight = rows / counts.sum().clamp(min=1)
    else:
        weight = rows / counts.clamp(min=1)[:, None] / (counts > 0).sum().clamp(min=1)
    weight = weight.reshape(lead)
    zero = torch.zeros((), dtype=torch.float64)
    total = lambda v: torch.where(live, weight * v, zero).sum()  # noqa: E731
    terms = [total(-kept), total(kl), total(outside)]
    loss = terms[0] + kl_weight * terms[1]
    grad = torch.autograd.grad(loss, z)[0] * grad_scale if loss.requires_grad else torch.zeros_like(z)
    g = torch.where(live, weight * (torch.where(outside > 0, zero, -ratio * A)
                                    + (kl_weight * (1 - torch.exp(d)) if ref_logp is not None else 0.0)), zero)
    return {"stats": torch.stack([loss, *terms]).detach(), "logp": torch.where(live, logp, zero).detach(),
            "grad": grad.detach(), "p": logsm.exp().detach(), "g": g.detach(), "slope": (weight * slope).detach(),
            "live": live}


def preference_loss(logits, tokens, ref_logp, offsets, *, beta=0.1, label_smoothing=0.0, grad_scale=1.0):
    z = logits.detach().double().requires_grad_(True)
    logsm = torch.log_softmax(z, -1)
    taken = tokens >= 0
    logp = logsm.gather(-1, tokens.clamp(min=0)[:, None])[:, 0]
    diff = torch.where(taken, logp - ref_logp.double(), torch.zeros((), dtype=torch.float64))
    bounds = offsets.tolist()
    pairs = len(bounds) // 2
    sums = [diff[a:b].sum() for a, b in zip(bounds, bounds[1:])]
    rewards = beta * torch.stack(sums) if sums else torch.zeros(0, dtype=torch.float64)
    h = rewards[:pairs] - rewards[pairs:]
    logsig = torch.nn.functional.logsigmoid
    losses = -(1 - label_smoothing) * logsig(h) - label_smoothing * logsig(-h)
    loss = losses.mean() if pairs else torch.zeros((), dtype=torch.float64)
    grad = torch.zeros_like(z)
    if pairs and loss.requires_grad:
        grad = torch.autograd.grad(loss, z)[0] * grad_scale
    inside = torch.zeros(len(tokens), dtype=torch.bool)
    inside[bounds[0]:bounds[-1]] = True
    live = taken & inside
    zero = torch.zeros((), dtype=torch.float64)
    return {"loss": loss.detach(), "rewards": rewards.detach(), "logp": torch.where(live, logp, zero).detach(),
            "grad": grad.detach(), "p": logsm.exp().detach(), "live": live}


def adamw(w, g, m, v, *, step, lr, betas, eps, weight_decay):
    """(w, m, v) after one step, float64."""
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    w = w - lr * weight_decay * w - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return w, m, v


def phases(count, step):
    """The share of a spacing that element i's magnitude is moved up by at a step, in 2^-20."""
    return torch.tensor([((i * 0x6A09E667 + step * 0x9E3779B9) % 2 ** 32) >> 12 for i in range(count)],
                        dtype=torch.float64) / 2 ** 20


def hold(x, phase, root):
    """x (whole blocks) in 8 bits: (spacings counted with the phase, before the cut; spacing; scale per block)."""
    blocks = x.double().view(-1, BLOCK)
    top = blocks.abs().amax(1)
    scale = torch.where(top >= 2.0 ** -100, top / 448, torch.zeros((), dtype=torch.float64))
    y = torch.where(scale[:, None] > 0, blocks.abs() / scale.clamp(min=1e-300)[:, None],
                    torch.zeros((), dtype=torch.float64))
    spacing = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    count = y / spacing + phase.view(-1, BLOCK)
    if root:
        count = torch.where((y > 0) & (count < 1), torch.ones((), dtype=torch.float64), count)
    return count.view(-1), spacing.view(-1), scale


def vocabulary_loss(hidden, weight, tokens, *, bias=None, mask=None, temperature=1.0, grad_scale=1.0):
    """dict of loss, logp and the gradients, and what a tolerance needs, all of the live rows (``at``, their places):
    x, p (softmax), g (the loss's derivative by a row's logits over the temperature) and the magnitudes of the products
    that make a logit."""
    lead, D = tokens.shape, hidden.shape[-1]
    live = tokens >= 0
    if mask is not None:
        live = live & mask
    at = live.reshape(-1).nonzero()[:, 0]
    x, w, y = hidden.reshape(-1, D)[at].double(), weight.double(), tokens.reshape(-1)[at]
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.double()
    z = torch.mm(x, w.t()) + b
    size = torch.mm(x.abs(), w.abs().t()) + torch.where(torch.isfinite(b) & (b.abs() < 1e30), b.abs(), 0.0)
    logsm = torch.log_softmax(z / temperature, 1)
    rows = torch.arange(at.numel())
    n = max(at.numel(), 1)
    logp = torch.zeros(live.numel(), dtype=torch.float64)
    logp[at] = logsm[rows, y]
    p = logsm.exp()
    g = p.clone()
    g[rows, y] -= 1.0
    factor = grad_scale / (temperature * n)
    dx = torch.zeros(live.numel(), D, dtype=torch.float64)
    dx[at] = torch.mm(g, w) * factor
    return {"loss": -logp.sum() / n, "logp": logp.view(lead), "hidden": dx.view(hidden.shape),
            "weight": torch.mm(g.t(), x) * factor, "bias": g.sum(0) * factor, "at": at, "x": x, "w": w, "p": p, "g": g,
            "z": z, "size": size, "factor": factor}


def philox(block, counter, seed):
    """The eight 16-bit numbers of a block: Philox 4x32 of ten rounds in Python's integers."""
    low = 0xFFFFFFFF
    c = [block & low, block >> 32, counter & low, counter >> 32]
    k = [seed & low, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return [w >> s & 0xFFFF for w in c for s in (0, 16)]


def dropout(x, p, seed, counter=0, residual=None, first=0):
    """(result, kept), elements counted from ``first`` on (a multiple of 8)."""
    border = int(p * 65536 + 0.5)
    drawn = [u for k in range(-(-x.numel() // 8)) for u in philox(first // 8 + k, counter, seed)][:x.numel()]
    kept = torch.tensor(drawn, dtype=torch.int64).view(x.shape) >= border
    y = torch.where(kept, x.double() / (1.0 - border / 65536.0 if border < 65536 else 1.0), 0.0)
    return (y if residual is None else y + residual.double()), kept
