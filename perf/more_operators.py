"""More training operators whose time is measured: a supervised step of a token network, for
networks that are then handed to the bound queries.

A case is a dict of plain values.  ``op`` names what is called:

* ``loss``          ``vocabulary_loss``: softmax cross entropy of a linear head over a vocabulary, with the
                    gradients of the hidden rows, the head's weight and its bias
* ``score``         the same without gradients: the tokens' log-probabilities (what the policy and the
                    preference losses take as those of an old or a reference policy)
* ``dropout``       ``dropout``: the mask from a counter-based generator, never stored, optionally added to
                    a residual
* ``dropout_grad``  ``dropout_grad``: the same mask on a gradient

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

LARGEST = 8 * 1023 * 4096 * 128000     # rows x width x vocabulary of the largest case


def listed() -> List[dict]:
    return [
        # the head of a small token policy with eight actions: latency alone
        {"name": "loss_actions", "op": "loss", "sequences": 512, "length": 1, "dim": 160, "vocab": 8,
         "dtype": "float32", "bias": True, "temperature": 1.0},
        # one short answer to learn from: as many rows as a request has tokens, the weight read and its gradient written
        {"name": "loss_answer", "op": "loss", "sequences": 1, "length": 8, "dim": 2048, "vocab": 32000,
         "dtype": "bfloat16", "bias": False, "temperature": 1.0},
        # odd sizes throughout: an odd vocabulary, an odd width, a bias
        {"name": "loss_odd", "op": "loss", "sequences": 17, "length": 59, "dim": 1025, "vocab": 50001,
         "dtype": "float16", "bias": True, "temperature": 1.0},
        # fp32 training of a middle-sized head
        {"name": "loss_fp32", "op": "loss", "sequences": 16, "length": 128, "dim": 1024, "vocab": 32000,
         "dtype": "float32", "bias": False, "temperature": 1.0},
        # a training batch, padded to a common length
        {"name": "loss_batch", "op": "loss", "sequences": 8, "length": 511, "dim": 2048, "vocab": 32000,
         "dtype": "bfloat16", "bias": False, "temperature": 1.0},
        # the largest: long responses over a large vocabulary
        {"name": "loss_long", "op": "loss", "sequences": 8, "length": 1023, "dim": 4096, "vocab": 128000,
         "dtype": "bfloat16", "bias": False, "temperature": 1.0},
        # two short pairs of responses scored by the reference: few rows over an odd vocabulary
        {"name": "score_pairs", "op": "score", "sequences": 4, "length": 11, "dim": 2048, "vocab": 50001,
         "dtype": "bfloat16", "bias": True, "temperature": 1.0},
        # a batch of sampled responses scored at the temperature they were sampled with
        {"name": "score_batch", "op": "score", "sequences": 8, "length": 511, "dim": 4096, "vocab": 128000,
         "dtype": "bfloat16", "bias": False, "temperature": 0.8},
        # the hidden layer of the small token policy
        {"name": "dropout_hidden", "op": "dropout", "rows": 512, "dim": 160, "pitch": 160, "dtype": "float32",
         "p": 0.1, "residual": False, "counter": "host"},
        # a training batch's stream of rows, the dropped branch added to it; the counter lies on the device, as
        # a captured step's does
        {"name": "dropout_stream", "op": "dropout", "rows": 16384, "dim": 4096, "pitch": 4096, "dtype": "bfloat16",
         "p": 0.1, "residual": True, "counter": "device"},
        # its backward pass
        {"name": "dropout_grad_stream", "op": "dropout_grad", "rows": 16384, "dim": 4096, "pitch": 4096,
         "dtype": "bfloat16", "p": 0.1, "residual": False, "counter": "device"},
        # a part of wider rows, of an odd width
        {"name": "dropout_grad_odd", "op": "dropout_grad", "rows": 4088, "dim": 1025, "pitch": 1031,
         "dtype": "float16", "p": 0.5, "residual": False, "counter": "host"},
    ]


def _size(rng, lo: int, hi: int) -> int:
    """A size spread over the logarithm of its range; half of them a multiple of 8, as widths often are."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 8:
        n = n // 8 * 8
    return max(lo, min(hi, n))


def draw(rng) -> dict:
    op = rng.choice(["loss", "loss", "score", "dropout", "dropout_grad"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    if op in ("loss", "score"):
        rows, dim = _size(rng, 1, 8184), _size(rng, 16, 4096)
        room = LARGEST // (rows * dim) // (8 if dtype == "float32" else 1)
        vocab = _size(rng, 4, max(4, min(128000, room)))
        sequences = _size(rng, 1, max(1, min(64, rows)))
        return {"op": op, "sequences": sequences, "length": max(1, rows // sequences), "dim": dim, "vocab": vocab,
                "dtype": dtype, "bias": rng.random() < 0.4, "temperature": rng.choice([1.0, 1.0, 0.8, 1.3])}
    dim = _size(rng, 16, 4096)
    return {"op": op, "rows": _size(rng, 1, 16384), "dim": dim, "pitch": dim + rng.choice([0, 0, 8, 5]),
            "dtype": dtype, "p": rng.choice([0.05, 0.1, 0.2, 0.5]),
            "residual": op == "dropout" and rng.random() < 0.5, "counter": rng.choice(["host", "device"])}


# ---------------------------------------------------------------------------
# sizes that follow from a case alone

def _lengths(case) -> np.ndarray:
    """Response lengths of a padded batch: between 60 and 100 per cent of the padded length."""
    r = random.Random(f"lengths {case['sequences']} {case['length']}")
    return np.array([max(1, round(case["length"] * r.uniform(0.6, 1.0))) for _ in range(case["sequences"])])


def work(case) -> dict:
    size, d = SIZES[case["dtype"]], case["dim"]
    if case["op"] in ("loss", "score"):
        n, v, grad = case["sequences"] * case["length"], case["vocab"], case["op"] == "loss"
        live = int(_lengths(case).sum())
        return {"bytes": size * (d * (v * (1 + grad) + live + n * grad) + v * case["bias"] * (1 + grad)) + n * (8 + 1 + 4),
                "flops": 2 * live * d * v * (3 if grad else 1)}
    n = case["rows"] * d
    return {"bytes": size * n * (2 + case["residual"]), "flops": n * (1 + case["residual"])}


# ---------------------------------------------------------------------------
# inputs

def _tokens(n: int, vocab: int, gen) -> torch.Tensor:
    """Tokens in order of falling frequency, as a vocabulary is: the share of the first v is (v / vocab)^(1/3)."""
    u = torch.rand(n, device="cuda", generator=gen)
    return (u * u * u * vocab).long().clamp_(max=vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if case["op"] in ("loss", "score"):
        B, T, D, V = case["sequences"], case["length"], case["dim"], case["vocab"]
        # logits of a partly trained network: a spread of 2, the right token's raised
        weight = torch.empty(V, D, device="cuda", dtype=dtype).normal_(0.0, 2.0 / math.sqrt(D), generator=gen)
        ids = _tokens(B * T, V, gen)
        lift = torch.rand(B * T, 1, device="cuda", generator=gen) * (math.log(V) + 4.0)
        # the network answers for T + 1 positions; the last predicts nothing that is learned
        hidden = normal(B, T + 1, D)
        hidden[:, :T] += (lift / 4.0 * weight[ids].float()).view(B, T, D)
        s["hidden"] = hidden.to(dtype)[:, :T]
        s["weight"], s["ids"] = weight, ids.view(B, T)
        s["head_bias"] = (normal(V) * 0.5).to(dtype) if case["bias"] else None
        lengths = torch.from_numpy(_lengths(case)).cuda()
        s["mask"] = torch.arange(T, device="cuda")[None, :] < lengths[:, None]
        return s
    rows = lambda: normal(case["rows"], case["pitch"]).to(dtype)[:, :case["dim"]]  # noqa: E731
    s["x"] = rows()
    s["stream"] = rows() if case["residual"] else None
    s["seed"] = 0x9E3779B97F4A7C15 ^ int(seed)
    s["at"] = 12 * 1000 + int(seed) % 1000        # a layer's place in a step
    if case["counter"] == "device":
        s["at"] = torch.full((), s["at"], dtype=torch.int64, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass

def run(s):
    if own:
        return _call(s)
    return {"loss": _loss, "score": _loss, "dropout": _dropout, "dropout_grad": _dropout}[s["op"]](s)


def _call(s):
    from boundflow_amd import training

    if s["op"] in ("loss", "score"):
        r = training.vocabulary_loss(s["hidden"], s["weight"], s["ids"], bias=s["head_bias"], mask=s["mask"],
                                     temperature=s["temperature"], with_grad=s["op"] == "loss")
        return {"loss": r.loss, "logp": r.logp, "hidden": r.grad_hidden, "weight": r.grad_weight, "bias": r.grad_bias}
    if s["op"] == "dropout":
        return training.dropout(s["x"], s["p"], seed=s["seed"], counter=s["at"], residual=s["stream"])
    return training.dropout_grad(s["x"], s["p"], seed=s["seed"], counter=s["at"])


def _loss(s):
    hidden, weight, bias, inv_t = s["hidden"], s["weight"], s["head_bias"], 1.0 / s["temperature"]
    x = hidden.float().flatten(0, 1)
    w = weight.float()
    ids, live = s["ids"].flatten(), s["mask"].flatten()
    z = x @ w.t()
    if bias is not None:
        z += bias.float()
    z *= inv_t
    z -= z.amax(1, keepdim=True)
    chosen = z.gather(1, ids[:, None])
    p = z.exp_()
    total = p.sum(1, keepdim=True)
    logp = torch.where(live, (chosen - total.log())[:, 0], 0.0)
    count = live.sum().clamp(min=1)
    out = {"loss": -logp.sum() / count, "logp": logp.view(s["ids"].shape), "hidden": None, "weight": None,
           "bias": None}
    if s["op"] == "score":
        return out
    g = p.div_(total)
    g.scatter_add_(1, ids[:, None], torch.full_like(chosen, -1.0))
    g *= torch.where(live, inv_t / count, 0.0)[:, None]
    out["hidden"] = (g @ w).to(hidden.dtype).view(hidden.shape)
    out["weight"] = (g.t() @ x).to(weight.dtype)
    if bias is not None:
        out["bias"] = g.sum(0).to(bias.dtype)
    return out


def _fields(count: int, seed: int, at, device) -> torch.Tensor:
    """``count`` random 16-bit numbers: eight from each block of the Philox generator of four 32-bit words and
    ten rounds, whose counter is (block, ``at``) and whose key is the seed, in 64-bit integers."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 7) // 8, device=device, dtype=torch.int64)
    at = at if isinstance(at, torch.Tensor) else torch.full((), at, dtype=torch.int64, device=device)
    at = at.expand_as(block)
    a, b, c, d = block & low, block >> 32, at & low, at >> 32
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        one, two = a * 0xD2511F53, c * 0xCD9E8D57          # modulo 2^64: their 64 bits are right
        a, b, c, d = ((two >> 32) & low) ^ b ^ k0, two & low, ((one >> 32) & low) ^ d ^ k1, one & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([a, b, c, d], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).flatten()[:count]


def _dropout(s):
    x = s["x"]
    border = int(s["p"] * 65536 + 0.5)
    kept = _fields(x.numel(), s["seed"], s["at"], x.device).view(x.shape) >= border
    y = torch.where(kept, x.float() * (65536.0 / (65536 - border)), 0.0)
    if s["stream"] is not None:
        y += s["stream"].float()
    return y.to(x.dtype)


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_dropout(s) if case["op"].startswith("dropout") else _exact_loss(s)


def _exact_loss(s):
    """Row by row in pieces of 512: only rows that count."""
    hidden, weight = s["hidden"].double(), s["weight"].double()
    inv_t, learn = 1.0 / s["temperature"], s["op"] == "loss"
    bias = 0.0 if s["head_bias"] is None else s["head_bias"].double()
    rows = s["mask"].flatten().nonzero()[:, 0]
    n = rows.numel()
    logp = torch.zeros(s["ids"].numel(), dtype=torch.float64, device=weight.device)
    dx = torch.zeros(hidden.shape, dtype=torch.float64, device=weight.device).flatten(0, 1)
    dw, db = torch.zeros_like(weight) if learn else None, torch.zeros_like(weight[:, 0])
    flat, ids = hidden.flatten(0, 1), s["ids"].flatten()
    for part in rows.split(512):
        x, y = flat[part], ids[part]
        q = torch.log_softmax((torch.mm(x, weight.t()) + bias) * inv_t, 1)
        logp[part] = q[torch.arange(part.numel(), device=q.device), y]
        if learn:
            q = q.exp_()
            q[torch.arange(part.numel(), device=q.device), y] -= 1.0
            q *= inv_t / n
            dx[part] = torch.mm(q, weight)
            dw.addmm_(q.t(), x)
            db += q.sum(0)
    return {"loss": -logp.sum() / max(n, 1), "logp": logp.view(s["ids"].shape),
            "hidden": dx.view(hidden.shape) if learn else None, "weight": dw,
            "bias": db if learn and s["head_bias"] is not None else None}


def _exact_dropout(s):
    """The generator in numpy's unsigned 32-bit numbers, two elements a word."""
    x = s["x"].double().cpu().numpy()
    at = int(s["at"])
    blocks = np.arange(-(-x.size // 8), dtype=np.uint64)
    word = [blocks.astype(np.uint32), (blocks >> np.uint64(32)).astype(np.uint32),
            np.full(blocks.shape, at & 0xFFFFFFFF, np.uint32), np.full(blocks.shape, at >> 32, np.uint32)]
    for turn in range(10):
        keys = [np.uint32(((s["seed"] & 0xFFFFFFFF) + turn * 0x9E3779B9) & 0xFFFFFFFF),
                np.uint32(((s["seed"] >> 32) + turn * 0xBB67AE85) & 0xFFFFFFFF)]
        products = [word[0].astype(np.uint64) * np.uint64(0xD2511F53), word[2].astype(np.uint64) * np.uint64(0xCD9E8D57)]
        high = [(p >> np.uint64(32)).astype(np.uint32) for p in products]
        lower = [p.astype(np.uint32) for p in products]
        word = [high[1] ^ word[1] ^ keys[0], lower[1], high[0] ^ word[3] ^ keys[1], lower[0]]
    drawn = np.ascontiguousarray(np.stack(word, 1)).view("<u2").reshape(-1)[:x.size].reshape(x.shape)
    border = int(s["p"] * 65536 + 0.5)
    y = np.where(drawn >= border, x / (1.0 - border / 65536.0), 0.0)
    if s["stream"] is not None:
        y = y + s["stream"].double().cpu().numpy()
    return torch.from_numpy(y)
