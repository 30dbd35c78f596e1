"""Training operators of token networks on the HIP library.

The networks that the bound queries verify are trained, and repaired after a failed query,
with what is here: the lookup of token rows and its gradient (``embed_tokens``,
``embed_tokens_grad``), two losses of token logits with their gradients (``policy_loss``,
``preference_loss``) and the weights' update (``adamw_step``, ``AdamW``).  A token network is
bounded in embedding space: the looked-up rows are the centre of the input set.

As everywhere in the package, work goes on torch's current stream, gradients come from
explicit calls (hand ``grad_logits`` to ``logits.backward(grad)`` to continue through a network
made with autograd), there is no CPU path, and nothing synchronizes with the host: a value that
is wrong in a tensor on the device (a token past the vocabulary) shows in the result as NaN.
Tensors of fp32, bf16 and fp16; every sum and every softmax is held in fp32.

No counterpart in the reference, which bounds networks and does not train them.
"""

from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import HipError, ptr

_ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}

MOMENT_BLOCK = 128   # elements of an 8-bit moment that share a scale; every tensor's moments start at a multiple


def _device(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise HipError(f"{name} must be a HIP device tensor (the backend has no CPU path)")
    if t.get_device() != torch.cuda.current_device():
        raise HipError(f"{name} is on {t.device}, not on the current device")


def _elem(t: torch.Tensor, name: str) -> int:
    _device(t, name)
    code = _ELEM.get(t.dtype)
    if code is None:
        raise HipError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _tokens(t: torch.Tensor, shape, name: str = "tokens") -> Tuple[torch.Tensor, int]:
    _device(t, name)
    size = _TOKEN_BYTES.get(t.dtype)
    if size is None:
        raise HipError(f"{name} must be int32 or int64, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.contiguous(), size


def _floats(t: torch.Tensor, shape, name: str) -> torch.Tensor:
    _device(t, name)
    if t.dtype != torch.float32:
        raise HipError(f"{name} must be float32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.contiguous()


# ---------------------------------------------------------------------------
# Embedding

def embed_tokens(table: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[tokens]`` ([*tokens.shape, dim], of the table's type, rounded once).

    table [vocab, dim], rows contiguous (any row stride); tokens int32 or int64 of any shape.  A
    negative token is padding and gives zeros, one past the table gives NaN."""
    elem = _elem(table, "table")
    if table.dim() != 2 or (table.stride(1) != 1 and table.shape[1] > 1) or table.stride(0) < table.shape[1]:
        raise HipError(f"table must be [vocab, dim] with contiguous rows, got {tuple(table.shape)} with strides "
                       f"{table.stride()}")
    tokens, token_bytes = _tokens(tokens, None)
    vocab, dim = table.shape
    out = torch.empty(*tokens.shape, dim, dtype=table.dtype, device=table.device)
    _lib.call("bf_embed_rows", ptr(table), table.stride(0), vocab, ptr(tokens), token_bytes, tokens.numel(), dim,
              float(scale), elem, ptr(out), _lib.stream_handle())
    return out


def embed_tokens_grad(grad: torch.Tensor, tokens: torch.Tensor, vocab: int, *, scale: float = 1.0,
                      accumulate_into: Optional[torch.Tensor] = None,
                      dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Gradient of ``embed_tokens`` with respect to its table, from ``grad`` ([*tokens.shape, dim]).

    Row v is ``scale`` times the sum of the rows of the tokens of value v, in fp32 in the tokens'
    order, so it has the same bits on every call; [vocab, dim] of ``dtype`` (grad's type, or
    float32).  With ``accumulate_into`` (float32 [vocab, dim], contiguous) the sums are added to
    it in place and it is returned; rows without a token are not touched.  Tokens outside of
    [0, vocab) take no part."""
    elem = _elem(grad, "grad")
    tokens, token_bytes = _tokens(tokens, grad.shape[:-1])
    dim, count, vocab = grad.shape[-1], tokens.numel(), int(vocab)
    if vocab < 0:
        raise ValueError(f"vocab must be >= 0, got {vocab}")
    rows = grad if grad.dim() == 2 else grad.reshape(count, dim)
    if (dim > 1 and rows.stride(1) != 1) or (count > 1 and rows.stride(0) < dim):
        rows = rows.contiguous()
    if accumulate_into is not None:
        _floats(accumulate_into, (vocab, dim), "accumulate_into")
        if not accumulate_into.is_contiguous():
            raise HipError("accumulate_into must be contiguous")
        if dtype not in (None, torch.float32):
            raise ValueError(f"sums are added to float32, not to {dtype}")
        out = accumulate_into
    else:
        dtype = grad.dtype if dtype is None else dtype
        if dtype not in (grad.dtype, torch.float32):
            raise ValueError(f"dtype must be {grad.dtype} or float32, got {dtype}")
        out = torch.empty(vocab, dim, dtype=dtype, device=grad.device)
    space = torch.empty(_lib.load().bf_embed_grad_workspace(count, vocab, dim), device=grad.device)
    _lib.call("bf_embed_grad", ptr(rows), max(rows.stride(0), dim), elem, ptr(tokens), token_bytes, count, vocab, dim,
              float(scale), _ELEM[out.dtype], int(accumulate_into is not None), ptr(out), ptr(space),
              _lib.stream_handle())
    if accumulate_into is not None:
        torch.autograd.graph.increment_version(out)
    return out


# ---------------------------------------------------------------------------
# Losses

class PolicyLoss(NamedTuple):
    """``stats`` [4]: loss, policy term, KL, share of rows whose clip is active (each a weighted mean)."""

    stats: torch.Tensor
    logp: torch.Tensor
    grad_logits: Optional[torch.Tensor]

    @property
    def loss(self) -> torch.Tensor:
        return self.stats[0]


class PreferenceLoss(NamedTuple):
    """``rewards`` [2 * pairs]: beta times each response's summed log ratio, the chosen ones first."""

    loss: torch.Tensor
    rewards: torch.Tensor
    logp: torch.Tensor
    grad_logits: Optional[torch.Tensor]


def _rows_of(logits: torch.Tensor) -> torch.Tensor:
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        raise HipError(f"logits need a contiguous last axis, got strides {logits.stride()}")
    return logits


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_weight: float = 0.0, temperature: float = 1.0, reduction: str = "token",
                grad_scale: float = 1.0, with_grad: bool = True) -> PolicyLoss:
    """Clipped policy loss with a KL term against a reference policy, and its gradient.

    logits [B, T, V] or [N, V] (a view such as ``all_logits[:, :-1]`` is read in place); tokens,
    old_logp (float32, the log-probabilities the tokens were sampled with), ref_logp (float32) and
    mask (bool) of the leading shape; advantages (float32) of the leading shape, or [B] for one a
    sequence.  With p a token's log-probability at ``temperature``, r = exp(p - old_logp), d = ref_logp - p:

        term = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_weight (exp(d) - d - 1)

    and the loss is the terms' mean over the live rows (``reduction="token"``) or the mean over the
    sequences of each one's mean (``"sequence"``).  A row is live unless it is masked or its token
    is negative; the others are not read, and logp and gradient are 0 there.  A batch without a live
    row has loss 0.  ``grad_logits`` is ``grad_scale`` times the loss's gradient, of the logits' type."""
    elem = _elem(logits, "logits")
    if logits.dim() not in (2, 3) or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [B, T, V] or [N, V] with V >= 1, got {tuple(logits.shape)}")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"unknown reduction: {reduction}")
    if not temperature > 0.0:
        raise ValueError(f"temperature must be >0, got {temperature}")
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise ValueError(f"clip limits must be >=0, got {clip_low}, {clip_high}")
    _rows_of(logits)
    lead = logits.shape[:-1]
    V = logits.shape[-1]
    if logits.dim() == 3:
        B, T = lead
        ld_b, ld_t = logits.stride(0), logits.stride(1)
    else:
        B, T = lead[0], 1
        ld_b, ld_t = logits.stride(0), 0
    tokens, token_bytes = _tokens(tokens, lead)
    old_logp = _floats(old_logp, lead, "old_logp")
    if ref_logp is not None:
        ref_logp = _floats(ref_logp, lead, "ref_logp")
    _device(advantages, "advantages")
    if advantages.dtype != torch.float32:
        raise HipError(f"advantages must be float32, got {advantages.dtype}")
    if advantages.shape == lead:
        adv_b, adv_t = advantages.stride(0), advantages.stride(1) if logits.dim() == 3 else 0
    elif advantages.shape == (B,):
        adv_b, adv_t = advantages.stride(0), 0
    else:
        raise ValueError(f"advantages of shape {tuple(advantages.shape)}, expected {tuple(lead)} or ({B},)")
    if mask is not None:
        _device(mask, "mask")
        if mask.dtype != torch.bool:
            raise HipError(f"mask must be bool, got {mask.dtype}")
        if mask.shape != lead:
            raise ValueError(f"mask of shape {tuple(mask.shape)}, expected {tuple(lead)}")
        mask = mask.contiguous()
    dev = logits.device
    out = torch.empty(4 + B * T, device=dev)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if with_grad else None
    space = torch.empty(_lib.load().bf_policy_loss_workspace(B, T, V, elem), device=dev)
    _lib.call("bf_policy_loss", ptr(logits), elem, B, T, V, ld_b, ld_t, ptr(tokens), token_bytes, ptr(old_logp),
              ptr(ref_logp), ptr(advantages), adv_b, adv_t, ptr(mask), float(clip_low), float(clip_high),
              float(kl_weight), float(temperature), int(reduction == "sequence"), float(grad_scale), ptr(out[4:]),
              ptr(out), ptr(grad), ptr(space), _lib.stream_handle())
    return PolicyLoss(out[:4], out[4:].view(lead), grad)


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, ref_logp: torch.Tensor, offsets: torch.Tensor, *,
                    beta: float = 0.1, label_smoothing: float = 0.0, grad_scale: float = 1.0,
                    with_grad: bool = True) -> PreferenceLoss:
    """Preference loss of chosen and rejected responses, and its gradient.

    The responses' rows lie one after another: logits [N, V] (any row stride), tokens [N], ref_logp
    [N] (float32, the reference's log-probabilities of the tokens), offsets int64 [2 * pairs + 1]
    ascending, response k being rows offsets[k] to offsets[k + 1] (it may be empty): the chosen
    ones first, then the rejected ones in the same order.  With s the sum of logp - ref_logp over a
    response and h = beta (s_chosen - s_rejected),

        loss = mean over pairs of -(1 - label_smoothing) log sigma(h) - label_smoothing log sigma(-h).

    Rows of no response and rows of a negative token take no part (logp and gradient 0)."""
    elem = _elem(logits, "logits")
    if logits.dim() != 2 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [N, V] with V >= 1, got {tuple(logits.shape)}")
    _rows_of(logits)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
    N, V = logits.shape
    tokens, token_bytes = _tokens(tokens, (N,))
    ref_logp = _floats(ref_logp, (N,), "ref_logp")
    _device(offsets, "offsets")
    if offsets.dtype != torch.int64:
        raise HipError(f"offsets must be int64, got {offsets.dtype}")
    if offsets.dim() != 1 or offsets.numel() % 2 == 0:
        raise ValueError(f"offsets must be [2 * pairs + 1], got {tuple(offsets.shape)}")
    offsets = offsets.contiguous()
    pairs = offsets.numel() // 2
    dev = logits.device
    # loss, rewards and logp in one allocation
    out = torch.empty(1 + 2 * pairs + N, device=dev)
    logp = out[1 + 2 * pairs:]
    grad = torch.empty(N, V, dtype=logits.dtype, device=dev) if with_grad else None
    space = torch.empty(_lib.load().bf_preference_loss_workspace(N, V, pairs, elem), device=dev)
    _lib.call("bf_preference_loss", ptr(logits), elem, N, V, logits.stride(0), ptr(tokens), token_bytes, ptr(ref_logp),
              ptr(offsets), pairs, float(beta), float(label_smoothing), float(grad_scale), ptr(logp), ptr(out[1:]),
              ptr(out), ptr(grad), ptr(space), _lib.stream_handle())
    return PreferenceLoss(out[0], out[1:1 + 2 * pairs], logp, grad)


# ---------------------------------------------------------------------------
# AdamW

class AdamWMoments(NamedTuple):
    """Moments of a list of weights, flat: tensor k's elements start at the sum of the sizes before it,
    each rounded up to ``MOMENT_BLOCK``.

    In 32 bits ``m`` and ``v`` are float32 and the scales None; in 8 bits ``m`` and ``v`` are
    float8_e4m3fn, m and sqrt(v) over the ``m_scale`` and ``v_scale`` (float32) of their block.
    ``master``: float32 copies of the weights in the same layout, or None."""

    m: torch.Tensor
    v: torch.Tensor
    m_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None
    master: Optional[torch.Tensor] = None


def moment_offsets(sizes: Sequence[int]) -> List[int]:
    """First element of every tensor in the flat moments, and their length."""
    at = [0]
    for n in sizes:
        at.append(at[-1] + -(-int(n) // MOMENT_BLOCK) * MOMENT_BLOCK)
    return at


def adamw_moments(params: Sequence[torch.Tensor], *, bits: int = 32, master: bool = False) -> AdamWMoments:
    """Zero moments for ``params`` (``bits`` 32 or 8); with ``master`` fp32 copies of the weights."""
    if bits not in (32, 8):
        raise ValueError(f"bits must be 32 or 8, got {bits}")
    if not params:
        raise ValueError("no parameters")
    for k, p in enumerate(params):
        _elem(p, f"params[{k}]")
    dev = params[0].device
    at = moment_offsets([p.numel() for p in params])
    total = at[-1]
    copies = None
    if master:
        copies = torch.zeros(total, device=dev)
        for a, p in zip(at, params):
            copies[a:a + p.numel()].copy_(p.detach().reshape(-1))
    if bits == 32:
        return AdamWMoments(torch.zeros(total, device=dev), torch.zeros(total, device=dev), None, None, copies)
    m, v = (torch.zeros(total, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    scales = [torch.zeros(total // MOMENT_BLOCK, device=dev) for _ in range(2)]
    return AdamWMoments(m, v, scales[0], scales[1], copies)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], moments: AdamWMoments, *, step: int,
               lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, grad_scale: Union[float, torch.Tensor] = 1.0) -> None:
    """One AdamW step (torch.optim.AdamW's formula) over all ``params``, in place.

    ``step`` counts from 1.  params of one type and grads of one type (each float32, bfloat16 or
    float16), contiguous, pairwise of the same shape.  ``grad_scale`` multiplies every gradient: a
    number, or a float32 scalar tensor on the device (the factor of a clipped norm).  The step is
    computed in fp32 and each weight rounded once; with ``moments.master`` the copies are stepped
    and the weights follow them.  The parameters' versions are raised, so that bound queries remake
    what they keep of them."""
    if len(params) != len(grads):
        raise ValueError(f"{len(params)} parameters, {len(grads)} gradients")
    if step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    if not params:
        return
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0):
        raise ValueError(f"betas must be in [0, 1) and eps >=0, got {betas}, {eps}")
    p_elem, g_elem = _elem(params[0], "params[0]"), _elem(grads[0], "grads[0]")
    p_type, g_type, dev = params[0].dtype, grads[0].dtype, params[0].device
    sizes, total = [], 0
    for k, (p, g) in enumerate(zip(params, grads)):
        if p.dtype != p_type or g.dtype != g_type or p.device != dev or g.device != dev:
            raise HipError(f"params[{k}] and grads[{k}] must be {p_type} and {g_type} on {dev}, as the first are")
        if p.shape != g.shape:
            raise ValueError(f"params[{k}] of shape {tuple(p.shape)}, grads[{k}] of {tuple(g.shape)}")
        if not (p.is_contiguous() and g.is_contiguous()):
            raise HipError(f"params[{k}] and grads[{k}] must be contiguous")
        n = p.numel()
        sizes.append(n)
        total += -(-n // MOMENT_BLOCK) * MOMENT_BLOCK
    m, v, m_scale, v_scale, master = moments
    eight = m_scale is not None or v_scale is not None
    kind = torch.float8_e4m3fn if eight else torch.float32
    expected = [("m", m, kind, total), ("v", v, kind, total)]
    if eight:
        expected += [("m_scale", m_scale, torch.float32, total // MOMENT_BLOCK),
                     ("v_scale", v_scale, torch.float32, total // MOMENT_BLOCK)]
    if master is not None:
        expected.append(("master", master, torch.float32, total))
    for name, t, want, length in expected:
        if t is None:
            raise ValueError(f"moments.{name} is missing")
        _device(t, f"moments.{name}")
        if t.dtype != want:
            raise HipError(f"moments.{name} must be {want}, got {t.dtype}")
        if t.numel() != length or not t.is_contiguous():
            raise ValueError(f"moments.{name} must be flat of {length} elements, got {tuple(t.shape)}")
    factor, factor_dev = grad_scale, None
    if isinstance(grad_scale, torch.Tensor):
        _device(grad_scale, "grad_scale")
        if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
            raise HipError("grad_scale must be a float32 scalar")
        factor, factor_dev = 1.0, grad_scale
    _lib.call("bf_adamw_multi", len(sizes), _lib.ptr_array(params), _lib.ptr_array(grads), _lib.i64_array(sizes), p_elem,
              g_elem, ptr(m), ptr(v), ptr(m_scale), ptr(v_scale), ptr(master), float(lr), float(b1), float(b2),
              float(eps), float(weight_decay), int(step), float(factor), ptr(factor_dev), _lib.stream_handle())
    torch.autograd.graph.increment_version([*params, *(t for t in moments if t is not None)])


class AdamW:
    """AdamW over a fixed list of parameters: their moments and the step count around ``adamw_step``."""

    def __init__(self, params: Sequence[torch.Tensor], *, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, bits: int = 32, master: bool = False):
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.moments = adamw_moments(self.params, bits=bits, master=master)
        self.t = 0

    def step(self, grads: Optional[Sequence[torch.Tensor]] = None, *, lr: Optional[float] = None,
             grad_scale: Union[float, torch.Tensor] = 1.0) -> None:
        """One step with ``grads`` (the parameters' ``.grad`` where none are given)."""
        if grads is None:
            grads = [p.grad for p in self.params]
            missing = [k for k, g in enumerate(grads) if g is None]
            if missing:
                raise ValueError(f"parameters {missing} have no gradient")
        adamw_step(self.params, grads, self.moments, step=self.t + 1, lr=self.lr if lr is None else lr,
                   betas=self.betas, eps=self.eps, weight_decay=self.weight_decay, grad_scale=grad_scale)
        self.t += 1

    def moment(self, k: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(m, v) of parameter k as float32 tensors of its shape (what 8-bit moments stand for)."""
        at = moment_offsets([p.numel() for p in self.params])
        p, lo, hi = self.params[k], at[k], at[k + 1]
        m, v, m_scale, v_scale, _master = self.moments
        m, v = m[lo:hi].float(), v[lo:hi].float()
        if m_scale is not None:
            blocks = slice(lo // MOMENT_BLOCK, hi // MOMENT_BLOCK)
            m = (m.view(-1, MOMENT_BLOCK) * m_scale[blocks, None]).view(-1)
            v = (v.view(-1, MOMENT_BLOCK) * v_scale[blocks, None]).view(-1).square()
        return m[:p.numel()].view(p.shape), v[:p.numel()].view(p.shape)
