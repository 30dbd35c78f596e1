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

import ctypes
from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import HipError, current_raw_stream

_ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}

MOMENT_BLOCK = 128   # elements of an 8-bit moment that share a scale; every tensor's moments start at a multiple


# Every call checks a dozen tensors before a kernel of a few microseconds: the checks are plain
# attribute reads, and addresses go to the library as numbers (the tensors are this module's
# callers' or its own locals until the call has enqueued its kernels).  What the kernels write in
# fp32 is allocated as such by name: a program for 16-bit networks may have another default type.

def _current_device(t: torch.Tensor, name: str) -> int:
    """The device of the call's first tensor, which has to be the current one."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise HipError(f"{name} must be a HIP device tensor (the backend has no CPU path)")
    dev = t.get_device()
    if dev != torch.cuda.current_device():
        raise HipError(f"{name} is on {t.device}, not on the current device")
    return dev


def _on_device(t: torch.Tensor, dev: int, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise HipError(f"{name} must be a HIP device tensor (the backend has no CPU path)")
    if t.get_device() != dev:
        raise HipError(f"{name} is on {t.device}, not on the current device")


def _elem(t: torch.Tensor, name: str) -> int:
    code = _ELEM.get(t.dtype)
    if code is None:
        raise HipError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _tokens(t: torch.Tensor, shape, dev: int) -> Tuple[torch.Tensor, int]:
    _on_device(t, dev, "tokens")
    size = _TOKEN_BYTES.get(t.dtype)
    if size is None:
        raise HipError(f"tokens must be int32 or int64, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"tokens of shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.is_contiguous() else t.contiguous(), size


def _floats(t: torch.Tensor, shape, dev: int, name: str) -> torch.Tensor:
    _on_device(t, dev, name)
    if t.dtype != torch.float32:
        raise HipError(f"{name} must be float32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} of shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# Embedding

def embed_tokens(table: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[tokens]`` ([*tokens.shape, dim], of the table's type, rounded once).

    table [vocab, dim], rows contiguous (any row stride); tokens int32 or int64 of any shape.  A
    negative token is padding and gives zeros, one past the table gives NaN.  The rows come without a
    graph: a table that requires grad is refused while gradients are recorded (pass ``table.detach()``),
    because a ``backward()`` through the network would leave it untrained without an error."""
    dev = _current_device(table, "table")
    elem = _elem(table, "table")
    if table.requires_grad and torch.is_grad_enabled():
        raise HipError("table requires grad, but the rows come without a graph: pass table.detach() and get its "
                       "gradient from embed_tokens_grad")
    if table.dim() != 2:
        raise HipError(f"table must be [vocab, dim], got {tuple(table.shape)}")
    vocab, dim = table.shape
    ld, step = table.stride()
    if vocab <= 1:
        ld = dim      # a single row's stride leads nowhere, and may be anything
    if (step != 1 and dim > 1) or ld < dim:
        raise HipError(f"table must be [vocab, dim] with contiguous rows, got {tuple(table.shape)} with strides "
                       f"{table.stride()}")
    tokens, token_bytes = _tokens(tokens, None, dev)
    out = torch.empty((*tokens.shape, dim), dtype=table.dtype, device=table.device)
    _lib.call("bf_embed_rows", table.data_ptr(), ld, vocab, tokens.data_ptr(), token_bytes, tokens.numel(), dim,
              float(scale), elem, out.data_ptr(), current_raw_stream(dev))
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
    dev = _current_device(grad, "grad")
    elem = _elem(grad, "grad")
    if grad.dim() < 1:
        raise ValueError("grad must be [*tokens.shape, dim]")
    tokens, token_bytes = _tokens(tokens, grad.shape[:-1], dev)
    dim, count, vocab = grad.shape[-1], tokens.numel(), int(vocab)
    if vocab < 0:
        raise ValueError(f"vocab must be >= 0, got {vocab}")
    rows = grad if grad.dim() == 2 else grad.reshape(count, dim)
    if (dim > 1 and rows.stride(1) != 1) or (count > 1 and rows.stride(0) < dim):
        rows = rows.contiguous()
    if accumulate_into is not None:
        _floats(accumulate_into, (vocab, dim), dev, "accumulate_into")
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
    need = _lib.load().bf_embed_grad_workspace(count, vocab, dim)
    space = torch.empty(need, dtype=torch.float32, device=grad.device) if need else None
    _lib.call("bf_embed_grad", rows.data_ptr(), max(rows.stride(0), dim), elem, tokens.data_ptr(), token_bytes, count,
              vocab, dim, float(scale), _ELEM[out.dtype], accumulate_into is not None, out.data_ptr(), _address(space),
              current_raw_stream(dev))
    if accumulate_into is not None:
        torch.autograd.graph.increment_version(out)
    return out


# ---------------------------------------------------------------------------
# Losses

# A loss's small results are views of one buffer, and a workspace of up to this many floats lies behind them: a second
# allocation takes 1.2 us of the host, and a call on few rows (up to 2048 parts of 8 bytes) waits for the host (45
# preference rows 20.0 us against 21.0).  A larger one is a buffer of its own, or a caller that keeps a result would keep
# it too.
_SHARED_WORKSPACE = 8192


def _results_and_workspace(own: int, need: int, like: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """(``own`` floats of results, the buffer of ``need`` floats of workspace, the workspace's address), fp32 as
    ``like`` is and on its device."""
    if need > _SHARED_WORKSPACE:
        space = like.new_empty(need)
        return like.new_empty(own), space, space.data_ptr()
    out = like.new_empty(own + 3 + need)
    return out, out, out.data_ptr() + (own + 3) // 4 * 16


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
    dev = _current_device(logits, "logits")
    elem = _elem(logits, "logits")
    shape = logits.shape
    dims = len(shape)
    if dims not in (2, 3) or shape[-1] < 1:
        raise ValueError(f"logits must be [B, T, V] or [N, V] with V >= 1, got {tuple(shape)}")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"unknown reduction: {reduction}")
    if not temperature > 0.0:
        raise ValueError(f"temperature must be >0, got {temperature}")
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise ValueError(f"clip limits must be >=0, got {clip_low}, {clip_high}")
    strides = logits.stride()
    lead, V = shape[:-1], shape[-1]
    if strides[-1] != 1 and V > 1:
        raise HipError(f"logits need a contiguous last axis, got strides {strides}")
    B, T = (lead[0], lead[1]) if dims == 3 else (lead[0], 1)
    tokens, token_bytes = _tokens(tokens, lead, dev)
    old_logp = _floats(old_logp, lead, dev, "old_logp")
    if ref_logp is not None:
        ref_logp = _floats(ref_logp, lead, dev, "ref_logp")
    _on_device(advantages, dev, "advantages")
    if advantages.dtype != torch.float32:
        raise HipError(f"advantages must be float32, got {advantages.dtype}")
    if advantages.shape == lead:
        adv = advantages.stride()
        adv_b, adv_t = (adv[0], adv[1]) if dims == 3 else (adv[0], 0)
    elif advantages.shape == (B,):
        adv_b, adv_t = advantages.stride(0), 0
    else:
        raise ValueError(f"advantages of shape {tuple(advantages.shape)}, expected {tuple(lead)} or ({B},)")
    if mask is not None:
        _on_device(mask, dev, "mask")
        if mask.dtype != torch.bool:
            raise HipError(f"mask must be bool, got {mask.dtype}")
        if mask.shape != lead:
            raise ValueError(f"mask of shape {tuple(mask.shape)}, expected {tuple(lead)}")
        if not mask.is_contiguous():
            mask = mask.contiguous()
    N = B * T
    # stats, logp
    out, _space, space = _results_and_workspace(4 + N, _lib.load().bf_policy_loss_workspace(B, T, V, elem), old_logp)
    grad = logits.new_empty(shape) if with_grad else None
    at = out.data_ptr()
    _lib.call("bf_policy_loss", logits.data_ptr(), elem, B, T, V, strides[0], strides[1] if dims == 3 else 0,
              tokens.data_ptr(), token_bytes, old_logp.data_ptr(), _address(ref_logp), advantages.data_ptr(), adv_b, adv_t,
              _address(mask), float(clip_low), float(clip_high), float(kl_weight), float(temperature),
              reduction == "sequence", float(grad_scale), at + 16,
              at, _address(grad), space, current_raw_stream(dev))
    return PolicyLoss(out[:4], out[4:4 + N].view(lead), grad)


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
    dev = _current_device(logits, "logits")
    elem = _elem(logits, "logits")
    shape = logits.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"logits must be [N, V] with V >= 1, got {tuple(shape)}")
    N, V = shape
    ld, step = logits.stride()
    if step != 1 and V > 1:
        raise HipError(f"logits need a contiguous last axis, got strides {logits.stride()}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")
    tokens, token_bytes = _tokens(tokens, (N,), dev)
    ref_logp = _floats(ref_logp, (N,), dev, "ref_logp")
    _on_device(offsets, dev, "offsets")
    if offsets.dtype != torch.int64:
        raise HipError(f"offsets must be int64, got {offsets.dtype}")
    count = offsets.numel()
    if offsets.dim() != 1 or count % 2 == 0:
        raise ValueError(f"offsets must be [2 * pairs + 1], got {tuple(offsets.shape)}")
    if not offsets.is_contiguous():
        offsets = offsets.contiguous()
    pairs = count // 2
    own = 1 + 2 * pairs + N   # loss, rewards, logp
    out, _space, space = _results_and_workspace(own, _lib.load().bf_preference_loss_workspace(N, V, pairs, elem),
                                                ref_logp)
    grad = logits.new_empty(shape) if with_grad else None
    at = out.data_ptr()
    _lib.call("bf_preference_loss", logits.data_ptr(), elem, N, V, ld, tokens.data_ptr(), token_bytes,
              ref_logp.data_ptr(), offsets.data_ptr(), pairs, float(beta), float(label_smoothing), float(grad_scale),
              at + 4 + 8 * pairs, at + 4,
              at, _address(grad), space, current_raw_stream(dev))
    return PreferenceLoss(out[0], out[1:1 + 2 * pairs], out[1 + 2 * pairs:own], grad)


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
        _on_device(p, _current_device(params[0], "params[0]"), f"params[{k}]")
        _elem(p, f"params[{k}]")
    dev = params[0].device
    at = moment_offsets([p.numel() for p in params])
    total = at[-1]
    copies = None
    if master:
        copies = torch.zeros(total, dtype=torch.float32, device=dev)
        for a, p in zip(at, params):
            copies[a:a + p.numel()].copy_(p.detach().reshape(-1))
    if bits == 32:
        m, v = (torch.zeros(total, dtype=torch.float32, device=dev) for _ in range(2))
        return AdamWMoments(m, v, None, None, copies)
    m, v = (torch.zeros(total, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    scales = [torch.zeros(total // MOMENT_BLOCK, dtype=torch.float32, device=dev) for _ in range(2)]
    return AdamWMoments(m, v, scales[0], scales[1], copies)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], moments: AdamWMoments, *, step: int,
               lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, grad_scale: Union[float, torch.Tensor] = 1.0) -> None:
    """One AdamW step (torch.optim.AdamW's formula) over all ``params``, in place.

    ``step`` counts from 1.  params of one type and grads of one type (each float32, bfloat16 or
    float16), contiguous, pairwise of the same shape; weights that share memory are refused (tied
    ones are listed once, with their gradients' sum).  ``grad_scale`` multiplies every gradient: a
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
    dev = _current_device(params[0], "params[0]")
    _on_device(grads[0], dev, "grads[0]")
    p_elem, g_elem = _elem(params[0], "params[0]"), _elem(grads[0], "grads[0]")
    p_type, g_type = params[0].dtype, grads[0].dtype
    sizes, total = [], 0
    for k, (p, g) in enumerate(zip(params, grads)):
        if p.dtype != p_type or g.dtype != g_type or p.get_device() != dev or g.get_device() != dev:
            raise HipError(f"params[{k}] and grads[{k}] must be {p_type} and {g_type} on {params[0].device}, as the "
                           "first are")
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
    _moment(m, "m", kind, total, dev)
    _moment(v, "v", kind, total, dev)
    if eight:
        _moment(m_scale, "m_scale", torch.float32, total // MOMENT_BLOCK, dev)
        _moment(v_scale, "v_scale", torch.float32, total // MOMENT_BLOCK, dev)
    if master is not None:
        _moment(master, "master", torch.float32, total, dev)
    factor_dev = None
    if isinstance(grad_scale, torch.Tensor):
        _on_device(grad_scale, dev, "grad_scale")
        if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
            raise HipError("grad_scale must be a float32 scalar")
        factor_dev, grad_scale = grad_scale.data_ptr(), 1.0
    count = len(sizes)
    pointers, lengths = ctypes.c_void_p * count, ctypes.c_int64 * count
    _lib.call("bf_adamw_multi", count, pointers(*[p.data_ptr() for p in params]),
              pointers(*[g.data_ptr() for g in grads]), lengths(*sizes), p_elem, g_elem, m.data_ptr(), v.data_ptr(),
              _address(m_scale), _address(v_scale), _address(master), float(lr), float(b1), float(b2), float(eps),
              float(weight_decay), int(step), float(grad_scale),
              factor_dev, current_raw_stream(dev))
    torch.autograd.graph.increment_version([*params, *(t for t in moments if t is not None)])


def _moment(t: Optional[torch.Tensor], name: str, kind: torch.dtype, length: int, dev: int) -> None:
    if t is None:
        raise ValueError(f"moments.{name} is missing")
    _on_device(t, dev, f"moments.{name}")
    if t.dtype != kind:
        raise HipError(f"moments.{name} must be {kind}, got {t.dtype}")
    if t.numel() != length or not t.is_contiguous():
        raise ValueError(f"moments.{name} must be flat of {length} elements, got {tuple(t.shape)}")


class AdamW:
    """AdamW over a fixed list of parameters: their moments and the step count around ``adamw_step``.

    ``moments`` and ``t`` (steps taken) are the whole state: a checkpoint holds both, and is loaded by setting them."""

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
