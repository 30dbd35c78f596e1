"""What the training operators allocate, and hand to the library as addresses, without a device: the
library call is replaced by a recorder, so the tensors can lie on the CPU."""

import pytest
import torch

from boundflow_amd import _lib, training


@pytest.fixture
def recorded(monkeypatch):
    """(tensors allocated, calls made) while the operators run on CPU tensors."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run python -m boundflow_amd.build)")
    made, calls = [], []
    for owner, name in ((torch, "empty"), (torch, "zeros"), (torch.Tensor, "new_empty")):
        def record(*args, real=getattr(owner, name), **kw):
            made.append(real(*args, **kw))
            return made[-1]
        monkeypatch.setattr(owner, name, record)
    monkeypatch.setattr(training, "_current_device", lambda t, name: -1)
    monkeypatch.setattr(training, "_on_device", lambda t, dev, name: None)
    monkeypatch.setattr(training, "current_raw_stream", lambda dev: None)
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.append((name, args)))
    return made, calls


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64], ids=str)
def default_type(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


def fp32(*shape):
    return torch.ones(*shape, dtype=torch.float32)


def test_buffers_are_fp32_whatever_the_default_type(recorded, default_type):
    """fp32 inputs: everything that a kernel writes is fp32 (token arrays and 8-bit moments aside)."""
    made, calls = recorded
    tokens = torch.ones(3000, dtype=torch.int64)
    training.embed_tokens_grad(fp32(3000, 4), tokens, 5)
    training.embed_tokens_grad(fp32(3000, 4), tokens, 5, accumulate_into=fp32(5, 4))
    r = training.policy_loss(fp32(300, 700), tokens[:300], fp32(300), fp32(300))
    q = training.preference_loss(fp32(30, 70), tokens[:30], fp32(30), torch.tensor([0, 20, 30]))
    for t in (r.stats, r.loss, r.logp, r.grad_logits, q.loss, q.rewards, q.logp, q.grad_logits):
        assert t.dtype == torch.float32
    weights = [fp32(200), fp32(3, 5)]
    for bits in (32, 8):
        moments = training.adamw_moments(weights, bits=bits, master=True)
        training.adamw_step(weights, [fp32(200), fp32(3, 5)], moments, step=1)
        assert moments.master.dtype == torch.float32
    assert [name for name, _ in calls] == ["bf_embed_grad"] * 2 + ["bf_policy_loss", "bf_preference_loss"] + \
        ["bf_adamw_multi"] * 2
    assert made and all(t.dtype in (torch.float32, torch.uint8) for t in made), [t.dtype for t in made]


def test_a_table_that_requires_grad_is_refused_where_its_gradient_would_be_lost(recorded):
    _made, calls = recorded
    table, tokens = fp32(4, 6).requires_grad_(True), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(_lib.HipError, match="table.detach()"):
        training.embed_tokens(table, tokens)
    assert not calls
    assert training.embed_tokens(table.detach(), tokens).shape == (3, 6)
    with torch.no_grad():
        assert training.embed_tokens(table, tokens).shape == (3, 6)


def test_a_table_of_one_row_may_have_any_stride(recorded):
    """[1, dim] as a transposed column has row stride 1: the stride of a single row leads nowhere."""
    _made, calls = recorded
    table = fp32(6, 1).t()
    assert table.stride() == (1, 1)
    assert training.embed_tokens(table, torch.zeros(3, dtype=torch.int64)).shape == (3, 6)
    assert calls[0][1][1] >= 6, "the library takes no stride below the width"


@pytest.mark.parametrize("rows,V", [(4, 5), (4, 70001), (40, 50001), (300, 700), (2100, 9), (3000, 2050), (9000, 520)])
def test_results_do_not_keep_the_workspace(recorded, rows, V):
    """A caller that keeps a step's log-probabilities keeps what the results take, and 32 KiB beside them at most."""
    _made, calls = recorded
    logits, tokens = torch.zeros(1, V).expand(rows, V), torch.zeros(rows, dtype=torch.int64)
    r = training.policy_loss(logits, tokens, fp32(rows), fp32(rows), with_grad=False)
    held = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in (r.stats, r.loss, r.logp)}
    assert sum(held.values()) <= 4 * (4 + rows) + 32768 + 16
    q = training.preference_loss(logits, tokens, fp32(rows), torch.tensor([0, rows // 2, rows]), with_grad=False)
    held = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in (q.loss, q.rewards, q.logp)}
    assert sum(held.values()) <= 4 * (3 + rows) + 32768 + 16
    # what kernels get as their workspace starts at a multiple of 16 bytes of its buffer, and lies within one
    lib, made = _lib.load(), {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in recorded[0]}
    for (name, args), need in zip(calls, (lib.bf_policy_loss_workspace(rows, 1, V, 0),
                                          lib.bf_preference_loss_workspace(rows, V, 1, 0))):
        space = args[-2]
        base = max(b for b in made if b <= space)
        assert (space - base) % 16 == 0 and space + 4 * need <= base + made[base], name
