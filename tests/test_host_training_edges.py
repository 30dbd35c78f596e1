"""What the training operators' entry points refuse before anything is enqueued.  No device call is made."""

import pytest
import torch

from boundflow_amd import _lib
from oracle import training_ref as ref


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run python -m boundflow_amd.build)")
    return _lib.load()


def adamw(lib, params, grads, sizes, moments, **kw):
    """Status of one step over host memory that must not be reached (the call has to be refused)."""
    args = dict(count=len(sizes), p=_lib.ptr_array(params), g=_lib.ptr_array(grads), n=_lib.i64_array(sizes), p_elem=0,
                g_elem=0, m=moments[0], v=moments[1], m_scale=None, v_scale=None, master=None, lr=0.1, b1=0.9, b2=0.9,
                eps=1e-8, wd=0.0, step=1, scale=1.0, scale_dev=None, stream=None)
    return lib.bf_adamw_multi(*{**args, **kw}.values())


@pytest.mark.parametrize("count", [2, 7, 97, 300])
def test_adamw_refuses_weights_that_share_memory(lib, count):
    flat = torch.zeros(64 * count)
    weights = list(flat.view(count, 64))
    m, v = torch.zeros(128 * count), torch.zeros(128 * count)
    at = [m.data_ptr(), v.data_ptr()]
    sizes = [64] * count
    tied = weights[:-1] + [weights[0]]
    assert adamw(lib, tied, weights, sizes, at) == 1 and b"share memory" in lib.bf_last_error()
    # the last of one is the first of another
    across = weights[:-1] + [flat[63:127]]
    assert adamw(lib, across, weights, sizes, at) == 1 and b"share memory" in lib.bf_last_error()
    assert adamw(lib, weights, weights, sizes, [at[0], at[0]]) == 1 and b"share memory" in lib.bf_last_error()
    assert adamw(lib, weights, weights, sizes, at, master=at[1]) == 1 and b"share memory" in lib.bf_last_error()
    assert adamw(lib, weights, weights, sizes, [flat.data_ptr(), at[1]]) == 1 and b"share memory" in lib.bf_last_error()


def test_adamw_refuses_a_late_tensor_before_it_steps_the_first(lib):
    """More tensors than a launch takes: the 120th is looked at before the first launch."""
    weights = list(torch.zeros(120, 64))
    m, v = torch.zeros(120 * 128), torch.zeros(120 * 128)
    at = [m.data_ptr(), v.data_ptr()]
    assert adamw(lib, weights, weights, [64] * 119 + [-1], at) == 1 and b"tensor 119" in lib.bf_last_error()
    assert adamw(lib, weights, weights[:119] + [None], [64] * 120, at) == 1 and b"tensor 119" in lib.bf_last_error()


def test_sizes_that_no_launch_takes_are_refused_before_the_first(lib):
    """A grid of 2^32 work-items or more is status 3 up front, not a launch that fails behind others."""
    some = torch.zeros(64)
    p = some.data_ptr()
    assert lib.bf_embed_grad(p, 1, 0, p, 8, 3000, 1 << 26, 1, 1.0, 0, 0, p, p, None) == 3   # two values a workgroup
    assert lib.bf_embed_grad(p, 1, 0, p, 8, 5, (1 << 30) - 1, 1, 1.0, 0, 0, p, p, None) == 3
    assert lib.bf_embed_grad(p, 8, 0, p, 8, 1 << 29, 9, 8, 1.0, 0, 0, p, p, None) == 3      # the pieces' sums joined
    rows = (1 << 24) - 1
    assert lib.bf_policy_loss(p, 0, 1, rows, 700, 0, 700, p, 8, p, None, p, 0, 0, None, 0.2, 0.2, 0.0, 1.0, 0, 1.0, p, p,
                              p, p, None) == 3
    assert lib.bf_preference_loss(p, 0, rows, 700, 700, p, 8, p, p, 1, 0.1, 0.0, 1.0, p, p, p, p, p, None) == 3
    assert lib.bf_preference_loss(p, 0, 5, 700, 700, p, 8, p, p, 1 << 24, 0.1, 0.0, 1.0, p, p, p, p, p, None) == 3
    assert lib.bf_policy_loss_workspace(1, rows, 700, 0) == 0 and lib.bf_preference_loss_workspace(rows, 700, 1, 0) == 0
    weights, at = list(torch.zeros(120, 64)), [1 << 60, 2 << 60]
    assert adamw(lib, weights, weights, [64] * 119 + [1 << 34], at) == 3   # in the second launch
    assert adamw(lib, weights, weights, [64] * 119 + [1 << 35], at, m_scale=p, v_scale=p) == 3


def test_workspaces_hold_what_their_kernels_write(lib):
    # a first place per value and the end, a place per token; per eight tokens an owner and two rows of sums
    for count, vocab, dim in ((2049, 1, 1), (5000, 10, 4), (16_384, 32_000, 4096), (20_001, 70_001, 129)):
        pieces = -(-count // 8)
        assert lib.bf_embed_grad_workspace(count, vocab, dim) >= vocab + 1 + count + pieces * (1 + 2 * dim)
    # 64 shares of the counts, live rows per sequence; four sums per workgroup (2048 at most for short rows, 4096 for
    # held ones); a largest logit and a sum per part of a row
    for B, T, V, elem, sums, parts in ((64, 16, 5, 0, 0, 0), (5000, 2, 100, 1, 4 * 2048, 0), (8, 600, 700, 2, 4 * 4096, 0),
                                       (1, 4, 70_001, 0, 0, 2 * 4 * 35), (3, 800, 140_000, 1, 0, 2 * 2400)):
        assert lib.bf_policy_loss_workspace(B, T, V, elem) >= 64 + B + sums + parts
    # four coefficients per row, a loss per pair
    for N, V, pairs, elem, parts in ((45, 50_001, 2, 0, 45 * 25), (9001, 50_001, 16, 1, 9001), (2047, 4099, 3, 2, 2047 * 2)):
        assert lib.bf_preference_loss_workspace(N, V, pairs, elem) >= 4 * N + 2 * parts + pairs


@pytest.mark.parametrize("beta2,steps", [(0.99, 400), (0.999, 1000)])
def test_phases_keep_a_slow_average_at_every_step(beta2, steps):
    """sqrt(v) of steady gradients of 0.1 to 1 beside one of a burst of 100 at step 20: within two spacings, a quarter, of
    the exact one at every step and at both of the usual decays."""
    level = torch.rand(256, generator=torch.Generator().manual_seed(3), dtype=torch.float64) * 0.9 + 0.1
    held, v, burst = (torch.zeros(256, dtype=torch.float64) for _ in range(3))
    burst[::128] = 100.0
    for t in range(1, steps + 1):
        g = level + (burst if t == 20 else 0.0 * burst)
        v = beta2 * v + (1 - beta2) * g * g
        count, spacing, scale = ref.hold((beta2 * held * held + (1 - beta2) * g * g).sqrt(), ref.phases(256, t), True)
        held = count.floor() * spacing * scale.repeat_interleave(128)
        ratio = (held / v.sqrt())[burst == 0]
        assert 0.75 < float(ratio.min()) and float(ratio.max()) < 1.25, t


def test_adamw_of_empty_weights_has_nothing_to_do(lib):
    """Weights without an element, alone, have moments without an address."""
    assert adamw(lib, [None, None], [None, None], [0, 0], [None, None]) == 0
    assert adamw(lib, [None], [None], [0], [None, None], m_scale=8, v_scale=8) == 0
