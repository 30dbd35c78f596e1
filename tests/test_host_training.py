"""Host side of the training operators: the C entry points refuse what they cannot take before
any launch, and the rounding of 8-bit moments (as the oracle states it) keeps what it should.
No device call is made."""

import pytest
import torch

from boundflow_amd import _lib, training
from boundflow_amd._lib import HipError
from oracle import training_ref as ref


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run python -m boundflow_amd.build)")
    return _lib.load()


def test_cpu_tensors_are_refused():
    with pytest.raises(HipError, match="device tensor"):
        training.embed_tokens(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(HipError, match="device tensor"):
        training.adamw_moments([torch.zeros(3)])


def test_entry_points_refuse_bad_arguments(lib):
    some = torch.zeros(64)
    p = some.data_ptr()
    assert lib.bf_embed_rows(p, 4, 4, p, 2, 1, 4, 1.0, 0, p, None) == 1 and b"token bytes 2" in lib.bf_last_error()
    assert lib.bf_embed_rows(p, 4, 4, p, 4, 1, 4, 1.0, 3, p, None) == 1
    assert lib.bf_embed_rows(p, 3, 4, p, 4, 1, 4, 1.0, 0, p, None) == 1          # a stride below the width
    assert lib.bf_embed_rows(p, 4, 4, None, 4, 1, 4, 1.0, 0, p, None) == 1
    assert lib.bf_embed_rows(p, 4, 1 << 31, p, 4, 1, 4, 1.0, 0, p, None) == 3
    assert lib.bf_embed_rows(None, 4, 4, None, 4, 0, 4, 1.0, 0, None, None) == 0  # nothing to do
    assert lib.bf_embed_grad(p, 4, 1, p, 4, 1, 4, 4, 1.0, 2, 0, p, p, None) == 1  # bf16 rows, fp16 sums
    assert lib.bf_embed_grad(p, 4, 1, p, 4, 1, 4, 4, 1.0, 1, 1, p, p, None) == 1  # added to bf16
    assert lib.bf_embed_grad(p, 4, 0, p, 4, 1 << 30, 4, 4, 1.0, 0, 0, p, p, None) == 3
    policy = lambda **k: lib.bf_policy_loss(*{**dict(  # noqa: E731
        logits=p, elem=0, B=1, T=2, V=4, ld_b=8, ld_t=4, tokens=p, token_bytes=8, old=p, ref=None, adv=p, adv_b=0,
        adv_t=0, mask=None, low=0.2, high=0.2, kl=0.0, temperature=1.0, by=0, scale=1.0, logp=p, stats=p, grad=p, space=p,
        stream=None), **k}.values())
    for bad in (dict(elem=5), dict(V=0), dict(temperature=0.0), dict(low=-1.0), dict(stats=None), dict(old=None),
                dict(token_bytes=1), dict(ld_t=-1)):
        assert policy(**bad) == 1, bad
    assert policy(V=1 << 30) == 3 and policy(T=1 << 24) == 3
    pref = lambda **k: lib.bf_preference_loss(*{**dict(  # noqa: E731
        logits=p, elem=0, N=2, V=4, ld=4, tokens=p, token_bytes=8, ref=p, offsets=p, pairs=1, beta=0.1, smoothing=0.0,
        scale=1.0, logp=p, rewards=p, loss=p, grad=p, space=p, stream=None), **k}.values())
    for bad in (dict(elem=-1), dict(smoothing=2.0), dict(loss=None), dict(offsets=None), dict(ref=None)):
        assert pref(**bad) == 1, bad
    assert pref(N=1 << 24) == 3
    ptrs, sizes = _lib.ptr_array([some]), _lib.i64_array([64])
    adamw = lambda **k: lib.bf_adamw_multi(*{**dict(  # noqa: E731
        count=1, p=ptrs, g=ptrs, n=sizes, p_elem=0, g_elem=0, m=p, v=p, m_scale=None, v_scale=None, master=None, lr=0.1,
        b1=0.9, b2=0.9, eps=1e-8, wd=0.0, step=1, scale=1.0, scale_dev=None, stream=None), **k}.values())
    for bad in (dict(count=-1), dict(step=0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(m_scale=p), dict(m=None),
                dict(g_elem=3), dict(n=_lib.i64_array([-1])), dict(g=_lib.ptr_array([None]))):
        assert adamw(**bad) == 1, bad
    assert adamw(count=0) == 0


def test_workspaces_grow_with_what_they_hold(lib):
    assert lib.bf_embed_grad_workspace(100, 10, 4) == 0      # few tokens: sorted and summed in one launch, in LDS
    assert lib.bf_embed_grad_workspace(5000, 10, 4) >= 11 + 5000 + 2 * (5000 // 64) * 4
    assert lib.bf_policy_loss_workspace(2, 3, 100, 0) >= 6 * 6 + 2
    assert lib.bf_policy_loss_workspace(2, 3, 100, 7) == 0
    assert lib.bf_preference_loss_workspace(5, 100, 2, 1) >= 5 * 6 + 2


def test_moment_offsets():
    assert training.moment_offsets([1, 128, 129, 0, 5]) == [0, 128, 256, 512, 512, 640]
    assert training.moment_offsets([]) == [0]


def test_phases_are_even_over_steps_and_elements():
    for series in (torch.stack([ref.phases(1, t)[0] for t in range(1, 257)]), ref.phases(256, 7)):
        gaps = torch.diff(torch.sort(series)[0])
        # the three-distance theorem: no gap of n multiples of such a fraction is much above 1 / n
        assert float(gaps.max()) < 3.0 / 256


def test_rounding_by_phase_follows_where_nearest_stays():
    """sqrt(v) at beta2 = 0.99 of steady gradients, one of a block with a burst of 100 at step 20.  The block's scale falls
    with the burst from then on, and the others have to rise against it by less than half a spacing a step: rounded
    with phases they are within two spacings (a quarter) of the exact ones after 400 steps, rounded to the nearest number
    they fell with the scale to less than half."""
    held = {"phase": torch.zeros(256, dtype=torch.float64), "nearest": torch.zeros(256, dtype=torch.float64)}
    v, burst = torch.zeros(256, dtype=torch.float64), torch.zeros(256, dtype=torch.float64)
    burst[::128] = 100.0
    for t in range(1, 401):
        g = 1.0 + (burst if t == 20 else 0.0 * burst)
        v = 0.99 * v + 0.01 * g * g
        for name, x in held.items():
            phase = ref.phases(256, t) if name == "phase" else torch.full((256,), 0.5, dtype=torch.float64)
            count, spacing, scale = ref.hold((0.99 * x * x + 0.01 * g * g).sqrt(), phase, True)
            x.copy_(count.floor() * spacing * scale.repeat_interleave(128))
    ratio = {name: (x / v.sqrt())[burst == 0] for name, x in held.items()}
    assert float(ratio["phase"].min()) > 0.75 and float(ratio["phase"].max()) < 1.25
    assert float(ratio["nearest"].max()) < 0.5
