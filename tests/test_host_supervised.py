"""Host side of the operators of a supervised step: what the C entry points refuse before any launch, what their
workspaces hold, and the generator of the dropout masks as the oracle states it.  No device call is made."""

import pytest
import torch

from boundflow_amd import _lib, training
from boundflow_amd._lib import HipError
from oracle import training_ref as ref
from tests.test_host_training_memory import default_type, fp32, recorded  # noqa: F401


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run python -m boundflow_amd.build)")
    return _lib.load()


def test_cpu_tensors_are_refused():
    with pytest.raises(HipError, match="device tensor"):
        training.vocabulary_loss(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(HipError, match="device tensor"):
        training.dropout(torch.zeros(3), 0.5, seed=1)


def test_philox_known_answers():
    """The published test vectors of Philox 4x32 of ten rounds: counters and keys of zeros, of ones and of pi's digits."""
    def words(counter, key):
        u = ref.philox(counter[0] | counter[1] << 32, counter[2] | counter[3] << 32, key[0] | key[1] << 32)
        return [u[2 * k] | u[2 * k + 1] << 16 for k in range(4)]

    ones = 0xFFFFFFFF
    assert words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([ones] * 4, [ones] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert words([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_entry_points_refuse_bad_arguments(lib):
    some = torch.zeros(64)
    p = some.data_ptr()
    assert p % 16 == 0
    loss = lambda **k: lib.bf_vocab_loss(*{**dict(  # noqa: E731
        hidden=p, elem=0, B=1, T=2, D=4, ld_b=8, ld_t=4, weight=p, V=3, ld_w=4, bias=p, tokens=p, token_bytes=8, mask=None,
        temperature=1.0, scale=1.0, logp=p, loss=p, dh=p, dw=p, dw_elem=0, db=p, space=p, room=1 << 30, stream=None), **k}.values())
    for bad in (dict(elem=5), dict(V=0), dict(D=0), dict(temperature=0.0), dict(temperature=float("nan")), dict(loss=None),
                dict(token_bytes=1), dict(ld_t=-1), dict(ld_w=3), dict(weight=None), dict(hidden=None), dict(tokens=None),
                dict(logp=None), dict(space=None), dict(space=p + 4), dict(dw=None), dict(dh=None), dict(db=None),
                dict(bias=None), dict(dw_elem=1), dict(B=-1), dict(room=-1)):
        assert loss(**bad) == 1, bad
    for far in (dict(T=1 << 24), dict(B=1 << 40, T=1 << 40), dict(V=1 << 31), dict(ld_w=1 << 21),
                dict(D=1 << 21, ld_w=1 << 21), dict(T=(1 << 23) - 1, V=1 << 29), dict(T=(1 << 23) - 1, V=1 << 28, room=1 << 60)):
        assert loss(**far) == 3, far
    drop = lambda **k: lib.bf_dropout(*{**dict(  # noqa: E731
        x=p, ld=4, residual=None, r_ld=0, elem=0, rows=2, dim=4, p=0.5, seed=1, counter=0, counter_dev=None, out=p,
        stream=None), **k}.values())
    for bad in (dict(elem=3), dict(p=1.5), dict(p=float("nan")), dict(x=None), dict(out=None), dict(rows=-1), dict(ld=3),
                dict(residual=p, r_ld=3)):
        assert drop(**bad) == 1, bad
    assert drop(rows=0) == 0 and drop(dim=0, ld=0) == 0
    assert drop(rows=1 << 41, dim=8, ld=8) == 3


def test_workspaces_hold_what_their_kernels_write(lib):
    size = lib.bf_vocab_loss_workspace
    for N, D, V, elem in ((1, 1, 1, 0), (8, 2048, 32000, 1), (1003, 1025, 50001, 2), (2048, 1024, 32000, 0),
                          (8184, 4096, 128000, 1)):
        some = 1 << 20        # an address that can be read as it lies
        alone, grad = size(N, D, V, elem, some, D, 0, 0, 256 << 20), size(N, D, V, elem, some, D, 1, 0, 256 << 20)
        assert 0 < alone < grad
        # a token, a place and statistics per row and tile of the vocabulary; the packed rows
        parts = 3 if elem == 0 else 1
        assert 4 * alone >= 8 * N + 2 * parts * N * D
        # G stays within the room (the logits would be 4 N V), the sums of the hidden rows' gradient within theirs
        assert 4 * (grad - alone) <= (256 << 20) + max(128 << 20, 4 * (N + 64) * (D + 64)) + 4096
        # no room: a piece of 256 tokens
        assert 4 * size(N, D, V, elem, some, D, 1, 0, 0) < 4 * alone + 600 * parts * (N + D + 128) + \
            max(128 << 20, 4 * (N + 64) * (D + 64)) + 4096
    room = 1 << 30
    assert size(0, 4, 4, 0, 0, 4, 1, 1, room) == 0 and size(4, 4, 4, 7, 0, 4, 1, 1, room) == 0
    assert size(1 << 24, 4, 4, 0, 0, 4, 1, 1, room) == 0 and size(4, 4, 4, 0, 0, 4, 1, 1, -1) == 0
    # a weight that has to be packed takes more
    assert size(100, 64, 1000, 1, 1 << 20, 64, 0, 0, room) < size(100, 64, 1000, 1, (1 << 20) + 2, 64, 0, 0, room)


def test_rows_of_the_softmax_stay_within_32_bit_offsets(lib):
    """The products address a tile of up to 256 rows of G by 32 bits of bytes, however much room there is: 2^23 tokens."""
    for N, parts in ((64, 2), (256, 1)):
        V, D = 1 << 27, 8
        stats = 8 * (V // 128) * N + (1 << 24)      # per row and tile; dx's sums of 128 MB, dw's none
        got = 4 * lib.bf_vocab_loss_workspace(N, D, V, 1, 1 << 20, D, 1, 0, 1 << 60)
        assert 2 * parts * N * (1 << 23) <= got <= 2 * parts * N * (1 << 23) + stats + (128 << 20)


def test_an_empty_batch_over_a_vocabulary_past_a_launch_is_refused(lib):
    p = torch.zeros(64).data_ptr()
    args = lambda V, D: (None, 1, 0, 2, D, 0, 0, p, V, D, None, None, 8, None, 1.0, 1.0, None, p, None, p, 1, None, None,  # noqa: E731
                         1 << 30, None)
    assert lib.bf_vocab_loss(*args(1 << 30, 1 << 20)) == 3
    assert lib.bf_vocab_loss(*args(1 << 25, 1 << 11)) == 3


def test_requires_grad_is_refused_before_the_device_is_asked():
    x = torch.zeros(3, requires_grad=True)
    with pytest.raises(HipError, match="dropout_grad"):
        training.dropout(x, 0.5, seed=1)


def test_buffers_follow_the_inputs_whatever_the_default_type(recorded, default_type):  # noqa: F811
    made, calls = recorded
    tokens = torch.ones(300, dtype=torch.int64)
    for dtype in (torch.float32, torch.bfloat16):
        r = training.vocabulary_loss(torch.ones(300, 24, dtype=dtype), torch.ones(70, 24, dtype=dtype), tokens,
                                     bias=torch.ones(70, dtype=dtype))
        assert r.loss.dtype == r.logp.dtype == torch.float32
        assert r.grad_hidden.dtype == r.grad_weight.dtype == r.grad_bias.dtype == dtype
        r = training.vocabulary_loss(torch.ones(300, 24, dtype=dtype), torch.ones(70, 24, dtype=dtype), tokens,
                                     weight_grad_dtype=torch.float32)
        assert r.grad_weight.dtype == torch.float32 and r.grad_bias is None
        assert training.dropout(torch.ones(5, 3, dtype=dtype), 0.5, seed=1).dtype == dtype
    assert [name for name, _ in calls] == ["bf_vocab_loss", "bf_vocab_loss", "bf_dropout"] * 2
    assert {t.dtype for t in made} == {torch.float32, torch.bfloat16}


@pytest.mark.parametrize("rows,V", [(4, 5), (300, 700), (2000, 40)])
def test_results_do_not_keep_the_workspace(recorded, rows, V):  # noqa: F811
    _made, calls = recorded
    r = training.vocabulary_loss(fp32(rows, 24), fp32(V, 24), torch.zeros(rows, dtype=torch.int64))
    held = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in r if t is not None}
    assert sum(held.values()) <= 4 * (1 + rows + 24 * (rows + V)) + 64
    need = _lib.load().bf_vocab_loss_workspace(rows, 24, V, 0, calls[0][1][7], 24, 1, 0, 2 << 30)
    space = calls[0][1][-3]
    base = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in recorded[0]}
    assert base[space] >= 4 * need


def test_seeds_and_counters_reach_the_library_whole(recorded):  # noqa: F811
    _made, calls = recorded
    training.dropout(fp32(6), 0.25, seed=(1 << 64) - 1, counter=(1 << 63) - 1)
    training.dropout(fp32(2, 3, 4)[:, 1:], 0.25, seed=5, counter=torch.tensor(9), residual=fp32(2, 2, 4))
    (_, a), (_, b) = calls
    assert a[8] == -1 and a[9] == (1 << 63) - 1 and a[10] is None and a[5:7] == (1, 6)
    assert b[8] == 5 and b[9] == 0 and b[10] is not None and b[5:7] == (4, 4)


def test_a_seed_or_counter_that_is_no_integer_is_refused(recorded):  # noqa: F811
    _made, calls = recorded
    for kw in ({"seed": 1, "counter": 1.5}, {"seed": 1.0}, {"seed": 1, "counter": 2.0}):
        with pytest.raises(TypeError):
            training.dropout(fp32(6), 0.25, **kw)
    assert not calls


@pytest.mark.parametrize("value", [float("inf"), 1e39, 2.0 ** 121, 2.0 ** -121, 1e-39, 5e-324])
def test_temperatures_that_fp32_does_not_hold_are_refused(lib, recorded, value):  # noqa: F811
    """Their inverse would be 0 or infinite in fp32, and that times a padded entry's -inf is no number."""
    _made, calls = recorded
    p = torch.zeros(64).data_ptr()
    assert lib.bf_vocab_loss(p, 0, 1, 2, 4, 8, 4, p, 3, 4, p, p, 8, None, value, 1.0, p, p, p, p, 0, p, p, 1 << 30, None) == 1
    with pytest.raises(ValueError, match="temperature"):
        training.vocabulary_loss(fp32(2, 4), fp32(3, 4), torch.zeros(2, dtype=torch.int64), temperature=value)
    assert not calls


@pytest.mark.parametrize("with_grad", [True, False])
@pytest.mark.parametrize("name", ["hidden", "weight", "bias"])
def test_tensors_that_require_grad_are_refused_where_their_gradient_would_be_lost(recorded, name, with_grad):  # noqa: F811
    """The loss has no graph: a backward() of a sum that it is part of would leave the head untrained without an error."""
    _made, calls = recorded
    args = {"hidden": fp32(2, 4), "weight": fp32(3, 4), "bias": fp32(3)}
    args[name].requires_grad_(True)
    kw = {"tokens": torch.zeros(2, dtype=torch.int64), "with_grad": with_grad}
    with pytest.raises(HipError, match=f"{name}.detach()"):
        training.vocabulary_loss(**args, **kw)
    assert not calls
    with torch.no_grad():
        assert not training.vocabulary_loss(**args, **kw).loss.requires_grad
    training.vocabulary_loss(**{**args, name: args[name].detach()}, **kw)
    assert len(calls) == 2


def test_room_reaches_the_library_whole(recorded):  # noqa: F811
    """A number past 63 bits would arrive cut to 64: 2^64 + 256 as 256, 2^63 as a negative one."""
    _made, calls = recorded
    args = (fp32(2, 4), fp32(3, 4), torch.zeros(2, dtype=torch.int64))
    for room in ((1 << 64) + 256, 1 << 63, -1):
        with pytest.raises(ValueError, match="room must be"):
            training.vocabulary_loss(*args, room=room)
    with pytest.raises(TypeError):
        training.vocabulary_loss(*args, room=2e9)
    assert not calls
    training.vocabulary_loss(*args, room=(1 << 63) - 1)
    assert calls[0][1][-2] == (1 << 63) - 1


def test_what_fits_a_launch_is_counted_in_the_tiles_that_are_made(lib):
    """Beside few rows the weight's gradient runs in tiles of 128 x 128: of 2^20 columns and 140000 tokens 2^13 x 1094 of 256
    threads, of which 2^24 are a launch of 2^32.  Counted in tiles of half the size they would be refused."""
    size = lib.bf_vocab_loss_workspace
    assert size(8, 1 << 20, 140_000, 1, 1 << 20, 1 << 20, 1, 0, 1 << 40) > 0
    assert size(8, 1 << 20, 270_000, 1, 1 << 20, 1 << 20, 1, 0, 1 << 40) == 0
