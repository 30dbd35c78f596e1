"""Sizes of the vocabulary loss that between them take every way through its kernels: which tiles, how often the logits are
formed, how the softmax's gradient is held.  What each takes is asked of the library (``plan``), so that a rule that moves
does not leave a way untested."""

import ctypes

import torch

from boundflow_amd import _lib

TILES = ("large", "mid", "deep", "slim", "thin", "registers")
ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ROOM = 2 << 30

# rows, width, vocabulary, gap between the weight's rows, bias, room; the tiles of the logits and of the gradients, and whether
# the logits are formed again, for 16-bit types and for fp32 (None: not run)
CASES = [
    ((600, 200, 10_001, 0, True, ROOM), ("mid", "deep", False), None),
    ((600, 200, 10_001, 0, True, 1 << 20), ("mid", "deep", True), None),
    ((1500, 328, 9001, 0, False, ROOM), ("large", "deep", False), ("large", "deep", False)),
    ((1500, 329, 9001, 0, True, ROOM), ("large", "deep", False), ("large", "deep", False)),
    ((1500, 328, 9001, 8, True, 8 << 20), ("large", "deep", True), ("large", "deep", True)),
    ((1500, 329, 9001, 3, False, 8 << 20), ("large", "deep", True), ("large", "deep", True)),
    ((1500, 520, 9001, 0, True, ROOM), ("large", "mid", False), ("large", "large", False)),
    ((1500, 1288, 9001, 0, True, ROOM), ("large", "large", False), None),
    ((1500, 1288, 9001, 0, False, 10 << 20), ("large", "mid", True), None),
    ((200, 200, 9000, 0, True, 1 << 20), ("deep", "deep", True), ("deep", "deep", True)),
    ((100, 520, 700, 0, True, 1 << 16), ("deep", "deep", True), ("registers", "registers", True)),
    ((300, 520, 700, 0, False, ROOM), ("deep", "deep", False), ("deep", "deep", False)),
    ((40, 136, 33_001, 0, True, ROOM), ("slim", "slim", False), ("registers", "registers", False)),
    ((40, 136, 33_001, 0, True, 1 << 20), ("slim", "thin", True), ("registers", "registers", True)),
    ((40, 136, 9001, 0, False, ROOM), ("thin", "slim", False), ("registers", "registers", False)),
    ((40, 136, 9001, 1, True, 1 << 16), ("thin", "thin", True), ("registers", "registers", True)),
    ((7, 520, 700, 0, False, ROOM), ("thin", "thin", False), ("registers", "registers", False)),
    ((40, 137, 9001, 0, True, ROOM), ("thin", "slim", False), ("registers", "registers", False)),     # scored: through registers
    ((7, 521, 700, 0, True, ROOM), ("thin", "thin", False), ("registers", "registers", False)),
]

# (case, type, what it takes)
RUNS = [(case, dtype, wide if dtype == torch.float32 else narrow) for case, narrow, wide in CASES for dtype in ELEM
        if (wide if dtype == torch.float32 else narrow) is not None]


def plan(N, D, V, gap, bias, room, dtype, with_grad=True, address=1 << 20):
    """(pieces, tile of the logits, tile of the gradients, parts of G, cuts of joined logits or 0, columns beside the softmax)"""
    out = (ctypes.c_int64 * 6)()
    status = _lib.load().bf_vocab_loss_plan(N, D, V, ELEM[dtype], address, D + gap, with_grad, bias, room,
                                            ctypes.addressof(out))
    assert status == 0, status
    return (out[0], TILES[out[1]], TILES[out[2]] if out[2] >= 0 else None, *out[3:])


def kernels(case, dtype, with_grad):
    """What a call launches of the products: (what, how a tile of logits ends, parts of G, tile)."""
    pieces, logits, grads, parts, summed, _ = plan(*case, dtype, with_grad)
    wide = dtype == torch.float32
    ways = {("logits", 2, parts if wide else 1, logits) if summed else ("logits", 0, parts, logits)}
    if with_grad:
        ways.add(("grads", None, parts, grads))
        if pieces > 1:
            ways.add(("logits", 1, parts, logits))
    return ways
