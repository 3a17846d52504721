"""Buffers of the 4-bit cache's operators that share memory: refused before anything is launched, whichever argument it is that an
output or the workspace lies over. Buffers that only lie side by side are taken."""
import pytest
import torch

from gpu_common import DEV, assert_bit_equal, device_status
from oracle import kv4_ref as ref

pytestmark = pytest.mark.gpu

TOKENS, DIM = 4, 64


def arena(*sizes):
    """One buffer cut into neighbouring pieces of these bytes (multiples of 16), and the buffer."""
    whole = torch.zeros(sum(sizes), dtype=torch.uint8, device=DEV)
    pieces, at = [], 0
    for n in sizes:
        pieces.append(whole[at:at + n])
        at += n
    return pieces, whole


def heads(piece, count):
    return piece.view(torch.bfloat16).view(TOKENS, count, DIM)


def refused(match, call, *args):
    with pytest.raises(RuntimeError, match=match):
        call(*args)


def last_row_over(piece, whole, count):
    """A heads tensor whose last row ends 16 bytes inside `piece`'s first bytes."""
    offset = piece.data_ptr() - whole.data_ptr() + 16 - TOKENS * count * DIM * 2
    return heads(whole[offset:offset + TOKENS * count * DIM * 2], count)


def test_rotation_inputs(ops):
    size = TOKENS * 2 * DIM * 2
    (front, table, positions, axis_of, slots), whole = arena(4 * size, 8 * DIM * 4, 2 * TOKENS * 8, 128, 32)
    q, k = torch.zeros(TOKENS, 2, DIM, dtype=torch.bfloat16, device=DEV), torch.zeros(TOKENS, 2, DIM, dtype=torch.bfloat16, device=DEV)
    cos_sin, places = table.view(torch.float32).view(8, DIM), positions.view(torch.long).view(2, TOKENS)
    axes, at = axis_of.view(torch.int32)[:DIM // 2], slots.view(torch.long)
    cache = torch.zeros(1, 2, 2, ref.block_bytes(16, DIM), dtype=torch.uint8, device=DEV)
    turn = (cos_sin, places, axes)
    text = "overlap cos_sin, positions"
    for piece in (table, positions, axis_of):
        over = last_row_over(piece, whole, 2)
        refused(text, ops.qk_norm_rope, q, k, None, None, *turn, over, k)
        refused(text, ops.qk_norm_rope, q, k, None, None, *turn, q, over)
        refused(text, ops.kv4_append, q, k, k, *turn, at, over, cache)
    refused("axis_of or slots", ops.kv4_append, q, k, k, *turn, at, last_row_over(slots, whole, 2), cache)
    # a cache that reaches into them
    bytes_of = cache.numel()
    space = torch.zeros(bytes_of + 4096, dtype=torch.uint8, device=DEV)
    inside = space[bytes_of - 16:]
    wide = space[:bytes_of].view(cache.shape)
    refused("axis_of or slots", ops.kv4_append, None, k, k, None, None, None, inside[:8 * TOKENS].view(torch.long), None, wide)
    refused("axis_of or slots", ops.kv4_append, None, k, k, inside[:8 * DIM * 4].view(torch.float32).view(8, DIM), places[0], None, at, None, wide)
    refused("axis_of or slots", ops.kv4_append, None, k, k, cos_sin, inside[:8 * TOKENS].view(torch.long), None, at, None, wide)
    refused("axis_of or slots", ops.kv4_append, None, k, k, cos_sin, places, inside[:2 * DIM].view(torch.int32), at, None, wide)
    # neighbours
    fresh = heads(front[-size:], 2)
    ops.qk_norm_rope(q, k, None, None, *turn, fresh, torch.empty_like(k))
    ops.kv4_append(q, k, k, *turn, at, fresh, cache)
    behind = space[bytes_of:bytes_of + 8 * TOKENS].view(torch.long)
    ops.kv4_append(None, k, k, None, None, None, behind, None, wide)
    assert device_status(ops) == 0


def test_attention_workspace(ops):
    need = ops.kv4_workspace_bytes()
    block = ref.block_bytes(16, DIM)
    space = torch.zeros(need + (1 << 16), dtype=torch.uint8, device=DEV)
    workspace, tail, behind = space[:need], space[need - 16:], space[need:]
    q = torch.randn(1, 2, DIM, device=DEV).bfloat16()
    out, want = torch.empty_like(q), torch.empty_like(q)
    cache = torch.randint(0, 256, (2, 2, 2, block), dtype=torch.uint8, device=DEV)
    ref.rows(cache, DIM)[1][..., 0] = 0.5
    ref.rows(cache, DIM)[1][..., 1] = 8
    table, starts, lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([[1, 0]], [0, 1], [20]))

    def on(place, t):
        there = place[:t.numel() * t.element_size()].view(t.dtype).view(t.shape)
        return there

    good = dict(cache=cache, table=table, starts=starts, lens=lens)
    for name, t in good.items():
        for place in (workspace, tail):
            args = {**good, name: on(place, t)}
            refused("must not overlap", ops.kv4_attention, q, args["cache"], args["table"], args["starts"], args["lens"], workspace, out, 0.1)
    ops.kv4_attention(q, cache, table, starts, lens, workspace, want, 0.1)
    at = 0
    for name, t in list(good.items()):                                  # side by side, right behind the workspace
        good[name] = on(behind[at:], t)
        good[name].copy_(t)
        at += -(-t.numel() * t.element_size() // 16) * 16
    ops.kv4_attention(q, good["cache"], good["table"], good["starts"], good["lens"], workspace, out, 0.1)
    assert_bit_equal(out, want, "neighbouring buffers")
    assert device_status(ops) == 0
