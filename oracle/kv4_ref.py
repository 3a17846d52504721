"""CPU restatements of the operators around the 4-bit key/value cache (test infrastructure).

The norm, the rotation and the attention are computed in 64 bits from their formulas; the encoding is computed with the
IEEE FP32 operations its definition names, so its bytes can be compared for equality."""
from __future__ import annotations

import torch


def block_bytes(page: int, dim: int) -> int:
    return page * (dim // 2 + 4)


def angles(cos_sin, positions, axis_of, tokens):
    """FP64 cosine and sine [tokens, rotary / 2] of each pair."""
    half = cos_sin.shape[1] // 2
    positions = positions.reshape(-1, tokens)
    axis = torch.zeros(half, dtype=torch.long) if axis_of is None else axis_of.long()
    place = positions[axis].T                              # [tokens, half]
    column = torch.arange(half)
    return cos_sin.double()[place, column], cos_sin.double()[place, column + half]


def rotate(x, cosine, sine, adjacent):
    """x [tokens, heads, dim]; computed in x's own type, one IEEE operation at a time."""
    cosine, sine = cosine.to(x.dtype)[:, None], sine.to(x.dtype)[:, None]
    r = 2 * cosine.shape[-1]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if adjacent else (slice(0, r // 2), slice(r // 2, r))
    y = x.clone()
    y[..., first] = x[..., first] * cosine - x[..., second] * sine
    y[..., second] = x[..., second] * cosine + x[..., first] * sine
    return y


def norm(x, weight, eps, offset):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.double() + offset)


def encode(x):
    """FP32 [..., dim] -> (codes UINT8 [..., dim], BF16 scale [...], BF16 zero point [...])."""
    assert x.dtype == torch.float32
    x = torch.nan_to_num(x, nan=0.0, posinf=8.5e37, neginf=-8.5e37).clamp(-8.5e37, 8.5e37)
    low, high = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    step = (high - low) * torch.tensor(1.0 / 15.0)         # the FP32 number next to 1 / 15
    scale = torch.maximum(step.bfloat16(), torch.tensor(1e-20).bfloat16())
    s = scale.float()
    zero = torch.round(-low / s).clamp(0, 15) + 0.0        # a whole number: never minus zero
    codes = (torch.round(x / s[..., None]) + zero[..., None]).clamp(0, 15)
    return codes.to(torch.uint8), scale, zero.bfloat16()


def rows(cache, dim):
    """The cache's bytes as (code rows [pages, 2, heads, page, dim / 2], pairs BF16 [pages, 2, heads, page, 2]), views."""
    page = cache.shape[-1] // (dim // 2 + 4)
    codes = cache[..., : page * dim // 2].unflatten(-1, (page, dim // 2))
    return codes, cache[..., page * dim // 2:].unflatten(-1, (page, 4)).view(torch.bfloat16)


def store(cache, slots, k, v):
    """FP32 k, v [tokens, heads, dim] into the cache rows of slots (negative and too large ones are left out)."""
    codes, pairs = rows(cache, k.shape[-1])
    page = codes.shape[3]
    for side, x in enumerate((k, v)):
        c, scale, zero = encode(x)
        packed = c[..., 0::2] | (c[..., 1::2] << 4)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < cache.shape[0] * page:
                codes[slot // page, side, :, slot % page] = packed[t]
                pairs[slot // page, side, :, slot % page, 0] = scale[t]
                pairs[slot // page, side, :, slot % page, 1] = zero[t]


def values(cache, dim):
    """FP64 [pages, 2, heads, page, dim]: what the cache holds."""
    codes, pairs = rows(cache, dim)
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).double()
    return pairs[..., :1].double() * (c - pairs[..., 1:].double())


def attention(q, cache, block_table, q_starts, kv_lens, scale):
    """(out FP64 [tokens, q_heads, dim], the bound's weights: sum of p * |v|, and the largest score a row could have,
    dim * 15 steps * max |q| * scale)."""
    tokens, q_heads, dim = q.shape
    held = values(cache, dim)
    _, pairs = rows(cache, dim)
    kv_heads, page = held.shape[2], held.shape[3]
    out = torch.zeros(tokens, q_heads, dim, dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros(tokens, q_heads, 1, dtype=torch.float64)
    for b in range(len(kv_lens)):
        start, end, keys = int(q_starts[b]), int(q_starts[b + 1]), int(kv_lens[b])
        keys = max(0, min(keys, block_table.shape[1] * page))
        ids = block_table[b, : -(-keys // page)].long()
        good = ((ids >= 0) & (ids < cache.shape[0])).repeat_interleave(page)[:keys]
        ids = ids.clamp(0, cache.shape[0] - 1)
        kv = held[ids].permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :keys]      # [2, heads, keys, dim]
        step = pairs[ids, 0, :, :, 0].double().permute(1, 0, 2).flatten(1)[:, :keys]
        for i in range(end - start):
            seen = torch.nonzero(good & (torch.arange(keys) <= keys - (end - start) + i)).flatten()
            if not len(seen):
                continue
            for h in range(q_heads):
                k, v = kv[0, h * kv_heads // q_heads, seen], kv[1, h * kv_heads // q_heads, seen]
                row = q[start + i, h].double()
                p = (k @ row * scale).softmax(0)
                out[start + i, h] = p @ v
                spread[start + i, h] = p @ v.abs()
                reach[start + i, h] = row.abs().max() * 15 * dim * step[h * kv_heads // q_heads, seen].max() * scale
    return out, spread, reach
