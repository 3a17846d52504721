"""What is measured of the operators around the 4-bit key/value cache: their cases, inputs and plain forms.

Four operators sit between the QKV projection and the output projection of a layer whose products run in INT8:

  norm    every query and key head RMS-normalised and rotated to its position, in one pass
  append  keys rotated on the way, keys and values encoded into a paged 4-bit cache (queries rotated beside them)
  read    rows of that cache back as the BF16 values they stand for
  attend  causal attention of single tokens and of prompts over that cache

``own`` False computes them with elementary torch operations in FP32, rounded once at the end; True calls
``consumer_int8.ops``.

The cache is UINT8 [pages, 2 (keys, values), heads, page * (dim / 2 + 4)]: for each page, side and head first ``page``
rows of dim / 2 bytes (byte j: component 2j in the low and 2j + 1 in the high four bits), then ``page`` pairs of BF16
numbers (scale, zero point); a code c stands for scale * (c - zero).
"""
import math
import random
import sys

import torch

own = False

DEVICE = "cuda"
WORKSPACE_BYTES = 64 << 20      # no call asks for more


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one generated token: the smallest call, latency counts (6 query heads to a key head, a quarter rotated)
        {"name": "norm one token", "op": "norm", "tokens": 1, "q_heads": 24, "kv_heads": 4, "dim": 256, "rotary": 64, "axes": 1, "adjacent": False},
        # a prompt's chunk with positions on three axes (time, height, width), an odd number of tokens
        {"name": "norm three axes", "op": "norm", "tokens": 4099, "q_heads": 16, "kv_heads": 16, "dim": 64, "rotary": 64, "axes": 3, "adjacent": False},
        # a long prompt's chunk, the ordinary head layout
        {"name": "norm prompt", "op": "norm", "tokens": 16384, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 1, "adjacent": True},
        # a batch of generated tokens into scattered pages, two rows of padding among them; what the cache holds is read back
        {"name": "append batch", "op": "append", "tokens": 16, "q_heads": 24, "kv_heads": 4, "dim": 256, "rotary": 64, "axes": 1, "adjacent": False, "page": 16, "padding": 2},
        # a prompt's chunk into the cache
        {"name": "append prompt", "op": "append", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 1, "adjacent": False, "page": 64, "padding": 0},
        # a short prefix handed to another consumer
        {"name": "read short", "op": "read", "tokens": 250, "kv_heads": 4, "dim": 256, "page": 16},
        # a long prefix
        {"name": "read long", "op": "read", "tokens": 65536, "kv_heads": 8, "dim": 128, "page": 64},
        # one user, one token, a short history: latency
        {"name": "attend one token", "op": "attend", "batch": 1, "q": 1, "kv": 1000, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "ragged": False},
        # a serving batch with histories of all lengths
        {"name": "attend batch", "op": "attend", "batch": 64, "q": 1, "kv": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "ragged": True},
        # few users with long histories: the work has to be split along them
        {"name": "attend long", "op": "attend", "batch": 4, "q": 1, "kv": 65536, "q_heads": 24, "kv_heads": 4, "dim": 256, "page": 64, "ragged": False},
        # prompts' chunks of different lengths behind cached prefixes, single tokens may be among them
        {"name": "attend chunks", "op": "attend", "batch": 5, "q": 1000, "kv": 9000, "q_heads": 24, "kv_heads": 4, "dim": 256, "page": 16, "ragged": True},
        # a whole prompt
        {"name": "attend prompt", "op": "attend", "batch": 1, "q": 8192, "kv": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "ragged": False},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "read", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    case = {"op": op}
    if op in ("norm", "append"):
        # as many tokens as keep the heads' values below the largest listed case's
        most = 16384 * 40 * 128 if op == "norm" else 8192 * 48 * 128
        heads = q_heads + (2 if op == "append" else 1) * kv_heads
        case["tokens"] = _spread(rng, 1, max(1, min(16384, most // (heads * dim))))
        case.update(q_heads=q_heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([r for r in (16, 32, 64, 128, 256) if r <= dim]),
                    axes=rng.choice([1, 1, 2, 3]), adjacent=rng.random() < 0.3)
        if op == "append":
            case.update(page=page, padding=rng.randint(0, min(5, case["tokens"] - 1)))
    elif op == "read":
        case.update(tokens=_spread(rng, 1, 65536 * 8 * 128 // (kv_heads * dim)), kv_heads=kv_heads, dim=dim, page=page)
    else:
        kind = rng.choice(["single", "single", "prompt"])
        if kind == "single":
            batch = _spread(rng, 1, 128)
            kv = _spread(rng, 1, max(1, min(65536, 64 * 8192 * 8 * 128 // (batch * kv_heads * dim))))
            case.update(batch=batch, q=1, kv=kv)
        else:
            batch = _spread(rng, 1, 8)
            # queries x keys x heads x batch at most a quarter of the largest listed case's
            most = 8192 * 8192 * 32 * 128 // 4 // (batch * q_heads * dim)
            q = _spread(rng, 2, min(4096, math.isqrt(most)))
            kv = _spread(rng, q, min(32768, most // q))
            case.update(batch=batch, q=q, kv=kv)
        case.update(q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, ragged=rng.random() < 0.7)
    return case


def _lengths(case):
    """New tokens and cached tokens (the new ones among them) of each sequence of an attend case."""
    if not case["ragged"]:
        return [case["q"]] * case["batch"], [case["kv"]] * case["batch"]
    rng = random.Random(1000003 * case["batch"] + 1009 * case["q"] + case["kv"])
    news = [case["q"]] + [rng.randint(1, case["q"]) for _ in range(case["batch"] - 1)]
    kvs = [case["kv"]] + [rng.randint(max(n, case["kv"] // 16, 1), case["kv"]) for n in news[1:]]
    return news, kvs


def work(case):
    dim = case["dim"]
    row = dim // 2 + 4
    if case["op"] == "norm":
        n, r = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * dim, case["rotary"]
        return {"bytes": 4 * n + case["tokens"] * (4 * r + 8 * case["axes"]) + 4 * dim, "flops": 10 * n}
    if case["op"] == "append":
        t, hq, hk, r = case["tokens"], case["q_heads"], case["kv_heads"], case["rotary"]
        kept = t - case["padding"]
        append = t * (4 * hq + 4 * hk) * dim + 2 * kept * hk * row + t * (4 * r + 8 * case["axes"] + 8)
        return {"bytes": append + 2 * kept * hk * row + 4 * t * hk * dim, "flops": t * (6 * hq + 16 * hk) * dim}
    if case["op"] == "read":
        n = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": n * (row + 2 * dim) + 8 * case["tokens"], "flops": 2 * n * dim}
    news, kvs = _lengths(case)
    pairs = sum(n * (kv - n) + n * (n + 1) // 2 for n, kv in zip(news, kvs))
    cache = 2 * sum(kvs) * case["kv_heads"] * row
    return {"bytes": cache + 4 * sum(news) * case["q_heads"] * dim + 4 * sum(-(-kv // case["page"]) for kv in kvs),
            "flops": 4 * pairs * case["q_heads"] * dim}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _table(rows, rotary):
    """FP32 [rows, rotary]: the cosines of rotary / 2 angles, then their sines."""
    rate = 10000.0 ** (-torch.arange(rotary // 2, device=DEVICE, dtype=torch.float64) / (rotary // 2))
    angle = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _heads(g, tokens, heads, dim):
    """Values as a projection gives them: a few components of every head larger than the others."""
    x = torch.randn(tokens, heads, dim, device=DEVICE, generator=g)
    gain = 1 + 3 * (torch.rand(heads, dim, device=DEVICE, generator=g) < 0.02)
    return x.mul_(gain).bfloat16()


def _encode(x):
    """FP32 [..., dim] -> codes [..., dim] as whole FP32 numbers, BF16 scale and zero point [...]."""
    low, high = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    scale = ((high - low) / 15).bfloat16().clamp(min=1e-20)
    s = scale.float()
    zero = torch.round(-low / s).clamp(0, 15)
    codes = (torch.round(x / s[..., None]) + zero[..., None]).clamp_(0, 15)
    return codes, scale, zero.bfloat16()


def _pack(codes, scale, zero):
    """[pages, 2, heads, page, dim] codes and [pages, 2, heads, page] scales and zero points -> the cache."""
    c = codes.to(torch.uint8)
    rows = (c[..., 0::2] | (c[..., 1::2] << 4)).flatten(-2)
    words = torch.stack([scale, zero], dim=-1).view(torch.uint8).flatten(-2)
    return torch.cat([rows, words], dim=-1)


def _filled_cache(g, pages, heads, page, dim):
    x = _heads(g, pages * 2, heads * page, dim).view(pages, 2, heads, page, dim)
    return _pack(*_encode(x.float()))


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    op, dim = case["op"], case["dim"]
    if op in ("norm", "append"):
        t, hq, hk, r, axes = case["tokens"], case["q_heads"], case["kv_heads"], case["rotary"], case["axes"]
        # queries, keys and values are slices of the projection's one output
        qkv = _heads(g, t, hq + 2 * hk, dim)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        s["cos_sin"] = _table(32768, r)
        start = torch.randint(0, 32768 - 16384, (axes, 1), device=DEVICE, generator=g)
        s["positions"] = (start + torch.arange(t, device=DEVICE)[None, :] // torch.tensor([1, 7, 3], device=DEVICE)[:axes, None]).contiguous()
        # the frequencies are dealt to the axes in turn
        s["axis_of"] = (torch.arange(r // 2, device=DEVICE) % axes).int() if axes > 1 else None
        s["q_out"] = torch.empty(t, hq, dim, device=DEVICE, dtype=torch.bfloat16)
    if op == "norm":
        s["q_weight"] = (1 + 0.2 * torch.randn(dim, device=DEVICE, generator=g)).bfloat16()
        s["k_weight"] = (1 + 0.2 * torch.randn(dim, device=DEVICE, generator=g)).bfloat16()
        s["eps"] = 1e-6
        s["k_out"] = torch.empty(t, hk, dim, device=DEVICE, dtype=torch.bfloat16)
    if op in ("append", "read"):
        page, hk = case["page"], case["kv_heads"]
        pages = -(-case["tokens"] // page) + 3
        order = torch.randperm(pages, device=DEVICE, generator=g)
        at = torch.arange(case["tokens"], device=DEVICE)
        s["slots"] = order[at // page] * page + at % page
        s["keys"] = torch.empty(case["tokens"], hk, dim, device=DEVICE, dtype=torch.bfloat16)
        s["values"] = torch.empty(case["tokens"], hk, dim, device=DEVICE, dtype=torch.bfloat16)
        if op == "append":
            s["slots"][case["tokens"] - case["padding"]:] = -1
            s["cache"] = torch.zeros(pages, 2, hk, page * (dim // 2 + 4), device=DEVICE, dtype=torch.uint8)
        else:
            s["cache"] = _filled_cache(g, pages, hk, page, dim)
    if op == "attend":
        page, hk, hq = case["page"], case["kv_heads"], case["q_heads"]
        news, kvs = _lengths(case)
        need = [-(-kv // page) for kv in kvs]
        pages = sum(need) + 2
        s["cache"] = _filled_cache(g, pages, hk, page, dim)
        order = torch.randperm(pages, device=DEVICE, generator=g)
        width = max(need)
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEVICE)
        column = torch.arange(width, device=DEVICE)
        used = column[None, :] < torch.tensor(need, device=DEVICE)[:, None]
        s["block_table"] = torch.where(used, order[(first[:, None] + column).clamp(max=pages - 1)], -1).int()
        s["q_starts"] = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], device=DEVICE, dtype=torch.int32)
        s["kv_lens"] = torch.tensor(kvs, device=DEVICE, dtype=torch.int32)
        s["queries"] = torch.randn(sum(news), hq, dim, device=DEVICE, generator=g).bfloat16()
        s["out"] = torch.empty_like(s["queries"])
        s["workspace"] = torch.zeros(WORKSPACE_BYTES, device=DEVICE, dtype=torch.uint8)
        s["most_new"], s["scale"] = max(news), dim ** -0.5
    return s


# ---------------------------------------------------------------- one pass
def _ops():
    at = __file__.rsplit("/", 2)[0] + "/consumer-int8-kernels_b200"
    if at not in sys.path:
        sys.path.insert(0, at)
    from consumer_int8 import ops
    return ops


def run(state):
    s = state
    op = s["op"]
    if own:
        ops = _ops()
        if op == "norm":
            ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"], s["axis_of"],
                             s["q_out"], s["k_out"], s["eps"], 0.0, s["adjacent"])
            return {"q": s["q_out"], "k": s["k_out"]}
        if op == "append":
            ops.kv4_append(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["axis_of"], s["slots"], s["q_out"],
                           s["cache"], s["adjacent"])
        if op in ("append", "read"):
            ops.kv4_read(s["cache"], s["slots"], s["keys"], s["values"])
            held = {"keys": s["keys"], "values": s["values"]}
            return {**held, "q": s["q_out"]} if op == "append" else held
        ops.kv4_attention(s["queries"], s["cache"], s["block_table"], s["q_starts"], s["kv_lens"], s["workspace"],
                          s["out"], s["scale"])
        return s["out"]
    if op == "norm":
        return {"q": _rotate(_norm(s["q"].float(), s["q_weight"], s["eps"]), s).bfloat16(),
                "k": _rotate(_norm(s["k"].float(), s["k_weight"], s["eps"]), s).bfloat16()}
    if op == "append":
        q = _rotate(s["q"].float(), s).bfloat16()
        _store(s["cache"], s["slots"], torch.stack([_rotate(s["k"].float(), s), s["v"].float()], dim=1))
        return {**_rows(s), "q": q}
    if op == "read":
        return _rows(s)
    return _attend(s)


def _norm(x, weight, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()


def _rotate(x, s):
    """x FP32 [tokens, heads, dim]: its first ``rotary`` components turned by the angles of each token's position."""
    r = s["rotary"]
    half = r // 2
    if s["axis_of"] is None:
        row = s["cos_sin"][s["positions"][0]]
        cos, sin = row[:, None, :half], row[:, None, half:]
    else:
        place = s["positions"][s["axis_of"].long()].T                      # [tokens, half]
        column = torch.arange(half, device=x.device)
        cos, sin = s["cos_sin"][place, column][:, None], s["cos_sin"][place, column + half][:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if s["adjacent"] else (x[..., :half], x[..., half:r])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], dim=-1).flatten(-2) if s["adjacent"] else torch.cat([u, w], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _split_cache(cache, dim):
    """The cache's bytes as code rows [pages, 2, heads, page, dim / 2] and BF16 pairs [pages, 2, heads, page, 2] (views)."""
    page = cache.shape[-1] // (dim // 2 + 4)
    codes = cache[..., : page * dim // 2].unflatten(-1, (page, dim // 2))
    words = cache[..., page * dim // 2:].unflatten(-1, (page, 4)).view(torch.bfloat16)
    return codes, words


def _store(cache, slots, x):
    """x FP32 [tokens, 2, heads, dim] into the cache rows of slots; rows whose slot is negative are left out."""
    codes, words = _split_cache(cache, x.shape[-1])
    page = codes.shape[3]
    c, scale, zero = _encode(x)
    c = c.to(torch.uint8)
    packed, pair = c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([scale, zero], dim=-1)
    kept = slots >= 0
    at = slots[kept]
    codes[at // page, :, :, at % page] = packed[kept]
    words[at // page, :, :, at % page] = pair[kept]


def _decode(codes, words):
    """Code bytes [..., dim / 2] and BF16 pairs [..., 2] -> the FP32 values [..., dim] they stand for."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float()
    return words[..., 0:1].float() * (c - words[..., 1:2].float())


def _rows(s):
    """The values that the cache holds at slots, zero where a slot is negative."""
    codes, words = _split_cache(s["cache"], s["dim"])
    page = codes.shape[3]
    at = s["slots"].clamp(min=0)
    x = _decode(codes[at // page, :, :, at % page], words[at // page, :, :, at % page])
    x = torch.where((s["slots"] >= 0)[:, None, None, None], x, 0.0).bfloat16()
    return {"keys": x[:, 0], "values": x[:, 1]}


def _attend(s):
    hk, dim, group, most = s["kv_heads"], s["dim"], s["q_heads"] // s["kv_heads"], s["most_new"]
    codes, words = _split_cache(s["cache"], dim)
    pages = s["block_table"].clamp(min=0).long()                           # [batch, width]
    batch = pages.shape[0]
    # [batch, width, 2, heads, page, dim] -> [2, batch, heads, keys, dim]
    kv = _decode(codes[pages], words[pages]).permute(2, 0, 3, 1, 4, 5).flatten(3, 4)
    keys = kv.shape[3]
    starts, ends = s["q_starts"][:-1].long(), s["q_starts"][1:].long()
    step = torch.arange(most, device=kv.device)
    at = starts[:, None] + step                                            # [batch, most]
    real = at < ends[:, None]
    q = s["queries"].float()[at.clamp(max=len(s["queries"]) - 1)]          # [batch, most, q_heads, dim]
    q = q.unflatten(2, (hk, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)   # [batch, heads, group * most, dim]
    score = (q @ kv[0].transpose(-1, -2)).mul_(s["scale"])
    last = s["kv_lens"].long()[:, None] - (ends - starts)[:, None] + step  # the last key that each query sees
    hidden = torch.arange(keys, device=kv.device) > last[..., None]        # [batch, most, keys]
    score.unflatten(2, (group, most)).masked_fill_(hidden[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    o = (score @ kv[1]) / total.clamp(min=1e-30)
    o = o.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [batch, most, q_heads, dim]
    out = torch.zeros(s["queries"].shape, device=o.device, dtype=torch.bfloat16)
    out[at[real]] = o[real].bfloat16()
    return out


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op, dim = case["op"], case["dim"]
    if op in ("norm", "append"):
        t, r = case["tokens"], case["rotary"]
        angle_of = torch.zeros(t, r // 2, 2, dtype=torch.float64, device=DEVICE)
        for i in range(r // 2):
            where = s["positions"][i % case["axes"]]
            angle_of[:, i, 0] = s["cos_sin"].double()[where, i]
            angle_of[:, i, 1] = s["cos_sin"].double()[where, r // 2 + i]

        def turn(x):
            x = x.double().clone()
            z = torch.view_as_complex(angle_of)[:, None]
            one, two = (slice(0, r, 2), slice(1, r, 2)) if case["adjacent"] else (slice(0, r // 2), slice(r // 2, r))
            y = torch.complex(x[..., one], x[..., two]) * z
            x[..., one], x[..., two] = y.real, y.imag
            return x
    if op == "norm":
        def unit(x, w):
            x = x.double()
            return turn(x / (x.square().sum(-1, keepdim=True) / dim + s["eps"]).sqrt() * w.double())
        return {"q": unit(s["q"], s["q_weight"]), "k": unit(s["k"], s["k_weight"])}
    if op == "append":
        def held(x):
            x = x.double()
            low, high = x.min(-1, keepdim=True).values.clamp(max=0), x.max(-1, keepdim=True).values.clamp(min=0)
            # the scale is kept as the nearest BF16 number
            step = torch.clamp((high - low).div(15).float().bfloat16().double(), min=torch.tensor(1e-20).bfloat16().double().item())
            zero = torch.clamp((-low / step).round(), 0, 15)
            x = step * (torch.clamp((x / step).round() + zero, 0, 15) - zero)
            x[t - case["padding"]:] = 0
            return x
        return {"keys": held(turn(s["k"])), "values": held(s["v"]), "q": turn(s["q"])}
    page = case["page"]
    raw = s["cache"].view(s["cache"].shape[0], 2, case["kv_heads"], -1)
    pairs = raw[..., page * dim // 2:].contiguous().view(torch.bfloat16).double().view(*raw.shape[:3], page, 2)

    def cached(side, pages):
        """[heads, keys, dim] of the given pages"""
        b = raw[pages, side, :, : page * dim // 2].reshape(len(pages), -1, page, dim // 2)
        x = torch.empty(*b.shape[:3], dim, dtype=torch.float64, device=DEVICE)
        x[..., 0::2], x[..., 1::2] = b.remainder(16), b.div(16, rounding_mode="floor")
        p = pairs[pages, side]
        return ((x - p[..., 1:]) * p[..., :1]).transpose(0, 1).flatten(1, 2)
    if op == "read":
        order = s["slots"].div(page, rounding_mode="floor")[::page]
        return {n: cached(i, order)[:, : case["tokens"]].transpose(0, 1) for i, n in enumerate(("keys", "values"))}
    news, kvs = _lengths(case)
    if sum(n * kv for n, kv in zip(news, kvs)) * case["q_heads"] * dim > 1e12:
        return None
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(sum(news), case["q_heads"], dim, dtype=torch.float64, device=DEVICE)
    done = 0
    for b, (n, kv) in enumerate(zip(news, kvs)):
        pages = s["block_table"][b, : -(-kv // page)].long()
        k, v = cached(0, pages)[:, :kv], cached(1, pages)[:, :kv]
        seen = torch.ones(n, kv, dtype=torch.bool, device=DEVICE).tril(kv - n)
        for h in range(case["q_heads"]):
            q = s["queries"][done:done + n, h].double()
            p = (q @ k[h // group].T * s["scale"]).masked_fill(~seen, -math.inf).softmax(-1)
            out[done:done + n, h] = p @ v[h // group]
        done += n
    return out
