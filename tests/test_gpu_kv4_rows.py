"""qk_norm_rope, kv4_append and kv4_read against the CPU restatement.

Norm and rotation: one BF16 rounding (half a step, 2^-8 relative) plus FP32 noise, which is bounded by 16 roundings of
the two products that a rotated component is made of. Encoding and reading: equal bytes."""
import pytest
import torch

from gpu_common import DEV, assert_bit_equal, device_status, guarded
from oracle import kv4_ref as ref

pytestmark = pytest.mark.gpu


def table(rows, rotary):
    rate = 10000.0 ** (-torch.arange(rotary // 2).double() / (rotary // 2))
    angle = torch.arange(rows)[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def heads(g, tokens, count, dim):
    return (torch.randn(tokens, count, dim, generator=g) * (1 + 3 * (torch.rand(count, dim, generator=g) < 0.02))).bfloat16()


def placement(g, tokens, rotary, axes, rows):
    positions = torch.randint(0, rows, (axes, tokens), generator=g)
    axis_of = torch.randint(0, axes, (rotary // 2,), generator=g, dtype=torch.int32) if axes > 1 else None
    return positions, axis_of


def on(t):
    return None if t is None else t.to(DEV)


def noise(x, cos_sin):
    """Bound on the FP32 error of a rotated component: 16 roundings of both products (|cos|, |sin| <= 1)."""
    if cos_sin is None:
        return 16 * 2.0 ** -24 * x.abs()
    r = cos_sin.shape[1]
    bound = x.abs().clone()
    pair_sum = x[..., :r].abs().amax(-1, keepdim=True) * 2
    bound[..., :r] = pair_sum
    return 16 * 2.0 ** -24 * bound


@pytest.mark.parametrize("dim,q_heads,kv_heads,rotary,axes,adjacent", [
    (64, 1, 1, 64, 1, False), (64, 7, 3, 16, 1, True), (64, 16, 16, 64, 3, False),
    (128, 32, 8, 128, 1, False), (128, 5, 1, 32, 2, True), (128, 6, 2, 128, 4, False),
    (256, 24, 4, 64, 1, False), (256, 3, 1, 256, 1, True), (256, 8, 8, 48, 3, False)])
@pytest.mark.parametrize("tokens", [1, 3, 130])
def test_norm_and_rotation(ops, dim, q_heads, kv_heads, rotary, axes, adjacent, tokens):
    g = torch.Generator().manual_seed(dim + q_heads + tokens)
    qkv = heads(g, tokens, q_heads + 2 * kv_heads, dim)
    qw, kw = torch.randn(dim, generator=g).bfloat16(), (1 + 0.1 * torch.randn(dim, generator=g)).bfloat16()
    cos_sin = table(513, rotary)
    positions, axis_of = placement(g, tokens, rotary, axes, 513)
    cosine, sine = ref.angles(cos_sin, positions, axis_of, tokens)
    dev = qkv.to(DEV)
    q, k = dev[:, :q_heads], dev[:, q_heads:q_heads + kv_heads]
    q_out, q_check = guarded((tokens, q_heads, dim), torch.bfloat16, float("nan"))
    k_out, k_check = guarded((tokens, kv_heads, dim), torch.bfloat16, float("nan"))
    args = (on(qw), on(kw), on(cos_sin), on(positions), on(axis_of), q_out, k_out, 1e-5, 0.5, adjacent)
    ops.qk_norm_rope(q, k, *args)
    for got, x, w in ((q_out, qkv[:, :q_heads], qw), (k_out, qkv[:, q_heads:q_heads + kv_heads], kw)):
        unit = ref.norm(x, w, 1e-5, 0.5)
        want = ref.rotate(unit, cosine, sine, adjacent)
        tolerance = 2.0 ** -8 * want.abs() + noise(unit, cos_sin) * 1.01
        assert bool(((got.cpu().double() - want).abs() <= tolerance).all())
    q_check()
    k_check()
    # in place on the projection's output: the same bits, the values between untouched
    ops.qk_norm_rope(q, k, *args[:5], q, k, 1e-5, 0.5, adjacent)
    assert_bit_equal(dev[:, :q_heads], q_out, "q in place")
    assert_bit_equal(dev[:, q_heads:q_heads + kv_heads], k_out, "k in place")
    assert_bit_equal(dev[:, q_heads + kv_heads:], qkv[:, q_heads + kv_heads:], "values")
    assert device_status(ops) == 0


def test_norm_without_rotation_and_rotation_without_norm(ops):
    g = torch.Generator().manual_seed(3)
    q, k = heads(g, 5, 4, 128), heads(g, 5, 2, 128)
    w = torch.randn(128, generator=g).bfloat16()
    q_out, k_out = torch.empty_like(q, device=DEV), torch.empty_like(k, device=DEV)
    ops.qk_norm_rope(on(q), on(k), on(w), None, None, None, None, q_out, k_out)
    want = ref.norm(q, w, 1e-6, 0.0)
    assert bool(((q_out.cpu().double() - want).abs() <= (2.0 ** -8 + 17 * 2.0 ** -24) * want.abs()).all())
    assert_bit_equal(k_out, k, "no weight and no table: a copy")
    cos_sin, positions = table(64, 128), torch.tensor([0, 1, 63, 7, 7])
    ops.qk_norm_rope(on(q), on(k), None, None, on(cos_sin), on(positions), None, q_out, k_out)
    cosine, sine = ref.angles(cos_sin, positions, None, 5)
    assert_bit_equal(q_out, ref.rotate(q.float(), cosine, sine, False).bfloat16(), "rotation alone is exact FP32 arithmetic")
    zero = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=DEV)     # a zero head stays zero
    ops.qk_norm_rope(zero, zero.clone(), on(w), on(w), None, None, None, zero, torch.empty_like(zero), 1e-6)
    assert int((zero != 0).sum()) == 0
    empty = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope(empty, empty, on(w), on(w), None, None, None, empty, empty)


def test_bad_positions_give_nan_and_a_status(ops):
    g = torch.Generator().manual_seed(4)
    q, k = heads(g, 4, 4, 128), heads(g, 4, 2, 128)
    cos_sin, positions = table(16, 64), torch.tensor([3, 16, -1, 15])
    q_out, k_out = torch.empty_like(q, device=DEV), torch.empty_like(k, device=DEV)
    ops.qk_norm_rope(on(q), on(k), None, None, on(cos_sin), on(positions), None, q_out, k_out)
    bad = torch.tensor([False, True, True, False])
    for out in (q_out, k_out):
        assert torch.equal(out.cpu().isnan().all(-1).all(-1), bad) and not bool(out.cpu()[~bad].isnan().any())
    assert device_status(ops) == 8
    two = torch.stack([positions.clamp(0, 15)] * 2)
    axis_of = torch.zeros(32, dtype=torch.int32)
    axis_of[17] = 2                                                    # an axis that is not there
    ops.qk_norm_rope(on(q), on(k), None, None, on(cos_sin), on(two), on(axis_of), q_out, k_out)
    assert bool(q_out.isnan().all()) and device_status(ops) == 8


@pytest.mark.parametrize("dim,q_heads,kv_heads,rotary,axes,adjacent,page", [
    (64, 2, 1, 64, 1, False, 16), (64, 9, 3, 32, 2, True, 256), (128, 32, 8, 128, 1, False, 64),
    (128, 0, 5, 0, 1, False, 32), (256, 24, 4, 64, 1, False, 16), (256, 3, 3, 256, 3, True, 128), (128, 4, 4, 0, 1, False, 16)])
@pytest.mark.parametrize("tokens", [1, 19, 150])
def test_append_bytes(ops, dim, q_heads, kv_heads, rotary, axes, adjacent, page, tokens):
    g = torch.Generator().manual_seed(dim + page + tokens)
    qkv = heads(g, tokens, q_heads + 2 * kv_heads, dim)
    q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv_heads], qkv[:, q_heads + kv_heads:]
    v[0] = 0                                                           # an all-zero head
    v[-1, -1, 5] = float("nan")
    k[tokens // 2, 0, 3] = float("inf")
    k[tokens // 2, 0, 4] = float("-inf")
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 2:
        slots[1], slots[-1] = -1, -7                                   # padding
    cache, check = guarded((pages, 2, kv_heads, ref.block_bytes(page, dim)), torch.uint8, 0x5A)
    want = torch.full(cache.shape, 0x5A, dtype=torch.uint8)
    cos_sin = positions = axis_of = None
    turned_q, turned_k = q.float(), k.float()
    if rotary:
        cos_sin = table(300, rotary)
        positions, axis_of = placement(g, tokens, rotary, axes, 300)
        cosine, sine = ref.angles(cos_sin, positions, axis_of, tokens)
        turned_q, turned_k = (ref.rotate(t, cosine, sine, adjacent) for t in (turned_q, turned_k))
    ref.store(want, slots, turned_k, v.float())
    dev = qkv.to(DEV)
    q_out = torch.empty(tokens, q_heads, dim, dtype=torch.bfloat16, device=DEV) if q_heads else None
    ops.kv4_append(dev[:, :q_heads] if q_heads else None, dev[:, q_heads:q_heads + kv_heads], dev[:, q_heads + kv_heads:], on(cos_sin),
                   on(positions), on(axis_of), on(slots), q_out, cache, adjacent)
    assert_bit_equal(cache, want, "cache bytes")                       # rows that were not named are as they were
    check()
    if q_heads:
        assert_bit_equal(q_out, turned_q.bfloat16(), "rotated queries")
    # what is held is within half a step of what came in, and the clamped ends within the scale's rounding of that
    kept = torch.nonzero(slots >= 0).flatten()
    held = ref.values(want, dim)
    for side, x in ((0, turned_k), (1, v.float())):
        x = torch.nan_to_num(x, nan=0.0, posinf=8.5e37, neginf=-8.5e37).double()
        step = ref.rows(want, dim)[1][..., 0].double()
        for t in kept.tolist():
            at = int(slots[t])
            diff = (held[at // page, side, :, at % page] - x[t]).abs()
            assert bool((diff <= (0.5 + 15 * 2.0 ** -8) * step[at // page, side, :, at % page, None]).all())
    # read back
    k_out, v_out = (torch.full((tokens, kv_heads, dim), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.kv4_read(cache, on(slots), k_out, v_out)
    at = slots.clamp(min=0)
    expected = torch.where((slots >= 0)[:, None, None, None], held[at // page, :, :, at % page], 0.0).float().bfloat16() + 0.0
    assert_bit_equal(k_out + 0.0, expected[:, 0], "keys read")
    assert_bit_equal(v_out + 0.0, expected[:, 1], "values read")
    assert device_status(ops) == 0


def test_rounding_ties_and_extreme_ranges(ops):
    """Heads whose quotients are exact halves, tiny, huge and one-sided ones."""
    dim = 64
    x = torch.zeros(8, 1, dim)
    x[0, 0] = torch.arange(dim) % 16 - 7.5                             # range 15: every component is a tie
    x[1, 0] = (torch.arange(dim) % 31) * 0.5
    x[2, 0] = -(torch.arange(dim) % 31) * 0.5
    x[3, 0] = 1e-30
    x[4, 0] = torch.linspace(-3e38, 3e38, dim)
    x[5, 0] = torch.linspace(1e-19, 2e-19, dim)
    x[6, 0] = 4.0
    x[7, 0, 0] = -2.0
    x = x.bfloat16()
    cache = torch.zeros(1, 2, 1, ref.block_bytes(16, dim), dtype=torch.uint8, device=DEV)
    want = cache.cpu()
    slots = torch.arange(8)
    ref.store(want, slots, x.float(), x.flip(-1).float())
    ops.kv4_append(None, on(x), on(x.flip(-1)), None, None, None, on(slots), None, cache)
    assert_bit_equal(cache, want, "cache bytes")


def test_slots_and_positions_outside_are_left_out(ops):
    g = torch.Generator().manual_seed(9)
    q, k, v = heads(g, 4, 2, 128), heads(g, 4, 1, 128), heads(g, 4, 1, 128)
    cache, check = guarded((2, 2, 1, ref.block_bytes(16, 128)), torch.uint8, 0x11)
    want = torch.full(cache.shape, 0x11, dtype=torch.uint8)
    slots = torch.tensor([31, 32, 2 ** 40, 0])
    cos_sin, positions = table(8, 128), torch.tensor([1, 2, 3, 8])
    cosine, sine = ref.angles(cos_sin, positions.clamp(max=7), None, 4)
    ref.store(want, torch.tensor([31, -1, -1, -1]), ref.rotate(k.float(), cosine, sine, False), v.float())
    q_out = torch.empty_like(q, device=DEV)
    ops.kv4_append(on(q), on(k), on(v), on(cos_sin), on(positions), None, on(slots), q_out, cache)
    assert_bit_equal(cache, want, "cache bytes")
    check()
    assert device_status(ops) == 8
    assert_bit_equal(q_out[:3], ref.rotate(q.float(), cosine, sine, False).bfloat16()[:3], "queries")
    assert bool(q_out[3].isnan().all())
    k_out, v_out = torch.ones_like(k, device=DEV), torch.ones_like(v, device=DEV)
    ops.kv4_read(cache, on(slots), k_out, v_out)
    assert int((k_out[1:3] != 0).sum()) == 0 and device_status(ops) == 8


def test_row_operators_follow_a_captured_graph(ops):
    """Captured once, replayed with other inputs, positions and slots; on a stream of its own."""
    g = torch.Generator().manual_seed(21)
    tokens, dim, page = 6, 128, 16
    cos_sin = on(table(100, dim))
    w = on(torch.randn(dim, generator=g).bfloat16())
    qkv = heads(g, tokens, 8, dim).to(DEV)
    positions, slots = torch.arange(tokens, device=DEV), torch.arange(tokens, device=DEV)
    cache = torch.zeros(4, 2, 2, ref.block_bytes(page, dim), dtype=torch.uint8, device=DEV)
    q_out, k_out = (torch.empty(tokens, n, dim, dtype=torch.bfloat16, device=DEV) for n in (4, 2))
    k_back, v_back = torch.empty_like(k_out), torch.empty_like(k_out)

    def step():
        ops.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], w, w, cos_sin, positions, None, q_out, k_out)
        ops.kv4_append(None, k_out, qkv[:, 6:], None, None, None, slots, None, cache)
        ops.kv4_read(cache, slots, k_back, v_back)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        qkv.copy_(heads(g, tokens, 8, dim))
        positions.add_(40)
        slots.add_(20)
        graph.replay()
    stream.synchronize()
    got = [t.cpu() for t in (q_out, k_out, k_back, v_back, cache)]
    cache.zero_()
    cache[:1] = got[4][:1].to(DEV)
    step()
    for a, b in zip(got[:4], (q_out, k_out, k_back, v_back)):
        assert_bit_equal(a, b, "replayed against eager")
    assert_bit_equal(got[4][1:], cache[1:], "cache")


def test_row_operators_refuse(ops):
    t = lambda *s, d=torch.bfloat16: torch.zeros(*s, dtype=d, device=DEV)  # noqa: E731
    q, k, cos_sin, positions = t(4, 8, 128), t(4, 2, 128), t(16, 128, d=torch.float32), t(4, d=torch.long)
    slots, cache = torch.arange(4, device=DEV), t(2, 2, 2, ref.block_bytes(16, 128), d=torch.uint8)
    w = t(128)

    def refused(match, call, *args):
        with pytest.raises(RuntimeError, match=match):
            call(*args)

    rope, append, read = ops.qk_norm_rope, ops.kv4_append, ops.kv4_read
    refused("Head dimension", rope, t(4, 8, 96), t(4, 2, 96), None, None, None, None, None, t(4, 8, 96), t(4, 2, 96))
    refused("BF16 heads", rope, q.float(), k, None, None, None, None, None, q.clone(), k.clone())
    refused("heads of a token", rope, t(4, 128, 8).transpose(1, 2), k, None, None, None, None, None, q.clone(), k.clone())
    refused("aligned rows", rope, t(4 * 1024 + 8)[1:4097].view(4, 8, 128), k, None, None, None, None, None, q.clone(), k.clone())
    refused("cos_sin table", rope, q, k, None, None, t(16, 120, d=torch.float32), positions, None, q.clone(), k.clone())
    refused("cos_sin table", rope, q, k, None, None, t(16, 256, d=torch.float32), positions, None, q.clone(), k.clone())
    refused("needs positions", rope, q, k, None, None, cos_sin, None, None, q.clone(), k.clone())
    refused("need a cos_sin", rope, q, k, None, None, None, positions, None, q.clone(), k.clone())
    refused("positions", rope, q, k, None, None, cos_sin, positions[:3], None, q.clone(), k.clone())
    refused("need axis_of", rope, q, k, None, None, cos_sin, t(2, 4, d=torch.long), None, q.clone(), k.clone())
    refused("dtype", rope, q, k, None, None, cos_sin, positions.int(), None, q.clone(), k.clone())
    refused("norm weight", rope, q, k, t(64), None, None, None, None, q.clone(), k.clone())
    refused("Wrong query", rope, q, k, w, w, None, None, None, t(3, 8, 128), k.clone())
    refused("its own input", rope, q, k, w, w, None, None, None, q.clone(), q[:, :2])
    shifted = t(5, 8, 128)
    refused("its own input", rope, shifted[:4], k, w, w, None, None, None, shifted[1:], k.clone())
    refused("same CUDA device", rope, q, k.cpu(), w, w, None, None, None, q.clone(), k.clone())
    refused("UINT8 cache", append, None, k, k.clone(), None, None, None, slots, None, t(2, 2, 3, ref.block_bytes(16, 128), d=torch.uint8))
    refused("UINT8 cache", append, None, k, k.clone(), None, None, None, slots, None, t(2, 2, 2, 17, d=torch.uint8))
    refused("Cache pages", append, None, k, k.clone(), None, None, None, slots, None, t(2, 2, 2, ref.block_bytes(24, 128), d=torch.uint8))
    refused("slots", append, None, k, k.clone(), None, None, None, slots[:3], None, cache)
    refused("come together", append, q, k, k.clone(), None, None, None, slots, None, cache)
    refused("q_out may be q", append, t(4, 2, 128), k, k.clone(), None, None, None, slots, k, cache)
    refused("contiguous keys", read, cache, slots, q[:, :2], k.clone())
    refused("must not overlap", read, cache, slots, k, k)
