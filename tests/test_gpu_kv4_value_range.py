"""kv4_attention over values at the end of their range: kv4_append holds an infinity as 8.5e37, and sums of such values, before they
are divided by the weights' sum, leave FP32's range.

Bounds as derived beside the attention's own tests."""
import pytest
import torch

from gpu_common import DEV, device_status
from oracle import kv4_ref as ref
from test_gpu_kv4_attention import Case, run_and_check, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def workspace(ops):
    return torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV)


def set_value(case, b, key, value):
    """value FP32 [kv_heads, dim] as sequence b's value of one key."""
    codes, pairs = ref.rows(case.cache, case.dim)
    c, scale, zero = ref.encode(value)
    page, row = int(case.table[b, key // case.page]), key % case.page
    codes[page, 1, :, row] = c[..., 0::2] | (c[..., 1::2] << 4)
    pairs[page, 1, :, row] = torch.stack([scale, zero], -1)


def saturated(dim, heads, key):
    x = torch.randn(heads, dim, generator=torch.Generator().manual_seed(key))
    x[:, key % dim], x[:, (key + 5) % dim] = float("inf"), float("-inf")
    x[:, 3] = float("inf")                                              # one component that is always at the end
    return x


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sequences", [[(1, 3), (1, 70), (1, 700)], [(1, 5003)], [(7, 40), (12, 700)], [(90, 90), (100, 700), (1, 65)], [(40, 1500), (2, 900)]])
def test_every_value_saturated(ops, workspace, dim, sequences):
    """Equal weights (a query head of zeros), nearly equal ones, and ordinary ones, over one warp's keys, over warps and over CTAs."""
    case = Case(sequences, 4, 2, dim, 32, seed=dim)
    case.q[:, 0] = 0
    case.q[:, 1] *= 1e-3
    for b, (_, keys) in enumerate(sequences):
        for key in range(keys):
            set_value(case, b, key, saturated(dim, 2, key))
    out = run_and_check(ops, workspace, case)
    assert bool(out[:, :, 3].isfinite().all()) and float(out[:, :, 3].min()) > 7e37


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sequences", [[(1, 90), (1, 800)], [(70, 90), (130, 800)], [(20, 1500)]])
def test_scores_that_rise_towards_saturated_values(ops, workspace, dim, sequences):
    """Weights up to 2^8 beside a running maximum that lags behind the scores: they rise by a little from key to key."""
    case = Case(sequences, 4, 2, dim, 16, seed=dim + 1)
    case.q.abs_().clamp_(max=1.0)
    codes, pairs = ref.rows(case.cache, dim)
    for b, (_, keys) in enumerate(sequences):
        for key in range(keys):
            page, row = int(case.table[b, key // 16]), key % 16
            codes[page, 0, :, row] = 0x88                               # code 8, zero point 7: every component is one step
            pairs[page, 0, :, row, 0] = 0.3 * key / keys
            pairs[page, 0, :, row, 1] = 7
            set_value(case, b, key, saturated(dim, 2, key))
    out = run_and_check(ops, workspace, case)
    assert bool(out[:, :, 3].isfinite().all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sequences", [[(1, 90), (1, 2500)], [(9, 90), (130, 800), (30, 1500)]])
def test_the_smallest_values(ops, workspace, dim, sequences):
    """Values at the least scale, 1e-20, alone: their sums stay within FP32's normal numbers."""
    case = Case(sequences, 4, 2, dim, 16, seed=dim + 2)
    for b, (_, keys) in enumerate(sequences):
        for key in range(keys):
            set_value(case, b, key, torch.randn(2, dim, generator=torch.Generator().manual_seed(key)) * 1e-20)
    run_and_check(ops, workspace, case)


def small_weights(case):
    """What the streaming kernel's FP16 weights lose beside the bound's relative 2^-11: they are multiples of 2^-24 in a unit in which
    the largest value scale that the row sees is between 64 and 128. A weight is off by at most half of that, 2^-25 * largest / 64,
    a component by 15 times that for each key, and the weights' sum that it is divided by is at least 1. [tokens, q_heads, 1]"""
    _, pairs = ref.rows(case.cache, case.dim)
    lost = torch.zeros(case.q.shape[0], case.kv_heads, 1, dtype=torch.float64)
    for b, keys in enumerate(case.lens.tolist()):
        ids = case.table[b, : -(-keys // case.page)].long()
        scales = pairs[ids, 1, :, :, 0].permute(1, 0, 2).flatten(1)[:, :keys].double()     # [heads, keys]
        start, end = int(case.starts[b]), int(case.starts[b + 1])
        for row in range(start, end):
            count = keys - (end - start) + row - start + 1
            if count > 0:
                lost[row, :, 0] = scales[:, :count].amax(1) * count * 15 * 2.0 ** -31
    return lost.repeat_interleave(case.q.shape[1] // case.kv_heads, 1)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [1e9, float("inf")])
@pytest.mark.parametrize("q_heads,kv_heads", [(4, 2), (2, 2), (24, 2)])
def test_large_values_that_are_hidden_from_a_row(ops, workspace, dim, size, q_heads, kv_heads):
    """New rows do not see the rows behind them: those before one with very large values answer as if it were not there. The large
    ones stand first, in the middle and last among the new rows, and alone behind a long prefix whose parts are joined."""
    sequences = [(5, 40), (9, 130), (2, 2), (4, 1500), (1, 20), (30, 63), (90, 130)]
    case = Case(sequences, q_heads, kv_heads, dim, 16, seed=dim + q_heads)
    large = {0: [4], 1: [3, 8], 2: [1], 3: [2], 5: [15, 29], 6: [40]}
    for b, rows in large.items():
        n, keys = sequences[b]
        for row in rows:
            x = torch.randn(kv_heads, dim, generator=torch.Generator().manual_seed(row)).clamp(-3, 3)
            set_value(case, b, keys - n + row, x * size)
    out = torch.full(case.q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    ops.kv4_attention(*case.device(), workspace, out, case.scale)
    want, spread, reach = case.want()
    bound = tolerance(want, spread, reach) + small_weights(case)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    assert device_status(ops) == 0
