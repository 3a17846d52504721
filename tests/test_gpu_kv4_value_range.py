"""kv4_attention over values at the end of their range: kv4_append holds an infinity as 8.5e37, and sums of such values, before they
are divided by the weights' sum, leave FP32's range.

Bounds as derived beside the attention's own tests."""
import pytest
import torch

from gpu_common import DEV
from oracle import kv4_ref as ref
from test_gpu_kv4_attention import Case, run_and_check

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
