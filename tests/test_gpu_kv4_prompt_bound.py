"""Prompts held to the prompt kernel's own score error. The bound beside the attention's other tests gives every row the streaming
kernel's 2^-16 of the largest score R. Rows of the prompt kernel have no fixed point: their products are exact, accumulated over at
most 16 steps with 2^-23 of the largest partial sum each (2^-19 R), and the key's scale times the softmax scale, that number itself
and its product are rounded to FP32 (3 * 2^-24 R): below 2^-18 R. A weight times its value's scale is held in units of 2^40 as a BF16 number,
of which the smallest normal one is 2^-126: what is below 2^-86 may be lost, for a component 15 times that a key, over a sum of at
least 1. (Such components are those of which every key with a larger weight holds an exact 0.)"""
import pytest
import torch

from gpu_common import DEV, device_status
from test_gpu_kv4_attention import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def workspace(ops):
    return torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("magnitude", [1.0, 6.0, 20.0])
@pytest.mark.parametrize("q_heads,kv_heads,sequences", [(4, 4, [(70, 70), (129, 400), (0, 9), (257, 300)]), (6, 1, [(40, 1500)]), (8, 2, [(33, 200), (17, 17)])])
def test_prompts(ops, workspace, dim, magnitude, q_heads, kv_heads, sequences):
    assert all(n == 0 or n * q_heads // kv_heads > 64 for n, _ in sequences)      # more rows than the streaming kernel takes
    case = Case(sequences, q_heads, kv_heads, dim, 16, seed=dim + q_heads, magnitude=magnitude)
    out = torch.full(case.q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    ops.kv4_attention(*case.device(), workspace, out, case.scale)
    want, spread, reach = case.want()
    bound = 2.0 ** -8 * want.abs() + (1.05 * 2.0 ** -8 + torch.expm1(2 * 2.0 ** -18 * reach)) * spread + int(case.lens.max()) * 15 * 2.0 ** -86
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    assert device_status(ops) == 0
