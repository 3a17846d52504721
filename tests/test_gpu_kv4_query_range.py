"""kv4_attention with query heads of zeros, of very small components and of NaN, and with keys at the end of their range,
wherever keys are hidden from them: behind the row, behind the sequence, on pages that cannot be followed, in another part of a
history that is split.

Bounds as derived beside the attention's own tests. A query head of zeros has scores of exactly 0: its output is the mean of the
values, and the score's error is 0. Components below 2^-100 are held to a grid of 2^-100 / 32639, which moves a score by
2^-116 * dim * 15 steps * scale at most: nothing beside the 5 % that the bound leaves to FP32 sums."""
import pytest
import torch

from gpu_common import DEV, device_status
from oracle import kv4_ref as ref
from test_gpu_kv4_attention import Case, run_and_check

pytestmark = pytest.mark.gpu

LENGTHS = [0, 1, 31, 32, 33, 63, 64, 65, 100]


@pytest.fixture(scope="module")
def workspace(ops):
    return torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV)


def quiet(case):
    """Heads of zeros and of tiny components beside ordinary ones; the first row as a whole."""
    heads = case.q.shape[1]
    case.q[0] = 0
    case.q[:, 0] = 0
    for head, size in ((1, 2.0 ** -60), (2, 2.0 ** -110), (3, 2.0 ** -130)):
        if head < heads:
            case.q[:, head] *= size
    if heads > 4:
        case.q[:, 4] = 0
        case.q[:, 4, 7] = 2.0 ** -133                                   # BF16's smallest number, alone
    return case


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 2), (12, 1)])
def test_single_tokens(ops, workspace, dim, q_heads, kv_heads):
    run_and_check(ops, workspace, quiet(Case([(1, n) for n in LENGTHS], q_heads, kv_heads, dim, 16, seed=dim + q_heads, spare_rows=2)))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(6, 2), (4, 4)])
def test_few_and_many_rows(ops, workspace, dim, q_heads, kv_heads):
    """Both kernels: rows of one sequence hide keys from one another, some rows see nothing."""
    sequences = [(5, 5), (9, 100), (4, 2), (1, 65), (70, 70), (90, 333), (80, 30), (0, 7)]
    run_and_check(ops, workspace, quiet(Case(sequences, q_heads, kv_heads, dim, 32, seed=dim + q_heads)))


@pytest.mark.parametrize("dim,sequences", [(64, [(1, 5003), (1, 1)]), (128, [(1, 4000), (1, 2501)]), (256, [(1, 3001), (1, 33)]), (128, [(40, 1500), (2, 900)]),
                                           (256, [(30, 1501)])])
def test_histories_that_are_split_and_joined(ops, workspace, dim, sequences):
    run_and_check(ops, workspace, quiet(Case(sequences, 8, 2, dim, 64, seed=dim)))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_bad_pages(ops, workspace, dim):
    case = quiet(Case([(1, 100), (1, 64), (20, 120), (100, 160)], 8, 2, dim, 16, seed=5))
    pages = case.cache.shape[0]
    case.table[0, 2], case.table[0, 5] = -1, pages
    case.table[1, :4] = 2 ** 31 - 1                                     # a sequence without one good page
    case.table[2, 0] = case.table[3, 3] = -2 ** 31
    run_and_check(ops, workspace, case, status=8)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_queries_that_see_nothing_are_zeros(ops, workspace, dim):
    """Rows without a key are zeros whatever the query holds (padding is rarely initialised); rows that see one are NaN."""
    case = Case([(1, 0), (1, 40), (4, 2), (1, 30), (90, 20)], 4, 2, dim, 16, seed=6)
    case.table[3, :2] = -1                                              # no page that can be followed
    case.q[0, 1, 3] = case.q[1, 1, 3] = case.q[7, 0, 0] = float("nan")
    case.q[2, 2] = float("inf")
    case.q[6] = float("nan")
    case.q[7, 3] = float("nan")
    case.q[8, 1] = float("nan")
    q, cache, table, starts, lens = case.device()
    out = torch.full_like(q, 5.0)
    ops.kv4_attention(q, cache, table, starts, lens, workspace, out, case.scale)
    got = out.cpu()
    seen = torch.tensor([0] + [1] + [0, 0, 1, 1] + [0] + [0] * 70 + [1] * 20, dtype=torch.bool)
    assert not bool((got[~seen] != 0).any()) and not bool(got[~seen].isnan().any())
    nan = case.q.isnan().any(-1) | case.q.isinf().any(-1)
    assert torch.equal(got[seen].isnan().all(-1), nan[seen]) and not bool(got[seen][~nan[seen]].isnan().any())
    assert device_status(ops) == 8


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sequences", [[(1, 70), (1, 300)], [(3, 70), (20, 300)], [(3, 70), (100, 300)]])
def test_a_key_at_the_end_of_its_range_takes_all_the_weight(ops, workspace, dim, sequences):
    """An infinite key component is held as 8.5e37. Queries of up to 2.5 make products of up to 2.2e38, within FP32: the rows
    that see the key answer with its value, the others as if it were not there."""
    heads, place = 4, 20
    case = Case(sequences, heads, 2, dim, 16, seed=dim)
    case.q[:, :, 0] = case.q[:, :, 0].abs().clamp(max=2.0) + 0.5
    codes, pairs = ref.rows(case.cache, dim)
    key = torch.zeros(2, dim)
    key[:, 0] = float("inf")
    c, scale, zero = ref.encode(key)
    for b in range(2):
        at = int(case.table[b, place // 16]), place % 16
        codes[at[0], 0, :, at[1]] = c[..., 0::2] | (c[..., 1::2] << 4)
        pairs[at[0], 0, :, at[1]] = torch.stack([scale, zero], -1)
    out = run_and_check(ops, workspace, case).cpu()
    held = ref.values(case.cache, dim)
    for b, (rows, keys) in enumerate(sequences):
        value = held[int(case.table[b, place // 16]), 1, :, place % 16].repeat_interleave(heads // 2, 0)
        first = int(case.starts[b]) + max(0, place - (keys - rows))
        diff = (out[first:int(case.starts[b + 1])].double() - value).abs()
        assert bool((diff <= 2.0 ** -8 * value.abs()).all())            # one rounding: weight 1 and its value's scale are exact


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sequences", [[(1, 70), (9, 300)], [(100, 300), (80, 80), (30, 1500)]])
def test_scores_far_beyond_2_to_the_24(ops, workspace, dim, sequences):
    """Scores of about 1e12, of which an FP32 number holds no fraction: one key takes all the weight, and the output is finite.
    (The bound says no more here: a score's own rounding is larger than the distance between keys.)"""
    case = Case(sequences, 4, 2, dim, 16, seed=dim, magnitude=1e5)
    case.q *= 1e6
    out = run_and_check(ops, workspace, case).cpu().double()
    held = ref.values(case.cache, dim)
    for b, (rows, keys) in enumerate(sequences):
        ids = case.table[b, : -(-keys // 16)].long()
        values = held[ids, 1].permute(1, 0, 2, 3).flatten(1, 2)[:, :keys]                  # [heads, keys, dim]
        start = int(case.starts[b])
        for h in range(4):
            low, high = values[h // 2].amin(0), values[h // 2].amax(0)
            got = out[start:start + rows, h]
            room = 2.0 ** -8 * torch.maximum(low.abs(), high.abs())
            assert bool((got >= low - room).all()) and bool((got <= high + room).all())
