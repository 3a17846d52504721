"""The 4-bit cache's operators as a server calls them: repeated, side by side, captured, padded, with many sequences. Bounds as
derived beside the attention's own tests."""
import pytest
import torch

from gpu_common import DEV, assert_bit_equal, device_status, guarded
from oracle import kv4_ref as ref
from test_gpu_kv4_attention import Case, run_and_check, tolerance

pytestmark = pytest.mark.gpu

SPLIT = [(40, 1500), (1, 900)]                                          # few row tiles over a long prefix: split and joined
MIXES = [(128, 8, 2, 64, [(1, 3000), (1, 17), (1, 700)]), (256, 6, 1, 16, SPLIT), (64, 8, 8, 32, [(3, 500), (300, 400), (0, 0), (17, 60)]),
         (128, 4, 1, 16, [(260, 600), (16, 400), (1, 1)])]


@pytest.fixture(scope="module")
def workspace(ops):
    return torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("dim,q_heads,kv_heads,page,sequences", MIXES)
def test_the_same_call_gives_the_same_bits(ops, workspace, dim, q_heads, kv_heads, page, sequences):
    case = Case(sequences, q_heads, kv_heads, dim, page, seed=31)
    first = run_and_check(ops, workspace, case)
    args = case.device()
    for _ in range(5):
        out = torch.empty_like(first)
        ops.kv4_attention(*args, workspace, out, case.scale)
        assert_bit_equal(out, first, "again")


def test_calls_side_by_side_with_a_workspace_each(ops):
    cases = [Case([(1, 4000), (1, 20)], 8, 2, 128, 16, seed=41), Case(SPLIT, 6, 1, 256, 64, seed=42), Case([(1, 2000)] * 3, 8, 1, 64, 32, seed=43)]
    spaces = [torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV) for _ in cases]
    want = [run_and_check(ops, space, case) for space, case in zip(spaces, cases)]
    args = [case.device() for case in cases]
    outs = [[torch.empty_like(w) for _ in range(8)] for w in want]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for i in range(8):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                ops.kv4_attention(*args[j], spaces[j], outs[j][i], cases[j].scale)
    torch.cuda.synchronize()
    for j, w in enumerate(want):
        for out in outs[j]:
            assert_bit_equal(out, w, f"stream {j}")
    assert device_status(ops) == 0


def test_a_captured_step_serves_prompts_and_single_tokens(ops, workspace):
    """The capture has room for 300 rows and four sequences; replays fill it differently, empty places and padding rows among them."""
    case = Case([(300, 1200), (0, 1000), (0, 1300), (0, 40)], 6, 2, 128, 16, seed=51)
    q, cache, table, starts, lens = case.device()
    out = torch.empty_like(q)
    ops.kv4_attention(q, cache, table, starts, lens, workspace, out, case.scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv4_attention(q, cache, table, starts, lens, workspace, out, case.scale)
    for rows, keys in [([300, 0, 0, 0], [1200, 0, 0, 0]), ([1, 1, 1, 1], [1200, 1000, 1300, 40]), ([20, 1, 260, 2], [20, 999, 261, 39]),
                       ([0, 0, 0, 0], [1, 1, 1, 1]), ([2, 40, 0, 17], [3, 700, 9, 17])]:
        case.starts = torch.tensor([sum(rows[:i]) for i in range(5)], dtype=torch.int32)
        case.lens = torch.tensor(keys, dtype=torch.int32)
        starts.copy_(case.starts)
        lens.copy_(case.lens)
        out.fill_(float("nan"))
        graph.replay()
        want, spread, reach = case.want()
        used = sum(rows)
        bad = (out[:used].cpu().double() - want[:used]).abs() > tolerance(want, spread, reach)[:used]
        assert not bool(bad.any()) and bool(out[used:].isnan().all()), (rows, keys)
    assert device_status(ops) == 0


def test_rows_before_the_first_sequence_are_left_alone(ops, workspace):
    for sequences in ([(1, 40), (1, 90)], [(20, 40), (1, 90)]):
        case = Case(sequences, 8, 2, 128, 16, seed=61, spare_rows=7)
        args = case.device()
        first = run_and_check(ops, workspace, case)
        rows = int(case.starts[-1])
        q = torch.cat([args[0][-3:], args[0][:-3]])                     # three rows more in front
        out = torch.full_like(q, float("nan"))
        ops.kv4_attention(q, args[1], args[2], args[3] + 3, args[4], workspace, out, case.scale)
        assert bool(out[:3].isnan().all()) and bool(out[3 + rows:].isnan().all())
        assert_bit_equal(out[3:3 + rows], first[:rows], "shifted")


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_thousands_of_sequences(ops, workspace, dim, page):
    g = torch.Generator().manual_seed(71)
    keys = torch.randint(0, 70, (2500,), generator=g).tolist()
    run_and_check(ops, workspace, Case([(1, n) for n in keys], 4, 2, dim, page, seed=72))
    mixed = [(int(r), int(r) + n) for r, n in zip(torch.randint(0, 4, (700,), generator=g), keys)]
    mixed[333] = (90, 150)
    run_and_check(ops, workspace, Case(mixed, 4, 2, dim, page, seed=73))


def test_a_padded_batch_whose_rows_all_belong_to_one_sequence(ops, workspace):
    """No more rows than sequences, but not one each."""
    run_and_check(ops, workspace, Case([(0, 0)] * 40 + [(50, 333)] + [(0, 5)] * 20, 8, 2, 128, 16, seed=81))


def test_the_same_slot_twice(ops):
    """Reading: both rows. Storing the same row twice: that row; its neighbours keep their bytes."""
    dim, heads, page = 128, 3, 16
    g = torch.Generator().manual_seed(91)
    k = torch.randn(1, heads, dim, generator=g).bfloat16().to(DEV).expand(6, -1, -1).contiguous()
    v = torch.randn(1, heads, dim, generator=g).bfloat16().to(DEV).expand(6, -1, -1).contiguous()
    cache = torch.randint(0, 256, (3, 2, heads, ref.block_bytes(page, dim)), dtype=torch.uint8, generator=g).to(DEV)
    want = cache.clone()
    ops.kv4_append(None, k[:1], v[:1], None, None, None, torch.tensor([21], device=DEV), None, want)
    ops.kv4_append(None, k, v, None, None, None, torch.full((6,), 21, device=DEV), None, cache)
    assert_bit_equal(cache, want, "cache")
    got_k, check_k = guarded((4, heads, dim), torch.bfloat16, float("nan"))
    got_v, check_v = guarded((4, heads, dim), torch.bfloat16, float("nan"))
    ops.kv4_read(cache, torch.tensor([21, 21, -1, 21], device=DEV), got_k, got_v)
    for got in (got_k, got_v):
        assert_bit_equal(got[0], got[1], "twice")
        assert_bit_equal(got[0], got[3], "thrice")
        assert not bool(got[2].any())
    check_k(), check_v()
    assert device_status(ops) == 0


def test_tables_of_more_than_2_to_the_30_tokens_are_refused(ops, workspace):
    case = Case([(1, 20)], 8, 2, 128, 16)
    q, cache, _, starts, lens = case.device()
    table = torch.zeros(1, 2 ** 26 + 1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="block_table"):
        ops.kv4_attention(q, cache, table, starts, lens, workspace, torch.empty_like(q), case.scale)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (2, 2), (14, 2)])
def test_rows_on_either_side_of_the_kernels_border(ops, workspace, dim, q_heads, kv_heads):
    """Sequences of one query row, of a few blocks of rows and of one row more than those, in one call."""
    group = q_heads // kv_heads
    around = [max(1, 64 // group + d) for d in (-1, 0, 1, 2)]
    run_and_check(ops, workspace, Case([(n, n + 75) for n in around] + [(1, 30), (n := 130 // group + 1, n)], q_heads, kv_heads, dim, 16, seed=dim + group))


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 16), (64, 256), (128, 64), (256, 128)])
def test_bad_pages_among_a_prompts_keys(ops, workspace, dim, page):
    """Page numbers outside the cache at a tile's start, middle and end, and in a sequence's last, partly filled page."""
    case = Case([(90, 3 * 256 + 5), (130, 700), (100, 100)], 4, 2, dim, page, seed=page + dim)
    pages = case.cache.shape[0]
    case.table[0, 0] = pages
    case.table[0, -(-(3 * 256 + 5) // page) - 1] = -7
    case.table[1, 700 // page // 2] = 2 ** 31 - 1
    case.table[1, (700 // page // 2) + 1] = -1
    run_and_check(ops, workspace, case, status=8)


@pytest.mark.parametrize("dim,q_heads,kv_heads,sequences", [
    (128, 96, 1, [(1, 70), (1, 333)]), (128, 96, 1, [(1, 70), (3, 150), (0, 9)]), (64, 1024, 1, [(1, 40), (1, 5)]),
    (64, 1024, 1, [(2, 90)]), (256, 260, 260, [(1, 20), (1, 33)]), (64, 130, 130, [(70, 90), (1, 33)])])
def test_many_heads(ops, workspace, dim, q_heads, kv_heads, sequences):
    """More query heads on a key head than a tile has rows, and more key heads than there are multiprocessors."""
    run_and_check(ops, workspace, Case(sequences, q_heads, kv_heads, dim, 16, seed=q_heads + len(sequences)))


def test_many_heads_in_the_row_operators(ops):
    """1024 query heads and 1024 key heads: appended, read back and compared with the checker; the norm against its definition."""
    dim, page, tokens, heads = 64, 16, 3, 1024
    g = torch.Generator().manual_seed(101)
    q, k, v = (torch.randn(tokens, heads, dim, generator=g).bfloat16() for _ in range(3))
    cache = torch.zeros(1, 2, heads, ref.block_bytes(page, dim), dtype=torch.uint8)
    on_device = cache.to(DEV)
    slots = torch.tensor([15, 0, 7])
    ops.kv4_append(None, k.to(DEV), v.to(DEV), None, None, None, slots.to(DEV), None, on_device)
    ref.store(cache, slots, k.float(), v.float())
    assert_bit_equal(on_device, cache.to(DEV), "cache")
    weight = torch.rand(dim, generator=g).bfloat16()
    q_out, k_out = torch.empty_like(q, device=DEV), torch.empty_like(k, device=DEV)
    ops.qk_norm_rope(q.to(DEV), k.to(DEV), weight.to(DEV), weight.to(DEV), None, None, None, q_out, k_out)
    for got, x in ((q_out, q), (k_out, k)):
        want = x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight.double()
        # one rounding to BF16; FP32 before it: 64 squares and their sum, rsqrt within 2 units, three products: 2^-20 in all
        assert bool(((got.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all())
