"""kv4_attention against the CPU restatement in 64 bits.

Bound of an output component y = sum of p_j v_j, with R = dim * 15 steps * max |q| * scale, the largest score of the row:
  one BF16 rounding of y: half a step, 2^-8 |y|;
  one rounding of every weight times its value's scale, to BF16 (prompts) or FP16 (generated tokens, 2^-11): 2^-8 of the sum
  of p_j |v_j|, FP32 sums and exponentials (2^-22) beside it: 5 % more;
  a score's error d, which moves every weight by at most a factor exp(2 d) (its own and the sum's). Generated tokens: a query
  component is a multiple of max |q| / 32639, off by at most 2^-16 of max |q| (half of 1 / 32639, rounded up); the sum of
  products with codes less zero points is exact, so d <= 2^-16 R and a few FP32 roundings, 2^-21 R. Prompts: the products
  are exact, accumulated over at most 16 steps with 2^-23 of the largest partial sum each: below 2^-18 R."""
import pytest
import torch

from gpu_common import DEV, assert_bit_equal, device_status, guarded
from oracle import kv4_ref as ref

pytestmark = pytest.mark.gpu


def tolerance(want, spread, reach):
    score = (2.0 ** -16 + 2.0 ** -21) * reach
    return 2.0 ** -8 * want.abs() + (1.05 * 2.0 ** -8 + torch.expm1(2 * score)) * spread


class Case:
    """Sequences (new rows, cached keys), their pages scattered over a cache whose unused rows are all ones (NaN scales)."""

    def __init__(self, sequences, q_heads, kv_heads, dim, page, seed=0, spare_rows=0, magnitude=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dim, self.kv_heads, self.page = dim, kv_heads, page
        need = [-(-max(keys, 0) // page) for _, keys in sequences]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g)
        self.cache = torch.full((pages, 2, kv_heads, ref.block_bytes(page, dim)), 0xFF, dtype=torch.uint8)
        width = max(need + [1]) + 1
        self.table = torch.full((len(sequences), width), -1, dtype=torch.int32)
        codes, pairs = ref.rows(self.cache, dim)
        done = 0
        for b, (_, keys) in enumerate(sequences):
            ids = order[done:done + need[b]]
            done += need[b]
            self.table[b, : need[b]] = ids
            if keys > 0:
                gain = 1 + 3 * (torch.rand(2, kv_heads, 1, dim, generator=g) < 0.03)
                x = torch.randn(2, kv_heads, keys, dim, generator=g) * gain * magnitude
                c, scale, zero = ref.encode(x.bfloat16().float())
                packed, pair = c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([scale, zero], dim=-1)
                at = torch.arange(keys)
                codes[ids[at // page], :, :, at % page] = packed.permute(2, 0, 1, 3)
                pairs[ids[at // page], :, :, at % page] = pair.permute(2, 0, 1, 3)
        rows = [n for n, _ in sequences]
        self.starts = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
        self.lens = torch.tensor([keys for _, keys in sequences], dtype=torch.int32)
        self.q = torch.randn(sum(rows) + spare_rows, q_heads, dim, generator=g).bfloat16()
        self.scale = dim ** -0.5

    def device(self):
        return [t.to(DEV) for t in (self.q, self.cache, self.table, self.starts, self.lens)]

    def want(self):
        return ref.attention(self.q, self.cache, self.table, self.starts, self.lens, self.scale)


@pytest.fixture(scope="module")
def workspace(ops):
    return torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV)


def run_and_check(ops, workspace, case, status=0):
    out, check = guarded(tuple(case.q.shape), torch.bfloat16, float("nan"))
    ops.kv4_attention(*case.device(), workspace, out, case.scale)
    want, spread, reach = case.want()
    rows = int(case.starts[-1])
    got = out.cpu()
    bad = (got[:rows].double() - want[:rows]).abs() > tolerance(want, spread, reach)[:rows]
    assert not bool(bad.any()) and not bool(got[:rows].isnan().any()), (int(bad.sum()), torch.nonzero(bad | got[:rows].isnan())[:4].tolist())
    assert bool(got[rows:].isnan().all()), "rows of no sequence were written"
    check()
    assert device_status(ops) == status
    return out


SINGLE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 31), (1, 33), (1, 64), (1, 100), (1, 129), (1, 300)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads,page", [(1, 1, 16), (6, 1, 32), (8, 2, 64), (10, 5, 16), (9, 1, 128), (32, 2, 16), (40, 2, 256)])
def test_single_tokens(ops, workspace, dim, q_heads, kv_heads, page):
    run_and_check(ops, workspace, Case(SINGLE, q_heads, kv_heads, dim, page, seed=dim + q_heads, spare_rows=2))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads,page", [(4, 4, 16), (6, 1, 64), (12, 4, 32), (17, 1, 16)])
def test_prompts(ops, workspace, dim, q_heads, kv_heads, page):
    """Whole prompts, chunks behind a prefix, single tokens and empty sequences in one call."""
    sequences = [(5, 5), (1, 40), (0, 10), (33, 33), (17, 200), (0, 0), (130, 130), (2, 129), (64, 65)]
    run_and_check(ops, workspace, Case(sequences, q_heads, kv_heads, dim, page, seed=dim + q_heads, spare_rows=3))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_that_see_nothing(ops, workspace, dim):
    """More new rows than cached keys, no keys at all, a negative length: zeros."""
    case = Case([(4, 2), (1, 0), (3, 3), (1, -5), (40, 7), (1, 1)], 6, 2, dim, 16, seed=3)
    out = run_and_check(ops, workspace, case)
    assert int((out[:2] != 0).sum()) == 0 and int((out[4] != 0).sum()) == 0
    single = Case([(1, 0), (1, 3), (1, -1)], 8, 2, dim, 16, seed=4)
    run_and_check(ops, workspace, single)


@pytest.mark.parametrize("dim,batch,keys,group", [(128, 1, 5000, 4), (256, 2, 3001, 6), (64, 3, 4111, 8), (128, 1, 2500, 16), (256, 1, 1500, 12)])
def test_long_histories_are_split_and_joined(ops, workspace, dim, batch, keys, group):
    case = Case([(1, keys - 7 * b) for b in range(batch)], 2 * group, 2, dim, 64, seed=keys)
    first = run_and_check(ops, workspace, case)
    for _ in range(3):                                                  # the same bits every time, whatever finishes first
        again = torch.empty_like(first)
        ops.kv4_attention(*case.device(), workspace, again, case.scale)
        assert_bit_equal(again, first, "repeated call")


@pytest.mark.parametrize("dim,sequences", [(128, [(3, 2000)]), (256, [(40, 1500), (2, 900)]), (64, [(200, 1300)])])
def test_few_rows_over_long_prefixes(ops, workspace, dim, sequences):
    run_and_check(ops, workspace, Case(sequences, 8, 2, dim, 16, seed=dim))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_mixed_magnitudes(ops, workspace, dim):
    """Large scores (one key takes all the weight), values far from 1, and scores that rise along the sequence so that
    the running maximum keeps moving."""
    case = Case([(1, 700), (1, 90)], 8, 2, dim, 32, seed=8, magnitude=6.0)
    run_and_check(ops, workspace, case)
    rising = Case([(1, 600), (40, 600)], 8, 2, dim, 32, seed=9)
    codes, pairs = ref.rows(rising.cache, dim)
    for b in range(2):
        for j in range(600):
            page = int(rising.table[b, j // 32])
            pairs[page, 0, :, j % 32, 0] *= 0.2 + 0.004 * j
            pairs[page, 1, :, j % 32, 0] *= 1e-3 if j % 50 == 0 else 1.0
    run_and_check(ops, workspace, rising)


def test_bad_page_numbers_are_not_followed(ops, workspace):
    case = Case([(1, 100), (1, 64), (20, 120)], 8, 2, 128, 16, seed=5)
    case.table[0, 2] = -1
    case.table[0, 5] = case.cache.shape[0]
    case.table[1, :4] = 2 ** 31 - 1                                     # a sequence without one good page
    case.table[2, 0] = -2 ** 31
    run_and_check(ops, workspace, case, status=8)


def test_lengths_beyond_the_table_are_cut(ops, workspace):
    case = Case([(1, 64), (2, 32)], 4, 2, 128, 16, seed=6)
    case.table = case.table[:, :4].contiguous()                         # room for 64 keys
    case.lens = torch.tensor([1000, 32], dtype=torch.int32)
    run_and_check(ops, workspace, case)


def test_strided_queries_and_other_streams(ops, workspace):
    case = Case([(1, 77), (1, 300), (1, 5)], 12, 4, 128, 16, seed=7)
    want = run_and_check(ops, workspace, case)
    q, cache, table, starts, lens = case.device()
    wide = torch.zeros(3, 12 + 8, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 4:16] = q
    out = torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.kv4_attention(wide[:, 4:16], cache, table, starts, lens, workspace, out, case.scale)
    stream.synchronize()
    assert_bit_equal(out, want, "a slice of a wider buffer")


def test_captured_call_follows_lengths_and_tables(ops, workspace):
    """One capture serves growing sequences: lengths, tables and queries are read when it is replayed."""
    case = Case([(1, 500), (1, 1200), (1, 3)], 8, 2, 128, 16, seed=11)
    q, cache, table, starts, lens = case.device()
    out = torch.empty_like(q)
    ops.kv4_attention(q, cache, table, starts, lens, workspace, out, case.scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv4_attention(q, cache, table, starts, lens, workspace, out, case.scale)
    for short in ([500, 1200, 3], [37, 1, 2], [0, 999, 1]):
        case.lens = torch.tensor(short, dtype=torch.int32)
        lens.copy_(case.lens)
        out.fill_(float("nan"))
        graph.replay()
        want, spread, reach = case.want()
        assert bool(((out.cpu().double() - want).abs() <= tolerance(want, spread, reach)).all())


def test_one_nan_query_stays_its_own(ops, workspace):
    for sequences in ([(1, 50), (1, 300)], [(20, 50), (9, 300)]):
        case = Case(sequences, 8, 2, 128, 16, seed=12)
        want = run_and_check(ops, workspace, case)
        case.q[0, 3, 5] = float("nan")
        q, cache, table, starts, lens = case.device()
        out = torch.empty_like(q)
        ops.kv4_attention(q, cache, table, starts, lens, workspace, out, case.scale)
        assert bool(out[0, 3].isnan().all())
        out[0, 3] = want[0, 3]
        assert_bit_equal(out, want, "the other rows")


def test_offsets_beyond_32_bits(ops, workspace):
    """A cache of 5 GB whose used pages lie at its end."""
    dim, page, kv_heads = 128, 256, 8
    per_page = 2 * kv_heads * ref.block_bytes(page, dim)
    pages = 5 * 2 ** 30 // per_page
    case = Case([(1, 700), (30, 300)], 16, kv_heads, dim, page, seed=13)
    cache = torch.empty(pages, 2, kv_heads, ref.block_bytes(page, dim), dtype=torch.uint8, device=DEV)
    small = case.cache.shape[0]
    cache[pages - small:] = case.cache.to(DEV)
    shifted = torch.where(case.table >= 0, case.table + pages - small, -1).int()
    q, _, _, starts, lens = case.device()
    out = torch.empty_like(q)
    ops.kv4_attention(q, cache, shifted.to(DEV), starts, lens, workspace, out, case.scale)
    want, spread, reach = case.want()
    assert bool(((out.cpu().double() - want).abs() <= tolerance(want, spread, reach)).all())
    slots = torch.tensor([(pages - 1) * page + 3, (pages - 2) * page], device=DEV)
    k = torch.randn(2, kv_heads, dim, device=DEV).bfloat16()
    ops.kv4_append(None, k, k, None, None, None, slots, None, cache)
    k_out, v_out = torch.empty_like(k), torch.empty_like(k)
    ops.kv4_read(cache, slots, k_out, v_out)
    assert_bit_equal(k_out, v_out, "read back")
    assert float((k_out - k).abs().max()) < 0.6


def test_attention_refuses(ops, workspace):
    case = Case([(1, 20)], 8, 2, 128, 16)
    q, cache, table, starts, lens = case.device()
    out = torch.empty_like(q)

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            ops.kv4_attention(*args)

    refused("multiple of the cache's heads", q[:, :7], cache, table, starts, lens, workspace, out[:, :7].contiguous(), 0.1)
    refused("Wrong output", q, cache, table, starts, lens, workspace, out[:, :4].contiguous(), 0.1)
    refused("workspace", q, cache, table, starts, lens, workspace[:-16], out, 0.1)
    refused("dtype", q, cache, table.long(), starts, lens, workspace, out, 0.1)
    refused("block_table", q, cache, table, starts[:1], lens, workspace, out, 0.1)
    refused("UINT8 cache", q, cache[..., :-1].contiguous(), table, starts, lens, workspace, out, 0.1)
    refused("softmax scale", q, cache, table, starts, lens, workspace, out, 0.0)
    refused("softmax scale", q, cache, table, starts, lens, workspace, out, float("nan"))
    refused("must not overlap", q, cache, table, starts, lens, workspace, q, 0.1)
    refused("same CUDA device", q, cache, table.cpu(), starts, lens, workspace, out, 0.1)
    empty = q[:0].contiguous()
    ops.kv4_attention(empty, cache, table, torch.zeros(2, dtype=torch.int32, device=DEV), lens, workspace, empty.clone(), 0.1)
    ops.kv4_attention(q, cache, table[:0], starts[:1], lens[:0], workspace, out.fill_(7), 0.1)     # no sequences: out is left alone
    assert bool((out == 7).all())
