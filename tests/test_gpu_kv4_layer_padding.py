"""Rows of no sequence (padding of a captured step) in the attention layer: defined, whatever ran before."""
import pytest
import torch

from consumer_int8.attention import Kv4AttentionLayer, make_cache
from test_kv4_layer import forward, layer


def test_the_attention_starts_from_zeros():
    """Without a GPU: what the attention does not write is zeros when it is quantized, in the first call and in later ones."""
    made, ops = layer()
    for _ in range(2):
        made.attended.fill_(float("nan"))
        forward(made)
        assert not bool(made.attended[:3].any()) and not bool(made.attended[:3].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dim,hq,hk", [(128, 8, 2), (256, 6, 1), (64, 4, 4)])
def test_padding_rows_do_not_remember(ops, dim, hq, hk):
    """The same padded call gives the same bits after another one that used every row, and its padding rows project zeros."""
    from gpu_common import DEV, assert_bit_equal, device_status

    g = torch.Generator().manual_seed(dim)
    k, n, tokens = 256, 320, 12
    weights = []
    for rows, columns in (((hq + 2 * hk) * dim, k), (n, hq * dim)):
        weights += [torch.randint(-127, 128, (rows, columns), dtype=torch.int8, generator=g).to(DEV), (torch.rand(rows, generator=g) * 1e-4).bfloat16().to(DEV)]
    made = Kv4AttentionLayer(*weights, hq, hk, dim, 16)
    made.attended.fill_(float("nan"))
    cache = make_cache(4, hk, 16, dim, DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    x = (torch.randn(tokens, k, generator=g) * 2).bfloat16().to(DEV)
    x[7:] = 0
    positions = torch.zeros(tokens, dtype=torch.long, device=DEV)

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    def padded():
        slots = torch.tensor([0, 1, 2, 3, 4, 32, 33] + [-1] * 5, device=DEV)
        return made.forward(x, positions, slots, cache, table, ints(0, 5, 7), ints(5, 2)).clone()

    first = padded()
    slots = torch.cat([torch.arange(6), 32 + torch.arange(6)]).to(DEV)
    made.forward((torch.randn(tokens, k, generator=g) * 2).bfloat16().to(DEV), positions, slots, cache, table, ints(0, 6, 12), ints(6, 6))
    assert_bit_equal(padded(), first, "after another call")
    assert not bool(first[7:].isnan().any()) and not bool(first[7:].any()) and bool(first[:7].any())
    # a captured step, its padding rows changing from replay to replay
    starts, lens = ints(0, 6, 12), ints(6, 6)
    static = torch.cat([torch.arange(6), 32 + torch.arange(6)]).to(DEV)
    made.forward(x, positions, static, cache, table, starts, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = made.forward(x, positions, static, cache, table, starts, lens)
    graph.replay()
    static.copy_(torch.tensor([0, 1, 2, 3, 4, 32, 33] + [-1] * 5))
    starts.copy_(ints(0, 5, 7))
    lens.copy_(ints(5, 2))
    graph.replay()
    assert_bit_equal(out, first, "replayed")
    assert device_status(ops) == 0
