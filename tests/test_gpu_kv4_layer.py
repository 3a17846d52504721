"""The attention half of a layer: every operator fed by the one before it, a prompt and then generated tokens, eager and
captured. Each stage is held to its own restatement on the stage's actual inputs."""
import pytest
import torch

from consumer_int8.attention import Kv4AttentionLayer, make_cache
from gpu_common import DEV, assert_bit_equal, device_status
from oracle import kv4_ref as ref
from oracle import w8a8_ref
from test_gpu_kv4_attention import tolerance
from test_gpu_kv4_rows import noise, table

pytestmark = pytest.mark.gpu


def weights(g, n, k):
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, generator=g)
    return w, (torch.rand(n, generator=g) * 0.01 / 127 + 0.002 / 127).bfloat16()


class Sequences:
    """Bookkeeping of two sequences' pages, in an order that is not the pages' own."""

    def __init__(self, batch, page, pages):
        self.page, self.lens = page, [0] * batch
        self.table = torch.full((batch, pages // batch), -1, dtype=torch.int32)
        self.free = [(7 * i + 3) % pages for i in range(pages)]

    def append(self, news):
        slots, positions = [], []
        for b, n in enumerate(news):
            for _ in range(n):
                at = self.lens[b]
                if at % self.page == 0:
                    self.table[b, at // self.page] = self.free.pop()
                slots.append(int(self.table[b, at // self.page]) * self.page + at % self.page)
                positions.append(at)
                self.lens[b] += 1
        starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
        return torch.tensor(positions), torch.tensor(slots), starts, torch.tensor(self.lens, dtype=torch.int32)


def check(layer, x, cache_before, cache, positions, slots, seqs, starts, lens, rotary):
    """Every stage of the last call against its restatement."""
    tokens, dim, hq, hk = x.shape[0], layer.dim, layer.q_heads, layer.kv_heads
    codes, scales = w8a8_ref.quantize_rows_ref(x.cpu())
    _, qkv = w8a8_ref.fused_channel_mm_ref(codes, layer.w_qkv.cpu(), scales, layer.qkv_scale.cpu(), fast=True)
    heads = qkv.view(tokens, -1, dim)
    q, k, v = heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:]
    got = layer.qkv[:tokens].cpu().view(tokens, -1, dim)
    got_q, got_k, got_v = got[:, :hq], got[:, hq:hq + hk], got[:, hq + hk:]
    assert_bit_equal(got_v, v, "values")
    cosine, sine = ref.angles(layer.cos_sin.cpu(), positions, None, tokens)
    want = cache_before.clone()
    if layer.q_weight is not None:
        for turned, plain, w in ((got_q, q, layer.q_weight), (got_k, k, layer.k_weight)):
            unit = ref.norm(plain, w.cpu(), layer.eps, layer.weight_offset)
            expected = ref.rotate(unit, cosine, sine, False)
            assert bool(((turned.double() - expected).abs() <= 2.0 ** -8 * expected.abs() + 1.01 * noise(unit, layer.cos_sin.cpu())).all())
        ref.store(want, slots, got_k.float(), v.float())
    else:
        assert_bit_equal(got_q, ref.rotate(q.float(), cosine, sine, False).bfloat16(), "rotated queries")
        assert_bit_equal(got_k, k, "keys are rotated on their way into the cache only")
        ref.store(want, slots, ref.rotate(k.float(), cosine, sine, False), v.float())
    assert_bit_equal(cache, want, "cache")
    attended, spread, reach = ref.attention(got_q, want, seqs.table, starts, lens, layer.scale)
    got = layer.attended[:tokens].cpu()
    assert bool(((got.double() - attended).abs() <= tolerance(attended, spread, reach)).all())
    codes, scales = w8a8_ref.quantize_rows_ref(got.view(tokens, -1))
    _, out = w8a8_ref.fused_channel_mm_ref(codes, layer.w_out.cpu(), scales, layer.out_scale.cpu(), fast=True)
    assert_bit_equal(layer.out[:tokens], out, "output projection")


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dim,hq,hk,rotary", [(128, 8, 2, 128), (256, 6, 1, 64), (64, 4, 4, 64)])
def test_prompt_then_generated_tokens(ops, norm, dim, hq, hk, rotary):
    g = torch.Generator().manual_seed(dim + norm)
    k, n = 256, 320
    w_qkv, s_qkv = weights(g, (hq + 2 * hk) * dim, k)
    w_out, s_out = weights(g, n, hq * dim)
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=g)).bfloat16().to(DEV) for _ in range(2)) if norm else (None, None)
    layer = Kv4AttentionLayer(*(t.to(DEV) for t in (w_qkv, s_qkv, w_out, s_out)), hq, hk, dim, 64, qw, kw, table(128, rotary).to(DEV), eps=1e-6)
    seqs = Sequences(2, 16, 12)
    cache = make_cache(12, hk, 16, dim, DEV)

    def step(news, call):
        before = cache.cpu()
        positions, slots, starts, lens = seqs.append(news)
        x = (torch.randn(sum(news), k, generator=g) * 2).bfloat16()
        call(x, positions, slots, starts, lens)
        check(layer, x, before, cache, positions, slots, seqs, starts, lens, rotary)

    step([33, 7], lambda x, p, s, st, ln: layer.forward(x.to(DEV), p.to(DEV), s.to(DEV), cache, seqs.table.to(DEV), st.to(DEV), ln.to(DEV)))
    # generated tokens: captured once, replayed with the next rows, positions, slots and lengths in place
    x_in = torch.zeros(2, k, dtype=torch.bfloat16, device=DEV)
    p_in, s_in = torch.zeros(2, dtype=torch.long, device=DEV), torch.full((2,), -1, device=DEV)
    t_in, st_in, l_in = seqs.table.to(DEV), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    layer.forward(x_in, p_in, s_in, cache, t_in, st_in, l_in)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(x_in, p_in, s_in, cache, t_in, st_in, l_in)

    def replay(x, p, s, st, ln):
        for to, t in ((x_in, x), (p_in, p), (s_in, s), (t_in, seqs.table), (l_in, ln)):
            to.copy_(t)
        graph.replay()

    for _ in range(3):
        step([1, 1], replay)
    assert device_status(ops) == 0


def test_two_layers_share_a_workspace_in_turn(ops):
    """One workspace serves call after call, of different shapes and kernels; the results do not depend on what ran before."""
    from test_gpu_kv4_attention import Case

    workspace = torch.zeros(ops.kv4_workspace_bytes(), dtype=torch.uint8, device=DEV)
    cases = [Case([(1, 3000)], 8, 2, 128, 64, seed=1), Case([(90, 700)], 8, 2, 64, 16, seed=2), Case([(1, 900), (1, 5)], 12, 1, 256, 32, seed=3)]

    def run(case):
        out = torch.empty_like(case.q, device=DEV)
        ops.kv4_attention(*case.device(), workspace, out, case.scale)
        return out

    first = [run(c) for c in cases]
    for _ in range(2):
        for c, want in zip(reversed(cases), reversed(first)):
            assert_bit_equal(run(c), want, "the same call again")
    assert int(workspace[:4096].count_nonzero()) == 0          # the counters are back at zero
