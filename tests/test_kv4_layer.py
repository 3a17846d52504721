"""The attention layer's host logic with a stand-in for the operators (no GPU): which operators are called on which
slices, and what is refused."""
import pytest
import torch

from consumer_int8.attention import Kv4AttentionLayer, make_cache


class Recorder:
    def __init__(self):
        self.calls = []

    def kv4_workspace_bytes(self):
        return 64

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args))


def layer(norm=True, rotary=32, **changes):
    ops = Recorder()
    weight = torch.ones(64, dtype=torch.bfloat16) if norm else None
    args = dict(w_qkv=torch.zeros(8 * 64, 96, dtype=torch.int8), qkv_scale=torch.ones(8 * 64), w_out=torch.zeros(80, 4 * 64, dtype=torch.int8),
                out_scale=torch.ones(80), q_heads=4, kv_heads=2, dim=64, max_tokens=10, q_weight=weight, k_weight=weight,
                cos_sin=torch.zeros(16, rotary) if rotary else None, operators=ops)
    args.update(changes)
    return Kv4AttentionLayer(**args), ops


def forward(made, tokens=3):
    ints = torch.zeros(4, dtype=torch.int32)
    cache = make_cache(2, 2, 16, 64, "cpu")
    return made.forward(torch.zeros(tokens, 96, dtype=torch.bfloat16), torch.zeros(tokens, dtype=torch.long),
                        torch.zeros(tokens, dtype=torch.long), cache, ints.view(1, 4), ints[:2], ints[:1])


@pytest.mark.parametrize("norm,rotary,names", [
    (True, 32, ["quantize_rows", "fused_channel_mm", "qk_norm_rope", "kv4_append", "kv4_attention", "quantize_rows", "fused_channel_mm"]),
    (True, 0, ["quantize_rows", "fused_channel_mm", "qk_norm_rope", "kv4_append", "kv4_attention", "quantize_rows", "fused_channel_mm"]),
    (False, 32, ["quantize_rows", "fused_channel_mm", "kv4_append", "kv4_attention", "quantize_rows", "fused_channel_mm"]),
    (False, 0, ["quantize_rows", "fused_channel_mm", "kv4_append", "kv4_attention", "quantize_rows", "fused_channel_mm"])])
def test_operators_called(norm, rotary, names):
    made, ops = layer(norm, rotary)
    out = forward(made)
    assert [n for n, _ in ops.calls] == names and out.shape == (3, 80) and out.data_ptr() == made.out.data_ptr()
    calls = dict(ops.calls)
    q, k, v = calls["kv4_append"][0], calls["kv4_append"][1], calls["kv4_append"][2]
    base = made.qkv.data_ptr()
    assert k.data_ptr() == base + 2 * 4 * 64 and v.data_ptr() == base + 2 * 6 * 64 and k.shape == v.shape == (3, 2, 64)
    assert (q is not None) == (not norm and rotary > 0)
    assert (calls["kv4_append"][3] is not None) == (not norm and rotary > 0)
    assert calls["kv4_attention"][0].data_ptr() == base and calls["kv4_attention"][7] == 64 ** -0.5


def test_refusals():
    for changes, match in ((dict(dim=96), "components"), (dict(q_heads=3), "multiple"), (dict(w_qkv=torch.zeros(8 * 64, 96)), "w_qkv"),
                           (dict(qkv_scale=torch.ones(3)), "w_qkv"), (dict(w_out=torch.zeros(80, 8, dtype=torch.int8)), "w_out"),
                           (dict(k_weight=None), "norm weights"), (dict(max_tokens=0), "max_tokens")):
        with pytest.raises(ValueError, match=match):
            layer(**changes)
    made, ops = layer()
    with pytest.raises(ValueError, match="buffers hold 10"):
        forward(made, 11)
    assert forward(made, 0).shape == (0, 80) and not ops.calls
    for bad in (dict(page=24), dict(dim=32), dict(pages=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            make_cache(**{**dict(pages=1, kv_heads=1, page=16, dim=64, device="cpu"), **bad})


def test_layers_share_a_workspace():
    shared = torch.zeros(64, dtype=torch.uint8)
    first, ops = layer(workspace=shared)
    second, _ = layer(workspace=shared)
    assert first.workspace.data_ptr() == second.workspace.data_ptr() == shared.data_ptr()
    forward(first)
    assert dict(ops.calls)["kv4_attention"][5] is shared
    for bad in (torch.zeros(63, dtype=torch.uint8), torch.zeros(64, dtype=torch.int8), torch.zeros(64, dtype=torch.uint8, device="meta")):
        with pytest.raises(ValueError, match="workspace"):
            layer(workspace=bad)
