"""The 4-bit cache operators without a GPU: schemas, tracing, and the C entries' refusals (before any launch)."""
import ctypes

import torch

P = ctypes.c_void_p
L = ctypes.c_longlong
F = ctypes.c_float


def test_row_entries_refuse(ops):
    lib, one, odd, null = ops.libci8, P(16), P(24), P(0)

    def rope(q=one, qs=1024, k=one, ks=256, qw=one, kw=one, table=one, rows=8, rotary=64, positions=one, axes=1, axis_of=null, qo=one,
             qos=1024, ko=one, kos=256, tokens=4, q_heads=8, kv_heads=2, dim=128, eps=1e-6):
        return lib.ci8_qk_norm_rope(q, L(qs), k, L(ks), qw, kw, table, rows, rotary, positions, axes, axis_of, qo, L(qos), ko, L(kos),
                                    tokens, q_heads, kv_heads, dim, F(eps), F(0), 0, null)

    assert rope(tokens=0) == 0
    for bad in (dict(dim=96), dict(q_heads=0), dict(kv_heads=1025), dict(tokens=-1), dict(q=null), dict(q=odd), dict(qs=1020), dict(qs=512),
                dict(ko=null), dict(kos=128), dict(qw=odd), dict(rotary=24), dict(rotary=256), dict(rotary=0), dict(rows=0), dict(axes=0),
                dict(axes=5, axis_of=one), dict(axes=2), dict(positions=null), dict(positions=P(20)), dict(table=P(20)), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert rope(**bad) == 1, bad

    def append(q=one, k=one, v=one, table=one, rotary=64, positions=one, axes=1, slots=one, qo=one, cache=one, pages=4, page=16, tokens=4,
               q_heads=8, kv_heads=2, dim=128, ks=256):
        return lib.ci8_kv4_append(q, L(1024), k, L(ks), v, L(256), table, 8, rotary, positions, axes, null, slots, qo, L(1024), cache, pages,
                                  page, tokens, q_heads, kv_heads, dim, 0, null)

    assert append(tokens=0) == 0
    for bad in (dict(page=8), dict(page=24), dict(page=512), dict(page=0), dict(pages=-1), dict(dim=32), dict(k=null), dict(v=odd), dict(ks=255),
                dict(slots=null), dict(slots=P(12)), dict(cache=null), dict(cache=odd), dict(qo=null), dict(q_heads=0), dict(kv_heads=0),
                dict(rotary=8), dict(axes=3)):
        assert append(**bad) == 1, bad

    def read(cache=one, slots=one, k=one, v=one, pages=4, page=16, tokens=4, kv_heads=2, dim=128):
        return lib.ci8_kv4_read(cache, slots, k, v, pages, page, tokens, kv_heads, dim, null)

    assert read(tokens=0) == 0
    for bad in (dict(cache=null), dict(cache=odd), dict(slots=null), dict(k=null), dict(v=odd), dict(page=17), dict(dim=512), dict(tokens=-2),
                dict(kv_heads=0)):
        assert read(**bad) == 1, bad


def test_attention_entry_refuses(ops):
    lib, one, odd, null = ops.libci8, P(16), P(24), P(0)

    def attend(q=one, qs=1024, cache=one, table=one, starts=one, lens=one, workspace=one, out=one, tokens=4, batch=2, width=3, pages=9, page=16,
               q_heads=8, kv_heads=2, dim=128, scale=0.1):
        return lib.ci8_kv4_attention(q, L(qs), cache, table, starts, lens, workspace, out, tokens, batch, width, pages, page, q_heads, kv_heads,
                                     dim, F(scale), null)

    assert attend(tokens=0) == 0 and attend(batch=0) == 0
    for bad in (dict(q=null), dict(q=odd), dict(qs=1000), dict(cache=null), dict(cache=odd), dict(table=null), dict(starts=null), dict(lens=P(6)),
                dict(workspace=null), dict(workspace=odd), dict(out=null), dict(tokens=-1), dict(batch=-1), dict(width=-1), dict(page=48),
                dict(width=2 ** 27, page=16), dict(q_heads=9), dict(kv_heads=0), dict(q_heads=1026), dict(dim=100), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan"))):
        assert attend(**bad) == 1, bad


def test_schemas_and_tracing(ops):
    from torch._subclasses.fake_tensor import FakeTensorMode

    schemas = {name: str(getattr(ops, name).default._schema) for name in ("qk_norm_rope", "kv4_append", "kv4_read", "kv4_attention")}
    assert "Tensor(a!)? q_out, Tensor(b!) cache" in schemas["kv4_append"]
    assert schemas["kv4_read"] == "consumer_int8::kv4_read(Tensor cache, Tensor slots, Tensor(a!) k, Tensor(b!) v) -> ()"
    assert ops.kv4_block_bytes(16, 128) == 16 * 68 and ops.kv4_workspace_bytes() % 16 == 0
    with FakeTensorMode():
        q = torch.empty(4, 8, 128, dtype=torch.bfloat16, device="cuda")
        k = torch.empty(4, 2, 128, dtype=torch.bfloat16, device="cuda")
        slots = torch.empty(4, dtype=torch.long, device="cuda")
        cache = torch.empty(2, 2, 2, ops.kv4_block_bytes(16, 128), dtype=torch.uint8, device="cuda")
        assert ops.qk_norm_rope(q, k, None, None, None, None, None, q, k) is None
        assert ops.kv4_append(None, k, k, None, None, None, slots, None, cache) is None
        assert ops.kv4_read(cache, slots, k, k) is None
        i32 = torch.empty(3, dtype=torch.int32, device="cuda")
        assert ops.kv4_attention(q, cache, i32[None, :2], i32, i32[:2], cache.view(-1), q, 0.1) is None
