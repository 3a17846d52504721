"""The attention half of an INT8 layer over a key/value cache held in 4 bits.

    quantize_rows -> fused_channel_mm (QKV) -> qk_norm_rope -> kv4_append -> kv4_attention -> quantize_rows
    -> fused_channel_mm (output projection)

A clear and seven launches (eight or nine when prompts are among the rows) on the current stream over buffers allocated
once, so a call can be captured in a CUDA graph; lengths, pages, slots and positions are read on the device, and a
replay follows their values. The cache is a tensor of the caller's (:func:`make_cache`), as is the bookkeeping of its pages.
"""

from __future__ import annotations

import torch

PAGES = (16, 32, 64, 128, 256)
DIMS = (64, 128, 256)


def make_cache(pages: int, kv_heads: int, page: int, dim: int, device) -> torch.Tensor:
    """An empty cache: UINT8 [pages, 2 (keys, values), kv_heads, page * (dim / 2 + 4)]."""
    if page not in PAGES or dim not in DIMS or pages <= 0 or kv_heads <= 0:
        raise ValueError(f"pages of {PAGES} tokens and heads of {DIMS} components: got {page} and {dim}")
    return torch.zeros(pages, 2, kv_heads, page * (dim // 2 + 4), dtype=torch.uint8, device=device)


class Kv4AttentionLayer:
    """One layer's attention for up to ``max_tokens`` rows a call.

    ``w_qkv`` INT8 [(q_heads + 2 kv_heads) * dim, K] with BF16 channel scales, ``w_out`` INT8 [N, q_heads * dim] likewise;
    ``q_weight`` / ``k_weight`` BF16 [dim] norm weights or None (no norm), ``cos_sin`` FP32 [rows, rotary] or None (no
    rotation). Without norm weights the rotation of queries and keys is part of the append and one launch is saved.
    ``workspace`` (UINT8 [``kv4_workspace_bytes()``], zeroed once) may be shared by layers that run one after the other; by
    default the layer has its own.
    """

    def __init__(self, w_qkv, qkv_scale, w_out, out_scale, q_heads: int, kv_heads: int, dim: int, max_tokens: int,
                 q_weight=None, k_weight=None, cos_sin=None, eps: float = 1e-6, weight_offset: float = 0.0,
                 adjacent: bool = False, scale: float | None = None, workspace=None, operators=None):
        if operators is None:
            from . import ops as operators  # the compiled operators; there is no fallback

        if dim not in DIMS or kv_heads <= 0 or q_heads <= 0 or q_heads % kv_heads:
            raise ValueError("heads of 64, 128 or 256 components, query heads a multiple of the key heads")
        width = (q_heads + 2 * kv_heads) * dim
        if w_qkv.dtype != torch.int8 or w_qkv.shape[0] != width or qkv_scale.shape != (width,):
            raise ValueError(f"w_qkv must be INT8 [{width}, K] with one scale a channel")
        if w_out.dtype != torch.int8 or w_out.shape[1] != q_heads * dim or out_scale.shape != (w_out.shape[0],):
            raise ValueError(f"w_out must be INT8 [N, {q_heads * dim}] with one scale a channel")
        if (q_weight is None) != (k_weight is None):
            raise ValueError("norm weights come for queries and keys or for neither")
        if max_tokens <= 0:
            raise ValueError("max_tokens must be positive")
        self.ops = operators   # tests of the host logic inject a stand-in here
        self.w_qkv, self.qkv_scale, self.w_out, self.out_scale = w_qkv, qkv_scale, w_out, out_scale
        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, dim
        self.q_weight, self.k_weight, self.cos_sin = q_weight, k_weight, cos_sin
        self.eps, self.weight_offset, self.adjacent = eps, weight_offset, adjacent
        self.scale = dim ** -0.5 if scale is None else scale
        device = w_qkv.device
        bf16 = dict(dtype=torch.bfloat16, device=device)
        self.codes = torch.empty(max_tokens, w_qkv.shape[1], dtype=torch.int8, device=device)
        self.row_scales = torch.empty(max_tokens, dtype=torch.float32, device=device)
        self.qkv = torch.empty(max_tokens, width, **bf16)
        self.attended = torch.empty(max_tokens, q_heads, dim, **bf16)
        self.attended_codes = torch.empty(max_tokens, q_heads * dim, dtype=torch.int8, device=device)
        self.out = torch.empty(max_tokens, w_out.shape[0], **bf16)
        if workspace is None:
            workspace = torch.zeros(operators.kv4_workspace_bytes(), dtype=torch.uint8, device=device)
        elif workspace.dtype != torch.uint8 or workspace.device != device or workspace.numel() < operators.kv4_workspace_bytes():
            raise ValueError(f"workspace must be UINT8 [{operators.kv4_workspace_bytes()}] on {device}")
        self.workspace = workspace

    def forward(self, x, positions, slots, cache, block_table, q_starts, kv_lens, axis_of=None):
        """x BF16 [tokens, K] -> BF16 [tokens, N], valid until the next call. positions INT64 [tokens] or [axes, tokens],
        slots INT64 [tokens] (where each row's key and value go, negative: padding); block_table INT32 [batch, width],
        q_starts INT32 [batch + 1] and kv_lens INT32 [batch] as ``kv4_attention`` takes them: a sequence's length counts
        the rows of this call. Rows of no sequence (padding) come out as the product of zeros."""
        tokens = x.shape[0]
        if tokens > self.out.shape[0]:
            raise ValueError(f"{tokens} rows: the layer's buffers hold {self.out.shape[0]}")
        if tokens == 0:
            return self.out[:0]
        ops = self.ops
        codes, scales, qkv = self.codes[:tokens], self.row_scales[:tokens], self.qkv[:tokens]
        attended = self.attended[:tokens]
        # rows of no sequence are left alone by the attention: without this they would be an earlier call's. Ahead of the
        # launches, which follow one another without a gap
        attended.zero_()
        ops.quantize_rows(x, codes, scales)
        ops.fused_channel_mm(codes, self.w_qkv, scales, self.qkv_scale, qkv)
        heads = qkv.view(tokens, -1, self.dim)
        q, k, v = heads.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)     # views
        cos_sin, at = self.cos_sin, positions if self.cos_sin is not None else None
        axis_of = axis_of if self.cos_sin is not None else None
        if self.q_weight is not None:
            ops.qk_norm_rope(q, k, self.q_weight, self.k_weight, cos_sin, at, axis_of, q, k, self.eps, self.weight_offset,
                             self.adjacent)
            ops.kv4_append(None, k, v, None, None, None, slots, None, cache, False)
        elif cos_sin is not None:
            ops.kv4_append(q, k, v, cos_sin, at, axis_of, slots, q, cache, self.adjacent)
        else:
            ops.kv4_append(None, k, v, None, None, None, slots, None, cache, False)
        ops.kv4_attention(q, cache, block_table, q_starts, kv_lens, self.workspace, attended, self.scale)
        flat = self.attended_codes[:tokens]
        ops.quantize_rows(attended.view(tokens, -1), flat, scales)
        out = self.out[:tokens]
        ops.fused_channel_mm(flat, self.w_out, scales, self.out_scale, out)
        return out
