"""AOT operators of the W8A8 linear path. Buffers belong to the caller; importing never compiles.

Same surface as the reference's ``consumer_int8.ops`` for this path
(src/consumer_int8/ops.py:20-34): every handle is ``torch.ops.consumer_int8.<name>``, writes
into caller-allocated outputs, returns ``None`` and can be captured in a CUDA graph.

  quantize_rows(input BF16[M,K], codes INT8[M,K], scales FP32[M])
  silu_mul(input BF16[M,2K] = gate|up, out BF16[M,K])                 SwiGLU feeding the down projection
  silu_mul_quantize(input BF16[M,2K], codes INT8[M,K], scales FP32[M])  = quantize_rows(silu_mul(input))
  quantize_grouped4096(input BF16[M,G,4096], codes INT8[G,M,4096], scales FP32[G,M])
      (alias: quantize_grouped_rows, the name the reference's README uses)
  fused_channel_mm(a INT8[M,K], w INT8[N,K], a_scale FP32[M], w_scale BF16[N], out BF16[M,N], schedule=0)
  cutlass_channel_mm(a, w, a_scale, w_scale, workspace INT32[M,N], out)
  channel_mm(a INT8[M,K], w UINT8[N,K] = code+128, a_scale, w_scale, out)
  unpack_allspark(packed UINT8[ceil(N/32)*32,K], packed_scales BF16[...], weight INT8[N,K], scales BF16[N])
  channel_gemv(x BF16[M,K], w INT8[N,K], scale BF16[N], out BF16[M,N])        W8A16, M <= 16
  grouped_channel_mm(codes INT8[G,M,4096], w INT8[N,G*4096], scales FP32[G,M], w_scale, out)
  grouped_channel_mm_ws(codes, w, scales, w_scale, workspace UINT8[grouped_workspace_bytes(M,N,G)] zeroed once, out)
      the same bits; the lent workspace lets the tiles of a thin last wave run split along the groups
  dynamic_channel_mm(x BF16[M,K], w, w_scale, codes, scales, out)     quantize_rows + fused_channel_mm in one call
  gate_up_silu_mm(a, w INT8[N,K] gate/up interleaved by 128, a_scale, w_scale, out BF16[M,N/2])  GEMM + SwiGLU
      additive: the grouped-scale GEMM in one launch
  fused_channel_mm_gather(a, w INT8[N/G,K], a_scale, w_scale BF16[N/G], gathered BF16[G,M,N/G],
                          peer_ptrs CPU INT64[G], rank, schedule=0)
      additive: an output-channel shard whose epilogue stores into every rank's gathered buffer
  fused_channel_mm_gather_sync(a, w, a_scale, w_scale, gathered, peer_ptrs, signal_ptrs CPU INT64[G],
                               state INT64[4], rank, schedule=0)
      the same, ending with a cross-GPU rendezvous inside the kernel (no collective has to follow)
  peer_rendezvous(signal_ptrs CPU INT64[G], state INT64[2], rank)
      that rendezvous as a one-thread kernel of its own, to follow fused_channel_mm_gather

The attention side of the layer, over a key/value cache held in 4 bits (UINT8 [pages, 2, kv_heads, kv4_block_bytes(page,
dim)]: rows of 4-bit codes and a BF16 scale and zero point for each token and head; heads tensors are BF16 [tokens, heads,
dim], dim 64, 128 or 256, and may be slices of one projection's output):

  qk_norm_rope(q, k, q_weight?, k_weight?, cos_sin?, positions?, axis_of?, q_out, k_out, eps, weight_offset, adjacent)
      RMS norm of every query and key head and the rotation to its position (one to four position axes), one launch
  kv4_append(q?, k, v, cos_sin?, positions?, axis_of?, slots INT64[T], q_out?, cache, adjacent)
      keys rotated on the way, keys and values encoded into the cache; the queries rotated in the same launch
  kv4_read(cache, slots INT64[T], k, v)     cache rows back as the BF16 values they stand for
  kv4_attention(q, cache, block_table INT32[B,W], q_starts INT32[B+1], kv_lens INT32[B], workspace, out, scale)
      causal attention of single tokens and prompts; workspace UINT8[kv4_workspace_bytes()] zeroed once

There is no CPU implementation and no fallback: if the compiled extension is missing the
import fails, and the operators only have a CUDA kernel registered.
"""

import ctypes
from pathlib import Path

import torch

_HERE = Path(__file__).resolve().parent
if not (_HERE / "libci8.so").exists() or not (_HERE / "_C.so").exists():
    raise ImportError(
        "consumer_int8: the compiled extension (libci8.so, _C.so) is missing next to ops.py; "
        "build it with `python build.py` in the package directory. There is no fallback path."
    )
# The kernels' C ABI first (the operator library links against it), then the operators.
libci8 = ctypes.CDLL(str(_HERE / "libci8.so"), mode=ctypes.RTLD_GLOBAL)
from . import _C  # noqa: E402,F401

silu_mul = torch.ops.consumer_int8.silu_mul
silu_mul_quantize = torch.ops.consumer_int8.silu_mul_quantize
quantize_rows = torch.ops.consumer_int8.quantize_rows
quantize_grouped4096 = torch.ops.consumer_int8.quantize_grouped4096
quantize_grouped_rows = quantize_grouped4096
channel_mm = torch.ops.consumer_int8.channel_mm
channel_gemv = torch.ops.consumer_int8.channel_gemv
unpack_allspark = torch.ops.consumer_int8.unpack_allspark
cutlass_channel_mm = torch.ops.consumer_int8.cutlass_channel_mm
fused_channel_mm = torch.ops.consumer_int8.fused_channel_mm
grouped_channel_mm = torch.ops.consumer_int8.grouped_channel_mm
grouped_channel_mm_ws = torch.ops.consumer_int8.grouped_channel_mm_ws
gate_up_silu_mm = torch.ops.consumer_int8.gate_up_silu_mm
dynamic_channel_mm = torch.ops.consumer_int8.dynamic_channel_mm
fused_channel_mm_gather = torch.ops.consumer_int8.fused_channel_mm_gather
fused_channel_mm_gather_sync = torch.ops.consumer_int8.fused_channel_mm_gather_sync
peer_rendezvous = torch.ops.consumer_int8.peer_rendezvous
qk_norm_rope = torch.ops.consumer_int8.qk_norm_rope
kv4_append = torch.ops.consumer_int8.kv4_append
kv4_read = torch.ops.consumer_int8.kv4_read
kv4_attention = torch.ops.consumer_int8.kv4_attention


@torch.library.register_fake("consumer_int8::fused_channel_mm")
def _fused_channel_mm_fake(a, w, a_scale, w_scale, out, schedule=0):
    return None


@torch.library.register_fake("consumer_int8::silu_mul")
def _silu_mul_fake(input, out):
    return None


@torch.library.register_fake("consumer_int8::silu_mul_quantize")
def _silu_mul_quantize_fake(input, codes, scales):
    return None


@torch.library.register_fake("consumer_int8::quantize_rows")
def _quantize_rows_fake(input, codes, scales):
    return None


@torch.library.register_fake("consumer_int8::quantize_grouped4096")
def _quantize_grouped4096_fake(input, codes, scales):
    return None


@torch.library.register_fake("consumer_int8::channel_mm")
def _channel_mm_fake(a, w, a_scale, w_scale, out):
    return None


@torch.library.register_fake("consumer_int8::unpack_allspark")
def _unpack_allspark_fake(packed, packed_scales, weight, scales):
    return None


@torch.library.register_fake("consumer_int8::channel_gemv")
def _channel_gemv_fake(x, w, scale, out):
    return None


@torch.library.register_fake("consumer_int8::cutlass_channel_mm")
def _cutlass_channel_mm_fake(a, w, a_scale, w_scale, workspace, out):
    return None


@torch.library.register_fake("consumer_int8::fused_channel_mm_gather")
def _fused_channel_mm_gather_fake(a, w, a_scale, w_scale, gathered, peer_ptrs, rank, schedule=0):
    return None


@torch.library.register_fake("consumer_int8::fused_channel_mm_gather_sync")
def _fused_channel_mm_gather_sync_fake(a, w, a_scale, w_scale, gathered, peer_ptrs, signal_ptrs, state, rank, schedule=0):
    return None


@torch.library.register_fake("consumer_int8::peer_rendezvous")
def _peer_rendezvous_fake(signal_ptrs, state, rank):
    return None


@torch.library.register_fake("consumer_int8::dynamic_channel_mm")
def _dynamic_channel_mm_fake(x, w, w_scale, codes, scales, out):
    return None


@torch.library.register_fake("consumer_int8::gate_up_silu_mm")
def _gate_up_silu_mm_fake(a, w, a_scale, w_scale, out):
    return None


@torch.library.register_fake("consumer_int8::grouped_channel_mm_ws")
def _grouped_channel_mm_ws_fake(codes, w, scales, w_scale, workspace, out):
    return None


def grouped_workspace_bytes(m: int, n: int, groups: int) -> int:
    """Bytes of (zero-initialised, UINT8) workspace with which ``grouped_channel_mm_ws`` splits the tiles of
    a thin last wave along the groups on the current device; 0 when the shape gains nothing from it."""
    libci8.ci8_grouped_workspace_bytes.restype = ctypes.c_longlong
    return int(libci8.ci8_grouped_workspace_bytes(m, n, groups))


@torch.library.register_fake("consumer_int8::grouped_channel_mm")
def _grouped_channel_mm_fake(codes, w, scales, w_scale, out):
    return None


@torch.library.register_fake("consumer_int8::qk_norm_rope")
def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos_sin, positions, axis_of, q_out, k_out, eps=1e-6, weight_offset=0.0, adjacent=False):
    return None


@torch.library.register_fake("consumer_int8::kv4_append")
def _kv4_append_fake(q, k, v, cos_sin, positions, axis_of, slots, q_out, cache, adjacent=False):
    return None


@torch.library.register_fake("consumer_int8::kv4_read")
def _kv4_read_fake(cache, slots, k, v):
    return None


@torch.library.register_fake("consumer_int8::kv4_attention")
def _kv4_attention_fake(q, cache, block_table, q_starts, kv_lens, workspace, out, scale):
    return None


def kv4_block_bytes(page: int, dim: int) -> int:
    """Last dimension of the 4-bit cache: the bytes that a page of one head's keys (or values) takes."""
    return page * (dim // 2 + 4)


def kv4_workspace_bytes() -> int:
    """Bytes of (zero-initialised, UINT8) workspace that ``kv4_attention`` asks for, whatever the shapes. Calls that may
    run at the same time need one each."""
    libci8.ci8_kv4_workspace_bytes.restype = ctypes.c_longlong
    return int(libci8.ci8_kv4_workspace_bytes())
