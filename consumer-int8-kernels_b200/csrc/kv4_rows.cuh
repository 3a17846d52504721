// The 4-bit key/value cache and the row operators in front of it: RMS norm and position rotation of the
// query and key heads, encoding into the cache, and reading it back.
//
// Cache block of (page, side, head): page_size rows of dim / 2 code bytes (byte j: component 2j in the low
// four bits, 2j + 1 in the high ones), then page_size pairs of BF16 numbers (scale, zero point). A code c
// stands for scale * (c - zero). Codes and pairs of a block are contiguous, so a run of tokens inside a page
// is two contiguous pieces and any page starts on a 16-byte boundary.
//
// A head of dim components is handled by dim / 8 neighbouring lanes of a warp, eight components (one
// 16-byte load) each, so a warp holds 4, 2 or 1 heads (dim 64, 128, 256) and all reductions are shuffles.
#pragma once
#include <cuda_bf16.h>
#include <cstdint>
#include "quantize.cuh"
#include "sm100_ptx.cuh"

namespace ci8 {

constexpr unsigned kStatusBadIndex = 8u;   // a position, slot or page number outside its table (the access was left out)

constexpr int kKv4Side = 2;                // keys, values
__host__ __device__ constexpr int64_t kv4_block_bytes(int page, int dim) {
  return static_cast<int64_t>(page) * (dim / 2 + 4);
}

struct Kv4RowParams {
  const uint16_t* q;         // [tokens, q_heads, dim], token stride in elements; null: no queries
  const uint16_t* k;
  const uint16_t* v;         // append only
  uint16_t* q_out;
  uint16_t* k_out;           // norm only
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  const uint16_t* q_weight;  // [dim] BF16 or null: no norm of the queries
  const uint16_t* k_weight;
  const float* cos_sin;      // [table_rows, rotary]: cosines, then sines; null: no rotation
  const int64_t* positions;  // [axes, tokens]
  const int32_t* axis_of;    // [rotary / 2] or null (one axis)
  const int64_t* slots;      // append only: page * page_size + row, negative: not stored
  uint8_t* cache;
  int64_t capacity;          // pages * page_size
  int table_rows, rotary, axes, adjacent;
  int tokens, q_heads, kv_heads, page_shift;
  int chunks;                // pieces that the heads of one token are cut into, one warp each
  float eps, weight_offset;
};

// Scale and zero point of one head whose smallest component is low <= 0 and largest high >= 0. The scale
// is rounded to BF16 before the codes are taken, so that the codes are the best ones for the scale that is
// kept; the zero point is a whole number, so the value 0 is kept exactly.
struct Kv4Code {
  float scale, inverse;
  int zero;
};
__device__ __forceinline__ Kv4Code kv4_code_of(float low, float high) {
  Kv4Code c;
  const float step = __fdiv_rn(__fsub_rn(high, low), 15.f);
  c.scale = fmaxf(__bfloat162float(__float2bfloat16_rn(step)), __bfloat162float(__float2bfloat16_rn(1e-20f)));
  c.inverse = __frcp_rn(c.scale);
  c.zero = min(15, __float2int_rn(__fdiv_rn(-low, c.scale)));
  return c;
}

// Eight components -> eight codes in one word, clamp(rint(x / scale) + zero, 0, 15) with the IEEE quotient:
// the quantizer's short path (a product with the reciprocal, proven equal away from ties) and its repair.
__device__ __forceinline__ uint32_t kv4_encode8(const float (&x)[8], const Kv4Code& code) {
  float worst = 0.f;
  int t[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 shifted = quantize_fast2(make_float2(x[j], x[j + 1]), make_float2(code.inverse, code.inverse), worst);
    t[j] = __float_as_int(shifted.x) - __float_as_int(kRoundMagic);
    t[j + 1] = __float_as_int(shifted.y) - __float_as_int(kRoundMagic);
  }
  if (!(fabsf(worst) < kTieGuard)) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!away_from_tie(x[j], code.inverse)) t[j] = __float2int_rn(__fdiv_rn(x[j], code.scale));
  }
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) word |= static_cast<uint32_t>(min(15, max(0, t[j] + code.zero))) << (4 * j);
  return word;
}

template <int kLanes>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int d = kLanes / 2; d; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
  x[4] = bf16_lo(w.z); x[5] = bf16_hi(w.z); x[6] = bf16_lo(w.w); x[7] = bf16_hi(w.w);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
}

// One warp takes a piece of one token's heads (queries, keys and, when appending, values, in that order): the
// token's angles stay in registers and up to kBatch heads per lane group are loaded before the first is used.
// Norm and rotation are FP32; products and sums of the rotation are rounded one by one (no FMA), so that what is
// encoded does not depend on how a compiler contracts them. Bound by memory: 4 bytes per component of the norm,
// 2 read + dim / 2 + 4 bytes per head written for what is appended.
template <int kDim, bool kNorm, bool kAppend>
__global__ void __launch_bounds__(256) kv4_rows_kernel(const Kv4RowParams p) {
  constexpr int kLanes = kDim / 8, kHeadsPerStep = 32 / kLanes, kBatch = 4;
  pdl_wait();
  const int warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int token = warp / p.chunks, chunk = warp % p.chunks;
  if (token >= p.tokens) return;      // whole warps
  const int lane = threadIdx.x % 32, l = lane % kLanes, sub = lane / kLanes;
  const int q_heads = p.q ? p.q_heads : 0;
  const int heads = q_heads + p.kv_heads * (kAppend ? 2 : 1);
  const int per_chunk = (heads + p.chunks - 1) / p.chunks;
  const int first = chunk * per_chunk, end = min(heads, first + per_chunk);

  // The token's angles: cosine and sine of each of this lane's components (adjacent pairs: of its four pairs).
  float cosine[8], sine[8];
  bool bad = false;
  const int half_lanes = p.rotary / 16;                 // lanes that hold the first components of the pairs
  const bool turns = p.cos_sin != nullptr && l < p.rotary / 8;
  if (p.cos_sin) {
    for (int a = 0; a < p.axes; ++a) {
      const int64_t place = p.positions[static_cast<int64_t>(a) * p.tokens + token];
      bad |= place < 0 || place >= p.table_rows;
    }
    const int pairs = p.rotary / 2;
    const int count = p.adjacent ? 4 : 8;
    const int f0 = p.adjacent ? 4 * l : 8 * (l < half_lanes ? l : l - half_lanes);
    if (turns && !bad) {
      if (!p.axis_of) {
        const float* row = p.cos_sin + p.positions[token] * p.rotary;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          if (j < count) {
            const float4 c = *reinterpret_cast<const float4*>(row + f0 + j);
            const float4 s = *reinterpret_cast<const float4*>(row + pairs + f0 + j);
            cosine[j] = c.x; cosine[j + 1] = c.y; cosine[j + 2] = c.z; cosine[j + 3] = c.w;
            sine[j] = s.x; sine[j + 1] = s.y; sine[j + 2] = s.z; sine[j + 3] = s.w;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < count) {
            const int axis = p.axis_of[f0 + j];
            if (axis < 0 || axis >= p.axes) {
              bad = true;
            } else {
              const float* row = p.cos_sin + p.positions[static_cast<int64_t>(axis) * p.tokens + token] * p.rotary;
              cosine[j] = row[f0 + j];
              sine[j] = row[pairs + f0 + j];
            }
          }
        }
      }
    }
  }
  bad = __any_sync(0xffffffffu, bad);

  int64_t slot = -1;
  if constexpr (kAppend) {
    slot = p.slots[token];
    if (slot >= p.capacity) {
      slot = -1;
      if (lane == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
    }
    if (bad) slot = -1;
  }
  if (bad && lane == 0) atomicOr(&g_ci8_status, kStatusBadIndex);

  for (int base = first; base < end; base += kBatch * kHeadsPerStep) {
    uint4 raw[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = base + i * kHeadsPerStep + sub;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (h < end) {
        const uint16_t* src = h < q_heads ? p.q + token * p.q_stride + static_cast<int64_t>(h) * kDim
                              : (!kAppend || h < q_heads + p.kv_heads)
                                  ? p.k + token * p.k_stride + static_cast<int64_t>(h - q_heads) * kDim
                                  : p.v + token * p.v_stride + static_cast<int64_t>(h - q_heads - p.kv_heads) * kDim;
        raw[i] = *reinterpret_cast<const uint4*>(src + 8 * l);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (base + i * kHeadsPerStep >= end) break;       // the same for the whole warp
      const int h = base + i * kHeadsPerStep + sub;
      const bool is_q = h < q_heads, is_v = kAppend && h >= q_heads + p.kv_heads;
      float x[8];
      unpack8(raw[i], x);
      if constexpr (kNorm) {
        float squares = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) squares = fmaf(x[j], x[j], squares);
        const float scale = rsqrtf(head_sum<kLanes>(squares) * (1.f / kDim) + p.eps);
        const uint16_t* weight = is_q ? p.q_weight : p.k_weight;
        if (weight) {
          float w[8];
          unpack8(*reinterpret_cast<const uint4*>(weight + 8 * l), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = x[j] * scale * (w[j] + p.weight_offset);
        }
      }
      if (p.cos_sin) {
        float y[8];
        if (p.adjacent) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            y[j] = __fsub_rn(__fmul_rn(x[j], cosine[j / 2]), __fmul_rn(x[j + 1], sine[j / 2]));
            y[j + 1] = __fadd_rn(__fmul_rn(x[j + 1], cosine[j / 2]), __fmul_rn(x[j], sine[j / 2]));
          }
        } else {
          const int partner = sub * kLanes + (turns ? (l < half_lanes ? l + half_lanes : l - half_lanes) : l);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float other = __shfl_sync(0xffffffffu, x[j], partner);
            const float kept = __fmul_rn(x[j], cosine[j]), mixed = __fmul_rn(other, sine[j]);
            y[j] = l < half_lanes ? __fsub_rn(kept, mixed) : __fadd_rn(kept, mixed);
          }
        }
        if (turns && !is_v) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = y[j];
        }
      }
      const bool real = h < end;
      if (!kAppend || is_q) {
        if (real) {
          uint4 w = pack8(x);
          if (bad) w = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);   // a position outside the table: NaN
          uint16_t* dst = is_q ? p.q_out + token * p.q_out_stride + static_cast<int64_t>(h) * kDim
                               : p.k_out + token * p.k_out_stride + static_cast<int64_t>(h - q_heads) * kDim;
          *reinterpret_cast<uint4*>(dst + 8 * l) = w;
        }
      }
      if constexpr (kAppend) {
        if (slot < 0 || base + i * kHeadsPerStep + kHeadsPerStep <= q_heads) continue;   // whole warps: nothing to encode here
        float low = 0.f, high = 0.f, worst = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) worst = max_abs_keep_nan(worst, x[j]);
        if (!(fabsf(worst) < 8.5e37f)) {
          // NaN counts as 0 and infinities as the largest value whose range still fits FP32, so that one such
          // component cannot spoil the scale and with it the whole head
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = x[j] != x[j] ? 0.f : fminf(fmaxf(x[j], -8.5e37f), 8.5e37f);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          low = fminf(low, x[j]);
          high = fmaxf(high, x[j]);
        }
#pragma unroll
        for (int d = kLanes / 2; d; d /= 2) {
          low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
          high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
        }
        const Kv4Code code = kv4_code_of(low, high);
        const uint32_t word = kv4_encode8(x, code);
        if (real && !is_q) {
          const int page = 1 << p.page_shift;
          const int64_t at = slot >> p.page_shift;
          const int row = static_cast<int>(slot & (page - 1));
          const int head = h - q_heads - (is_v ? p.kv_heads : 0);
          uint8_t* block = p.cache + ((at * kKv4Side + (is_v ? 1 : 0)) * p.kv_heads + head) * kv4_block_bytes(page, kDim);
          *reinterpret_cast<uint32_t*>(block + static_cast<int64_t>(row) * (kDim / 2) + 4 * l) = word;
          if (l == 0)
            *reinterpret_cast<uint32_t*>(block + static_cast<int64_t>(page) * (kDim / 2) + 4 * row) =
                pack2(code.scale, static_cast<float>(code.zero));
        }
      }
    }
  }
}

struct Kv4ReadParams {
  const uint8_t* cache;
  const int64_t* slots;
  uint16_t* k;               // [tokens, kv_heads, dim]
  uint16_t* v;
  int64_t capacity;
  int64_t rows;              // tokens * 2 * kv_heads
  int kv_heads, page_shift;
};

// One lane group takes a head of a token: eight codes (one word) per lane become eight BF16 values, one
// rounding each. Bound by memory (dim / 2 + 4 bytes read, 2 dim written per head).
template <int kDim>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
  constexpr int kLanes = kDim / 8, kBatch = 4;
  pdl_wait();
  const int page = 1 << p.page_shift;
  const int l = threadIdx.x % kLanes;
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (blockDim.x / kLanes);
  const int64_t group = static_cast<int64_t>(blockIdx.x) * (blockDim.x / kLanes) + threadIdx.x / kLanes;
  for (int64_t base = group; base < p.rows; base += groups * kBatch) {
    uint32_t word[kBatch], pair[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t row = base + i * groups;
      word[i] = 0;
      pair[i] = 0;                       // scale 0: the row reads as zeros
      if (row < p.rows) {
        const int64_t token = row / (2 * p.kv_heads);
        const int which = static_cast<int>(row % (2 * p.kv_heads));
        const int64_t slot = p.slots[token];
        if (slot >= p.capacity && l == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
        if (slot >= 0 && slot < p.capacity) {
          const uint8_t* block = p.cache + ((slot >> p.page_shift) * kKv4Side * p.kv_heads + which) * kv4_block_bytes(page, kDim);
          const int at = static_cast<int>(slot & (page - 1));
          word[i] = *reinterpret_cast<const uint32_t*>(block + static_cast<int64_t>(at) * (kDim / 2) + 4 * l);
          pair[i] = *reinterpret_cast<const uint32_t*>(block + static_cast<int64_t>(page) * (kDim / 2) + 4 * at);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t row = base + i * groups;
      if (row >= p.rows) break;
      const int64_t token = row / (2 * p.kv_heads);
      const int which = static_cast<int>(row % (2 * p.kv_heads));
      const float scale = bf16_lo(pair[i]), zero = bf16_hi(pair[i]);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = scale * (static_cast<float>((word[i] >> (4 * j)) & 15u) - zero);
      uint16_t* dst = which < p.kv_heads ? p.k + (token * p.kv_heads + which) * kDim
                                         : p.v + (token * p.kv_heads + which - p.kv_heads) * kDim;
      *reinterpret_cast<uint4*>(dst + 8 * l) = pack8(x);
    }
  }
}

}  // namespace ci8
