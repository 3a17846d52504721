// The 4-bit key/value cache and the row operators in front of it: RMS norm and position rotation of the
// query and key heads, encoding into the cache, and reading it back.
//
// Cache block of (page, side, head): page_size rows of dim / 2 code bytes (byte j: component 2j in the low
// four bits, 2j + 1 in the high ones), then page_size pairs of BF16 numbers (scale, zero point). A code c
// stands for scale * (c - zero). Codes and pairs of a block are contiguous, so a run of tokens inside a page
// is two contiguous pieces and any page starts on a 16-byte boundary.
//
// A head of dim components is handled by dim / 8 neighbouring lanes of a warp, eight components each (one
// 16-byte load, or two of 8 bytes where the lane holds both runs that a rotation pairs), so a warp holds 4, 2
// or 1 heads (dim 64, 128, 256) and all reductions are shuffles.
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
  int q_chunks, kv_chunks;   // pieces that the heads of one token are cut into, one warp each: q_chunks of queries, then
                             // kv_chunks of keys (and as many of values when appending)
  float eps, weight_offset;
};

// Scale and zero point of one head whose smallest component is low <= 0 and largest high >= 0. The scale is rounded to
// BF16 before the codes are taken, so that the codes are the best ones for the scale that is kept; the zero point is a
// whole number, so the value 0 is kept exactly.
struct Kv4Code {
  float scale, inverse, zero;   // inverse: an approximation, for the short path below
};
__device__ __forceinline__ float approximate_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ Kv4Code kv4_code_of(float low, float high) {
  Kv4Code c;
  const float step = __fmul_rn(__fsub_rn(high, low), 1.f / 15.f);
  c.scale = fmaxf(__bfloat162float(__float2bfloat16_rn(step)), __bfloat162float(__float2bfloat16_rn(1e-20f)));
  c.inverse = approximate_reciprocal(c.scale);
  float rounded = __fsub_rn(__fmaf_rn(-low, c.inverse, kRoundMagic), kRoundMagic);
  if (!away_from_tie(-low, c.inverse)) rounded = rintf(__fdiv_rn(-low, c.scale));
  c.zero = fminf(15.f, rounded);
  return c;
}

// Eight components -> eight codes in one word, clamp(rint(x / scale) + zero, 0, 15) with the IEEE quotient: the
// quantizer's short path (a product with the reciprocal, equal away from ties: with a reciprocal that is off by one unit
// in the last place the product is off by less than 17 * 2^-22, well inside the guard band) and its repair. The zero
// point goes into the constant that rounds (rint(q) + zero = rint(q + zero) but for ties, which are repaired), and the
// codes are put together as a sum of t * 16^j, whose constant part is taken off at the end.
__device__ __forceinline__ uint32_t kv4_encode8(const float2 (&x)[4], const Kv4Code& code) {
  const float2 inverse = make_float2(code.inverse, code.inverse), magic = make_float2(kRoundMagic, kRoundMagic);
  const float2 offset = make_float2(code.zero, code.zero);
  float worst = 0.f;
  float t[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 shifted = quantize_fast2(x[j], inverse, worst);
    const float2 moved = __fadd2_rn(shifted, offset);    // exact
    t[2 * j] = moved.x;
    t[2 * j + 1] = moved.y;
  }
  if (!(fabsf(worst) < kTieGuard)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = j % 2 ? x[j / 2].y : x[j / 2].x;
      if (!away_from_tie(v, code.inverse)) t[j] = kRoundMagic + (rintf(__fdiv_rn(v, code.scale)) + code.zero);
    }
  }
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    word += __float_as_uint(fminf(fmaxf(t[j], kRoundMagic), kRoundMagic + 15.f)) * (1u << (4 * j));
  return word - 0x4B400000u * 0x11111111u;
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
__device__ __forceinline__ float2 unpack2(uint32_t w) { return make_float2(bf16_lo(w), bf16_hi(w)); }
// Minimum and maximum that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One warp takes a piece of one token's query, key or value heads: the token's angles and the norm's weights stay in
// registers, and kBatch heads per lane group are loaded ahead of the one in work. A lane holds two runs of four
// components. Turning components (i, i + rotary / 2), it holds both of a pair: runs 4 l and rotary / 2 + 4 l, so the
// rotation needs no exchange between lanes; otherwise its runs are neighbours. FP32 throughout, two components to an
// instruction where nothing speaks against it. Bound by memory: 4 bytes per component of the norm, 2 read and
// dim / 2 + 4 bytes per head written for what is appended.
// Measured: norm of 16384 tokens, 32 and 8 heads of 128, 68 us (5.1 TB/s of a measured copy's 6.5); of 4099 tokens, 16 and
// 16 heads of 64, 8.3 us on the device; of one token 2.2 us; appending 8192 tokens, 32 and 8 heads of 128, 51 us: the queries
// 26 (5.1 TB/s), keys and values 24, bound by instruction issue (67 % of the cycles; 20 without the repairs of ties, which
// BF16 inputs meet in most warps' steps). One warp for all heads of a token, keys and queries mixed, took 112 for that norm.
// 64 registers and four CTAs of 256 threads an SM: three 52, five 118 us for that append (spills).
template <int kDim, bool kNorm, bool kAppend, bool kAdjacent>
__global__ void __launch_bounds__(256, 4) kv4_rows_kernel(const Kv4RowParams p) {
  constexpr int kLanes = kDim / 8, kHeadsPerStep = 32 / kLanes, kBatch = 4;
  pdl_wait();
  pdl_launch_dependents();
  const int warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int chunks = p.q_chunks + p.kv_chunks * (kAppend ? 2 : 1);
  const int token = warp / chunks;
  int chunk = warp - token * chunks;
  if (token >= p.tokens) return;      // whole warps
  const int kind = chunk < p.q_chunks ? 0 : chunk < p.q_chunks + p.kv_chunks ? 1 : 2;        // queries, keys, values
  chunk -= kind == 0 ? 0 : kind == 1 ? p.q_chunks : p.q_chunks + p.kv_chunks;
  const int lane = threadIdx.x % 32, l = lane % kLanes, sub = lane / kLanes;
  const int heads = kind == 0 ? p.q_heads : p.kv_heads, pieces = kind == 0 ? p.q_chunks : p.kv_chunks;
  const int per_chunk = (heads + pieces - 1) / pieces;
  const int first = chunk * per_chunk, end = min(heads, first + per_chunk);
  const bool turns = kind < 2 && l < p.rotary / 8;      // rotary is 0 without a table
  const bool split = turns && !kAdjacent;
  const int run0 = split ? 4 * l : 8 * l, run1 = split ? p.rotary / 2 + 4 * l : 8 * l + 4;

  const uint16_t* const src = (kind == 0 ? p.q + token * p.q_stride : kind == 1 ? p.k + token * p.k_stride : p.v + token * p.v_stride) + sub * kDim;
  uint2 raw[kBatch][2];
  auto load = [&](int i, int h) {
    raw[i][0] = raw[i][1] = make_uint2(0, 0);
    if (h + sub < end) {
      if constexpr (kAdjacent) {
        const uint4 w = *reinterpret_cast<const uint4*>(src + h * kDim + run0);
        raw[i][0] = make_uint2(w.x, w.y);
        raw[i][1] = make_uint2(w.z, w.w);
      } else {
        raw[i][0] = *reinterpret_cast<const uint2*>(src + h * kDim + run0);
        raw[i][1] = *reinterpret_cast<const uint2*>(src + h * kDim + run1);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kBatch; ++i) load(i, first + i * kHeadsPerStep);

  // The token's angles: this lane's four pairs.
  float c[4] = {}, s[4] = {};
  bool bad = false;
  if (p.cos_sin) {
    for (int a = 0; a < p.axes; ++a) {
      const int64_t place = p.positions[static_cast<int64_t>(a) * p.tokens + token];
      bad |= place < 0 || place >= p.table_rows;
    }
    const int f = 4 * l, pairs = p.rotary / 2;
    if (l < p.rotary / 8 && !bad) {
      if (!p.axis_of) {
        const float* row = p.cos_sin + p.positions[token] * p.rotary + f;
        const float4 cs = *reinterpret_cast<const float4*>(row), sn = *reinterpret_cast<const float4*>(row + pairs);
        c[0] = cs.x; c[1] = cs.y; c[2] = cs.z; c[3] = cs.w;
        s[0] = sn.x; s[1] = sn.y; s[2] = sn.z; s[3] = sn.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int axis = p.axis_of[f + j];
          if (axis < 0 || axis >= p.axes) {
            bad = true;
          } else {
            const float* row = p.cos_sin + p.positions[static_cast<int64_t>(axis) * p.tokens + token] * p.rotary + f + j;
            c[j] = row[0];
            s[j] = row[pairs];
          }
        }
      }
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  if (bad && lane == 0) atomicOr(&g_ci8_status, kStatusBadIndex);

  float2 weight[4];
  const uint16_t* const weights = kNorm ? (kind == 0 ? p.q_weight : p.k_weight) : nullptr;
  if (weights) {
    const uint2 a = *reinterpret_cast<const uint2*>(weights + run0), b = *reinterpret_cast<const uint2*>(weights + run1);
    const float2 offset = make_float2(p.weight_offset, p.weight_offset);
    weight[0] = __fadd2_rn(unpack2(a.x), offset);
    weight[1] = __fadd2_rn(unpack2(a.y), offset);
    weight[2] = __fadd2_rn(unpack2(b.x), offset);
    weight[3] = __fadd2_rn(unpack2(b.y), offset);
  }

  // Where the heads go: the outputs' rows, or the slot's page (null: not stored).
  uint16_t* const dst = kind == 0 ? p.q_out + token * p.q_out_stride + sub * kDim : kAppend ? nullptr : p.k_out + token * p.k_out_stride + sub * kDim;
  uint8_t* slot_page = nullptr;
  int slot_row = 0;
  const int page = 1 << p.page_shift;
  const unsigned block_bytes = page * (kDim / 2 + 4);    // at most 33792
  if (kAppend && kind > 0) {
    const int64_t slot = p.slots[token];
    if (slot >= p.capacity && lane == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
    if (slot < 0 || slot >= p.capacity || bad) return;
    slot_page = p.cache + ((slot >> p.page_shift) * kKv4Side + kind - 1) * p.kv_heads * static_cast<int64_t>(block_bytes);
    slot_row = static_cast<int>(slot & (page - 1));
  }

  for (int base = first; base < end; base += kBatch * kHeadsPerStep) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = base + i * kHeadsPerStep;
      if (h >= end) break;                               // the same for the whole warp
      const bool real = h + sub < end;
      float2 x[4] = {unpack2(raw[i][0].x), unpack2(raw[i][0].y), unpack2(raw[i][1].x), unpack2(raw[i][1].y)};
      load(i, h + kBatch * kHeadsPerStep);
      if (weights) {
        float2 squares = __fmul2_rn(x[0], x[0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) squares = __ffma2_rn(x[j], x[j], squares);
        float sum = squares.x + squares.y;
#pragma unroll
        for (int d = kLanes / 2; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float unit = rsqrtf(sum * (1.f / kDim) + p.eps);
        const float2 unit2 = make_float2(unit, unit);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __fmul2_rn(__fmul2_rn(x[j], unit2), weight[j]);
      }
      if (turns) {
        // Products and sums rounded one by one (single ones with a rounding mode; the packed ones may be contracted), so
        // that what is encoded does not depend on how a compiler contracts them.
        if constexpr (kAdjacent) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[j] = make_float2(__fsub_rn(__fmul_rn(x[j].x, c[j]), __fmul_rn(x[j].y, s[j])),
                               __fadd_rn(__fmul_rn(x[j].y, c[j]), __fmul_rn(x[j].x, s[j])));
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 a = x[j], b = x[j + 2];
            x[j] = make_float2(__fsub_rn(__fmul_rn(a.x, c[2 * j]), __fmul_rn(b.x, s[2 * j])),
                               __fsub_rn(__fmul_rn(a.y, c[2 * j + 1]), __fmul_rn(b.y, s[2 * j + 1])));
            x[j + 2] = make_float2(__fadd_rn(__fmul_rn(b.x, c[2 * j]), __fmul_rn(a.x, s[2 * j])),
                                   __fadd_rn(__fmul_rn(b.y, c[2 * j + 1]), __fmul_rn(a.y, s[2 * j + 1])));
          }
        }
      }
      if (!kAppend || kind == 0) {
        if (real) {
          uint2 a = make_uint2(pack2(x[0].x, x[0].y), pack2(x[1].x, x[1].y)), b = make_uint2(pack2(x[2].x, x[2].y), pack2(x[3].x, x[3].y));
          if (bad) a = b = make_uint2(0x7fff7fffu, 0x7fff7fffu);   // a position outside the table: NaN
          if constexpr (kAdjacent) {
            *reinterpret_cast<uint4*>(dst + h * kDim + run0) = make_uint4(a.x, a.y, b.x, b.y);
          } else {
            *reinterpret_cast<uint2*>(dst + h * kDim + run0) = a;
            *reinterpret_cast<uint2*>(dst + h * kDim + run1) = b;
          }
        }
        continue;
      }
      float low, high;
      auto range = [&]() {
        low = high = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          low = min_nan(low, min_nan(x[j].x, x[j].y));
          high = max_nan(high, max_nan(x[j].x, x[j].y));
        }
#pragma unroll
        for (int d = kLanes / 2; d; d /= 2) {
          low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, d));
          high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, d));
        }
      };
      range();
      if (__any_sync(0xffffffffu, !(low >= -8.5e37f && high <= 8.5e37f))) {
        // NaN counts as 0 and infinities as the largest value whose range still fits FP32, so that one such
        // component cannot spoil the scale and with it the whole head
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j].x = x[j].x != x[j].x ? 0.f : fminf(fmaxf(x[j].x, -8.5e37f), 8.5e37f);
          x[j].y = x[j].y != x[j].y ? 0.f : fminf(fmaxf(x[j].y, -8.5e37f), 8.5e37f);
        }
        range();
      }
      const Kv4Code code = kv4_code_of(low, high);
      const uint32_t word = kv4_encode8(x, code);
      if (real) {
        uint8_t* block = slot_page + (h + sub) * block_bytes;
        uint8_t* row = block + slot_row * (kDim / 2);
        *reinterpret_cast<uint16_t*>(row + run0 / 2) = static_cast<uint16_t>(word);
        *reinterpret_cast<uint16_t*>(row + run1 / 2) = static_cast<uint16_t>(word >> 16);
        if (l == 0) *reinterpret_cast<uint32_t*>(block + page * (kDim / 2) + 4 * slot_row) = pack2(code.scale, code.zero);
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
  int tokens, kv_heads, page_shift;
  int chunks;                // pieces that the heads of one token are cut into, one warp each
};

// One warp takes a piece of one token's heads (keys', then values'): eight codes (one word) per lane become eight BF16
// values. Two codes behind a mask are the BF16 numbers 128 + code; the zero point comes off exactly and the product
// with the scale is rounded once. Bound by memory (dim / 2 + 4 bytes read, 2 dim written per head). Measured: 65536 tokens,
// 8 heads of 128, 62 us (5.5 TB/s); one CTA per token and head took 126.
template <int kDim>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
  constexpr int kLanes = kDim / 8, kHeadsPerStep = 32 / kLanes, kBatch = 8;
  pdl_wait();
  pdl_launch_dependents();
  const int page = 1 << p.page_shift;
  const unsigned block_bytes = page * (kDim / 2 + 4);
  const int warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int token = warp / p.chunks, chunk = warp % p.chunks;
  if (token >= p.tokens) return;
  const int lane = threadIdx.x % 32, l = lane % kLanes, sub = lane / kLanes;
  const int heads = 2 * p.kv_heads, per_chunk = (heads + p.chunks - 1) / p.chunks;
  const int first = chunk * per_chunk, end = min(heads, first + per_chunk);
  const int64_t slot = p.slots[token];
  if (slot >= p.capacity && lane == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
  const bool there = slot >= 0 && slot < p.capacity;
  const uint8_t* src = p.cache + (there ? (slot >> p.page_shift) * heads * static_cast<int64_t>(block_bytes) : 0);
  const int row = static_cast<int>(slot & (page - 1));
  uint16_t* const k = p.k + static_cast<int64_t>(token) * p.kv_heads * kDim + 8 * l;
  uint16_t* const v = p.v + static_cast<int64_t>(token) * p.kv_heads * kDim + 8 * l;
  for (int base = first; base < end; base += kBatch * kHeadsPerStep) {
    uint32_t word[kBatch], pair[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = base + i * kHeadsPerStep + sub;
      word[i] = pair[i] = 0;                             // scale 0: the row reads as zeros
      if (there && h < end) {
        word[i] = *reinterpret_cast<const uint32_t*>(src + h * block_bytes + row * (kDim / 2) + 4 * l);
        pair[i] = *reinterpret_cast<const uint32_t*>(src + h * block_bytes + page * (kDim / 2) + 4 * row);
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = base + i * kHeadsPerStep + sub;
      if (h >= end) continue;
      const uint32_t scale = __byte_perm(pair[i], 0, 0x1010);
      uint32_t zero = __byte_perm(pair[i], 0, 0x3232), x[4];
      asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(zero) : "r"(0x43004300u));
#pragma unroll
      for (int j = 0; j < 4; ++j) {                      // components j and j + 4
        x[j] = ((word[i] >> (4 * j)) & 0x000f000fu) | 0x43004300u;
        asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(x[j]) : "r"(zero));
        asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(x[j]) : "r"(scale));
      }
      uint16_t* dst = h < p.kv_heads ? k + h * kDim : v + (h - p.kv_heads) * kDim;
      *reinterpret_cast<uint4*>(dst) = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410),
                                                  __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
    }
  }
}

}  // namespace ci8
