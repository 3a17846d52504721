// Causal attention over the 4-bit key/value cache.
#pragma once
#include "kv4_rows.cuh"

namespace ci8 {

// Division by a number that is known on the host: n / d for n below 2^31 as a product and a shift (m is
// 2^(31 + s) / d rounded up, s = ceil(log2 d), so the error n * (m - 2^(31+s)/d) / 2^(31+s) stays below 1 / d).
struct Kv4Divisor {
  unsigned m, s, d;
  __host__ static Kv4Divisor of(unsigned d) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    return {static_cast<unsigned>(((1ull << (31 + s)) + d - 1) / d), s, d};
  }
  __device__ __forceinline__ int quotient(int n) const { return static_cast<int>(__umulhi(2u * static_cast<unsigned>(n), m) >> s); }
};

struct Kv4AttendParams {
  const uint16_t* q;          // [tokens, q_heads, dim], token stride in elements
  int64_t q_stride;
  const uint8_t* cache;
  const int32_t* block_table; // [batch, width]
  const int32_t* q_starts;    // [batch + 1]
  const int32_t* kv_lens;     // [batch]
  uint16_t* out;              // [tokens, q_heads, dim]
  int tokens, batch, width, q_heads, kv_heads, page_shift, pages;
  float scale_log2;           // softmax scale * log2(e)
  Kv4Divisor group;           // query heads per key head
};

// The rows and keys of sequence b, with whatever the metadata says cut to the tensors' sizes.
struct Kv4Sequence {
  int start, rows, keys;      // first token row, token rows, cached keys
};
__device__ __forceinline__ Kv4Sequence kv4_sequence(const Kv4AttendParams& p, int b) {
  Kv4Sequence s;
  const int begin = max(0, p.q_starts[b]), end = min(p.tokens, p.q_starts[b + 1]);
  s.start = begin;
  s.rows = max(0, end - begin);
  const int64_t room = static_cast<int64_t>(p.width) << p.page_shift;
  const int keys = max(0, p.kv_lens[b]);
  s.keys = static_cast<int>(keys < room ? keys : room);
  return s;
}

// One CTA per token row and query head; every lane group walks its own keys.
template <int kDim>
__global__ void __launch_bounds__(128) kv4_attend_kernel(const Kv4AttendParams p) {
  constexpr int kLanes = kDim / 8, kGroups = 128 / kLanes;
  __shared__ float merged_m[kGroups], merged_l[kGroups], merged_o[kGroups][kDim];
  pdl_wait();
  const int token = blockIdx.x, head = blockIdx.y;
  int b = -1;
  Kv4Sequence s{};
  for (int i = 0; i < p.batch; ++i) {
    s = kv4_sequence(p, i);
    if (token >= s.start && token < s.start + s.rows) { b = i; break; }
  }
  if (b < 0) return;
  const int keys = s.keys - s.rows + (token - s.start) + 1;
  const int l = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int page = 1 << p.page_shift, kv_head = head / (p.q_heads / p.kv_heads);
  float q[8], o[8] = {}, m = -INFINITY, sum = 0.f;
  unpack8(*reinterpret_cast<const uint4*>(p.q + token * p.q_stride + static_cast<int64_t>(head) * kDim + 8 * l), q);
  for (int base = 0; base < keys; base += kGroups) {
    const int key = base + group;
    uint32_t kw = 0, vw = 0, kp = 0, vp = 0;
    bool seen = key < keys;
    if (seen) {
      const int id = p.block_table[static_cast<int64_t>(b) * p.width + (key >> p.page_shift)];
      seen = id >= 0 && id < p.pages;
      if (seen) {
        const uint8_t* block = p.cache + (static_cast<int64_t>(id) * 2 * p.kv_heads + kv_head) * kv4_block_bytes(page, kDim);
        const uint8_t* other = block + p.kv_heads * kv4_block_bytes(page, kDim);
        const int at = key & (page - 1);
        kw = *reinterpret_cast<const uint32_t*>(block + at * (kDim / 2) + 4 * l);
        kp = *reinterpret_cast<const uint32_t*>(block + page * (kDim / 2) + 4 * at);
        vw = *reinterpret_cast<const uint32_t*>(other + at * (kDim / 2) + 4 * l);
        vp = *reinterpret_cast<const uint32_t*>(other + page * (kDim / 2) + 4 * at);
      } else if (l == 0) {
        atomicOr(&g_ci8_status, kStatusBadIndex);
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) dot = fmaf(q[j], static_cast<float>((kw >> (4 * j)) & 15u) - bf16_hi(kp), dot);
    dot = head_sum<kLanes>(dot) * bf16_lo(kp) * p.scale_log2;
    if (seen) {
      const float top = fmaxf(m, dot), keep = exp2f(m - top), w = exp2f(dot - top);
      m = top;
      sum = sum * keep + w;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o[j] = o[j] * keep + w * bf16_lo(vp) * (static_cast<float>((vw >> (4 * j)) & 15u) - bf16_hi(vp));
    }
  }
  if (l == 0) { merged_m[group] = m; merged_l[group] = sum; }
#pragma unroll
  for (int j = 0; j < 8; ++j) merged_o[group][8 * l + j] = o[j];
  __syncthreads();
  float top = -INFINITY;
  for (int g = 0; g < kGroups; ++g) top = fmaxf(top, merged_m[g]);
  for (int c = threadIdx.x; c < kDim; c += 128) {
    float total = 0.f, value = 0.f;
    for (int g = 0; g < kGroups; ++g) {
      if (merged_l[g] == 0.f) continue;          // saw no key (a NaN score makes the sum NaN, which is kept)
      const float w = exp2f(merged_m[g] - top);
      total += w * merged_l[g];
      value += w * merged_o[g][c];
    }
    const float r = total == 0.f ? 0.f : value / total;
    p.out[(static_cast<int64_t>(token) * p.q_heads + head) * kDim + c] = static_cast<uint16_t>(pack2(r, 0.f));
  }
}

}  // namespace ci8
