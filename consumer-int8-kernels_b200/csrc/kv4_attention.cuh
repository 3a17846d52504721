// Causal attention over the 4-bit key/value cache: what its kernels share.
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

// 2^x within a relative error of 2^-22.
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

}  // namespace ci8
