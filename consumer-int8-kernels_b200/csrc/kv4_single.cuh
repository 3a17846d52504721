// Attention of few query rows per sequence (generated tokens) over the 4-bit key/value cache: bound by reading the
// cache, dim / 2 + 4 bytes per token and side, and as much by the instructions that unpack it: 530 for a warp's 32 keys of 128
// components (16 + 16 of them matrix products), with the schedulers issuing in 56 % of the cycles and the logic pipe
// busy in 50 %. Measured: 64 sequences of up to 8192 keys, 32 query heads and 8 key heads of 128, 76 us (3.9 TB/s); 4 of 65536,
// 24 and 4 heads of 256, 77 us (3.6 TB/s); one of 1000 keys 12 us, most of it a chain of dependent loads and joins. The same
// loads without the arithmetic reach 5.6 TB/s.
//
// Work is cut into tiles of 64 tokens (32 for dim 256) of one (sequence, key head, block of query rows) and the tiles of all of
// them, laid end to end, are dealt to the warps in equal contiguous ranges, so that ragged batches fill the GPU evenly and
// a long history is split as far as there are warps. Every warp runs on its own: its ring of tiles is filled by
// asynchronous copies it issues itself, and it keeps its own running maximum, sum and output. Ranges begin and end inside a
// sequence; what a warp has of such a sequence is joined with its neighbours' inside the CTA at the end, and across
// CTAs by whichever of them comes last, in the order of the CTAs (so the bits do not depend on the timing).
//
// The products run transposed on the tensor cores with register-fed operands (mma.sync), S^T[token, query] = K Q^T and
// O^T[component, query] = V^T P^T, so that eight query rows fill an instruction and the cache is the operand that is
// unpacked on the way, straight from its packed words. What limits the kernel beside the memory is the logic pipe
// (two cycles a mask-and-or), so each product takes the form that needs the fewest:
//   S^T  INT8 (m16n8k32): two masks give the eight codes of a word. The queries become 16-bit fixed point, two INT8
//        digits relative to the row's largest component, two exact integer products; a query component is off by at
//        most 1 / 65278 of the largest (half a step, 2^-16), which for BF16 components within a factor 128 of it is no more
//        than their own rounding (2^-9 of a component at least). The sums, less zero * sum of q, are exact integers, rounded
//        once to FP32 (they may have 28 bits) and then multiplied by the row's unit and the key's scale.
//   O^T  FP16 (m16n8k16): a mask-and-or gives 1024 + code or 1024 + 16 * code for two tokens, one packed FMA the exact
//        small integer code - zero (not zero points taken out of the sum afterwards: a sum over the whole history
//        would cancel). The weights carry the values' scales, relative to the largest scale that the row has seen so far, which
//        keeps them within FP16: 2^-11 relative rounding down to 2^-21 of the largest, multiples of 2^-31 of it below.
// Maxima, sums, scores and outputs are FP32.
#pragma once
#include "kv4_attention.cuh"

namespace ci8 {

constexpr int kKv4CounterBytes = 4096;                          // arrival counters at the head of the workspace
constexpr int kKv4MaxCtas = kKv4CounterBytes / 4;

template <int kDim, int kQ>                                     // kQ: groups of eight query rows per warp
struct Kv4SingleConfig {
  static constexpr int kRows = 8 * kQ;
  // Tokens per ring stage: 64 halve what a tile costs beside its products, 32 are what the ring has room for at dim 256.
  // Warps: as many as the registers allow (output and queries take kDim * kQ * 3 / 8 a thread). Measured (us, 64 sequences of
  // up to 8192 keys, 4 heads a key head): 32 tokens and 16 warps 91, 64 and 12 83, 64 and 8 87, 32 and 12 94.
  static constexpr int kTile = kDim <= 128 ? 64 : 32;
  static constexpr int kWarps = kDim * kQ == 64 ? 16 : kDim * kQ == 128 || kDim == 256 && kQ == 1 ? 12 : 8;
  static constexpr int kParts = kTile / 16;                     // a part lies on one page
  static constexpr int kCodeBytes = kTile * kDim / 2;
  static constexpr int kPairBytes = kTile * 4;
  static constexpr int kStageBytes = 2 * (kCodeBytes + kPairBytes);
  static constexpr int kRing = 204 * 1024 / (kWarps * kStageBytes);
  static constexpr int kStages = kRing > 6 ? 6 : kRing;
  static constexpr int kPieceFloats = kRows * (kDim + 2);       // maximum, sum and output of every row
  static constexpr int kSmemBytes = kWarps * kStages * kStageBytes;
  static_assert(kStages >= 2 && kPieceFloats * 4 <= kStages * kStageBytes, "a warp's last piece is kept in its ring");
};

// Workspace: counters, then two slots per CTA (pieces of sequences shared with the CTA before and behind), then one
// per warp (the piece that ends inside the warp's range).
template <int kDim, int kQ>
__host__ __device__ constexpr long long kv4_single_workspace(long long ctas) {
  return kKv4CounterBytes + ctas * (2 + Kv4SingleConfig<kDim, kQ>::kWarps) * Kv4SingleConfig<kDim, kQ>::kPieceFloats * 4;
}

struct Kv4SingleParams {
  Kv4AttendParams a;
  unsigned* counters;
  float* slots;
  int most_rows;              // sequences with more query rows (rows * heads per key head) are left to another kernel
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes (unsigned) x digits (signed)
__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Four-bit codes of two tokens, at bits 0..3 and 16..19 of w (i = 0) or at bits 4..7 and 20..23 (i = 1), less the tokens'
// zero points, as FP16: the mask-and-or gives 1024 + code (1024 + 16 * code), and what is subtracted is 1024 + zero
// (64 + zero).
template <int i>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, uint32_t ones, uint32_t minus_low, uint32_t minus_high) {
  uint32_t x;
  if constexpr (i == 0) {
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(x) : "r"(w), "r"(ones));   // (w & mask) | ones, ones = 0x64006400
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(minus_low));
  } else {
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(x) : "r"(w), "r"(ones));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(x) : "r"(0x2c002c00u), "r"(minus_high));   // * 1/16
  }
  return x;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds32(const uint8_t* at) { return *reinterpret_cast<const uint32_t*>(at); }
__device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t (&w)[1]) { w[0] = lds32(at); }
__device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t (&w)[2]) {
  const uint2 v = *reinterpret_cast<const uint2*>(at);
  w[0] = v.x; w[1] = v.y;
}
__device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t (&w)[4]) {
  const uint4 v = *reinterpret_cast<const uint4*>(at);
  w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}
// Sixteen bytes to shared memory past the registers and the L1, at a fixed offset from both addresses.
template <int kDst, int kSrc>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(kDst), "n"(kSrc) : "memory");
}
// The same with what is beyond `bytes` filled with zeros.
template <int kDst, int kSrc>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(kDst), "n"(kSrc) : "memory");
}
// Code rows, 512 bytes at a time: kCopies copies at kDst + 512 * i, every other one from dst_odd.
template <int kCopies, int kDst, int i = 0>
__device__ __forceinline__ void copy_rows(uint32_t dst, uint32_t dst_odd, const uint8_t* src) {
  if constexpr (i < kCopies) {
    copy16<kDst + 512 * i, 512 * i>(i % 2 ? dst_odd : dst, src);
    copy_rows<kCopies, kDst, i + 1>(dst, dst_odd, src);
  }
}
// Of those rows the first `rows`; the lane's row of the first copy is lane_row, and a copy covers kPerCopy.
template <int kCopies, int kDst, int kPerCopy, int i = 0>
__device__ __forceinline__ void copy_rows(uint32_t dst, uint32_t dst_odd, const uint8_t* src, int rows, int lane_row) {
  if constexpr (i < kCopies) {
    copy16<kDst + 512 * i, 512 * i>(i % 2 ? dst_odd : dst, src, lane_row + i * kPerCopy < rows ? 16 : 0);
    copy_rows<kCopies, kDst, kPerCopy, i + 1>(dst, dst_odd, src, rows, lane_row);
  }
}
// The places in shared memory that the lanes (g, c) of a warp read together: 16 bytes (dim 64: 8) of the keys of rows
// kv4_row(g) at c, 16 (8, 4) bytes of the values of the rows kv4_row(2c) or kv4_row(2c + 1) at g. Which token a row of
// S^T stands for is free, and so is the order of a row's 16-byte pieces (piece ^ kv4_turn(row)): chosen such that the
// eight (sixteen, thirty-two) lanes of one access lie in different banks for keys and for values.
template <int kDim>
__device__ __forceinline__ int kv4_row(int g) {
  return kDim == 64 ? g ^ (g >> 2 & 1) : kDim == 128 ? g ^ (g >> 1 & 1) : g >> 1 | (g & 1) << 2;
}
template <int kDim>
__device__ __forceinline__ int kv4_turn(int row) {
  return kDim == 64 ? 0 : kDim == 128 ? row >> 1 & 2 : ((row & 3) << 1) ^ (row & 4);
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Number of keys the last row of a block of query rows sees, and the tiles they make (one at least: rows that see
// nothing have to be written too).
__device__ __forceinline__ int kv4_block_keys(const Kv4Sequence& s, const Kv4Divisor& group, int rows_per_block, int block) {
  const int last = min(s.rows * static_cast<int>(group.d), (block + 1) * rows_per_block) - 1;
  return max(0, s.keys - s.rows + group.quotient(last) + 1);
}
template <int kTile>
__device__ __forceinline__ int kv4_block_tiles(int keys) { return max(1, (keys + kTile - 1) / kTile); }
// Tiles of one key head of a sequence.
template <int kTile>
__device__ __forceinline__ long long kv4_head_tiles(const Kv4Sequence& s, const Kv4Divisor& group, int rows_per_block, int most_rows) {
  const int rows = s.rows * static_cast<int>(group.d);
  if (rows == 0 || rows > most_rows) return 0;
  long long tiles = 0;
#pragma unroll 1
  for (int block = 0; block * rows_per_block < rows; ++block) tiles += kv4_block_tiles<kTile>(kv4_block_keys(s, group, rows_per_block, block));
  return tiles;
}

// What a warp leaves of a sequence it shares with a neighbour.
struct Kv4Piece {
  int kind;                       // 0 none, 1 ends the sequence's tiles (in the workspace), 2 open at its end (in the ring)
  int starts;                     // it holds the first tile
  unsigned first, tiles;          // place of the first tile among all, number of tiles
  int start, row, rows, head;     // first token row of the sequence, first query row of the block, its rows, key head
};

template <int kDim, int kQ>
__global__ void __launch_bounds__(Kv4SingleConfig<kDim, kQ>::kWarps * 32, 1) kv4_single_kernel(const Kv4SingleParams params) {
  using Cfg = Kv4SingleConfig<kDim, kQ>;
  constexpr int kWarps = Cfg::kWarps, kThreads = kWarps * 32, kStages = Cfg::kStages, kRows = Cfg::kRows;
  constexpr int kTile = Cfg::kTile, kParts = Cfg::kParts;
  constexpr int kKWords = kDim / 32;                     // a lane's words of a key row
  constexpr int kVWords = kDim / 64;                     // a lane's words of a value row
  constexpr int kLoad = kKWords > 4 ? 4 : kKWords;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ int4 infos[kWarps][kStages];
  __shared__ long long scans[kThreads], warp_sums[kWarps];
  __shared__ Kv4Piece pieces[2 * kWarps];
  __shared__ Kv4Piece shared_units[2];                   // sequences shared with the CTA before [0] and behind [1]
  __shared__ float piece_m[2 * kWarps][kRows], piece_l[2 * kWarps][kRows], group_m[2 * kWarps][kRows], group_l[2 * kWarps][kRows];
  __shared__ float weights[2 * kWarps][kRows];
  __shared__ int comes_last[2];
  const Kv4AttendParams& p = params.a;
  const int thread = threadIdx.x, warp = thread / 32, lane = thread % 32, g = lane / 4, c = lane % 4;
  const int group = p.group.d;

  if (thread < 2 * kWarps) pieces[thread].kind = 0;
  if (thread < 2) shared_units[thread].kind = comes_last[thread] = 0;
  pdl_wait();
  pdl_launch_dependents();

  // ---- every tile's place: thread t sums the sequences of its share, then a scan over the threads
  const int share = (p.batch + kThreads - 1) / kThreads;
  long long scan = 0;
  for (int b = thread * share; b < min(p.batch, (thread + 1) * share); ++b)
    scan += kv4_head_tiles<kTile>(kv4_sequence(p, b), p.group, kRows, params.most_rows) * p.kv_heads;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long other = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += other;
  }
  scans[thread] = scan;
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  long long sums = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
  for (int d = 1; d < kWarps; d *= 2) {
    const long long other = __shfl_up_sync(0xffffffffu, sums, d);
    if (lane >= d) sums += other;
  }
  const long long all_tiles = __shfl_sync(0xffffffffu, sums, kWarps - 1);
  if (all_tiles == 0) return;
  if (all_tiles >> 31) {                                 // 10^11 keys, many minutes of work, or overlapping sequences: refused
    if (thread == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
    return;
  }
  const unsigned total = static_cast<unsigned>(all_tiles);
  // No more CTAs than get kLeast tiles each: below that, joining them costs more than the tiles. Measured (us for 1, 4, 16):
  // one sequence of 100 keys, 8 key heads of 128, 10.4, 7.7, 11.8; of 1000 12.2, 11.5, 13.5; of 8000 15.1, 15.4, 20.3.
  constexpr unsigned kLeast = 4;
  const unsigned ctas = min(gridDim.x, (total + kLeast - 1) / kLeast);
  if (blockIdx.x >= ctas) return;
  const unsigned per_cta = total / ctas, longer = total - per_cta * ctas;   // the first `longer` CTAs take one more
  const unsigned cta_tiles = per_cta + (blockIdx.x < longer ? 1 : 0);
  const unsigned cta_first = blockIdx.x * per_cta + min(blockIdx.x, longer);
  const int per_warp = cta_tiles / kWarps, more = cta_tiles % kWarps;
  const int count = per_warp + (warp < more ? 1 : 0);
  const unsigned range = cta_first + warp * per_warp + min(warp, more);

  // ---- where this warp's range begins
  int b = 0, head = 0, block = 0, tile = 0, keys = 0, tiles = 0;
  Kv4Sequence seq{};
  if (count > 0) {
    const int w = __popc(__ballot_sync(0xffffffffu, lane < kWarps && sums <= range));           // the warp, then the thread
    const long long before = w ? __shfl_sync(0xffffffffu, sums, w - 1) : 0;
    const long long within = scans[w * 32 + lane];
    const int t = __popc(__ballot_sync(0xffffffffu, before + within <= range));                 // whose share holds the first tile
    unsigned rest = range - static_cast<unsigned>(before) - (t ? static_cast<unsigned>(__shfl_sync(0xffffffffu, within, t - 1)) : 0);
    unsigned per_head = 0;
    for (b = (w * 32 + t) * share;; ++b) {
      seq = kv4_sequence(p, b);
      per_head = static_cast<unsigned>(kv4_head_tiles<kTile>(seq, p.group, kRows, params.most_rows));
      if (rest < per_head * p.kv_heads) break;
      rest -= per_head * p.kv_heads;
    }
    head = rest / per_head;
    rest -= head * per_head;
    for (block = 0;; ++block) {
      keys = kv4_block_keys(seq, p.group, kRows, block);
      tiles = kv4_block_tiles<kTile>(keys);
      if (rest < static_cast<unsigned>(tiles)) break;
      rest -= tiles;
    }
    tile = rest;
  }

  // ---- the loader's side of the ring: the tiles of the range in order, copied by the lanes in pieces of 16 bytes; the
  // lanes hold the next 32 page numbers of the sequence
  const int page = 1 << p.page_shift;
  const unsigned block_bytes = page * (kDim / 2 + 4), page_bytes = block_bytes * kKv4Side * p.kv_heads;   // at most 70 MB
  const uint32_t ring_base = smem_u32(ring) + warp * kStages * Cfg::kStageBytes;
  const bool small_page = page % kTile != 0;             // a tile may touch several pages
  constexpr int kRowPieces = kDim / 32;                  // 16-byte pieces of a code row
  constexpr int kCopies = kRowPieces / 2, kPerCopy = 32 / kRowPieces;          // copies for a part's codes, rows a copy covers
  constexpr int kValues = Cfg::kCodeBytes + Cfg::kPairBytes;
  const int lane_row = lane / kRowPieces;                // the lane's row among those one copy covers
  // Pieces are stored in an order that depends on the row, so that the lanes that read together read different banks
  // (kv4_turn); at dim 256 every other copy has its rows' bit 2 set, which moves its pieces by 4.
  const int lane_piece = lane % kRowPieces ^ kv4_turn<kDim>(lane_row);
  const uint32_t lane_code = ring_base + 16 * (lane_row * kRowPieces + lane_piece);
  const uint32_t lane_code_odd = ring_base + 16 * (lane_row * kRowPieces + (kDim == 256 ? lane_piece ^ 4 : lane_piece));
  const unsigned value_offset = p.kv_heads * block_bytes;
  // the pairs: a lane takes four tokens' of one side
  const int pair_token = 4 * (lane % (kTile / 4)), pair_side = lane / (kTile / 4);
  const unsigned pair_offset = page * (kDim / 2) + (pair_side ? value_offset : 0);
  const uint32_t pair_dst = ring_base + Cfg::kCodeBytes + 4 * pair_token + pair_side * kValues;
  const uint8_t* head_src = nullptr;
  int window = -1, window_first = 0;
  auto load_window = [&]() {
    window_first = tile * kTile >> p.page_shift;
    const int index = window_first + lane;
    window = static_cast<int64_t>(index) << p.page_shift < keys ? p.block_table[static_cast<int64_t>(b) * p.width + index] : -1;
  };
  auto begin_unit = [&]() {
    head_src = p.cache + static_cast<uint64_t>(head) * block_bytes;
    load_window();
  };
  auto page_src = [&](int id) { return head_src + static_cast<uint64_t>(static_cast<unsigned>(id)) * page_bytes; };
  auto issue = [&](int stage) {
    const int token = tile * kTile;
    const int rows = min(kTile, keys - token);           // none or fewer: rows that see nothing
    if (((token + kTile - 1) >> p.page_shift) - window_first >= 32) load_window();
    const int pair_at = token + pair_token;
    int id = __shfl_sync(0xffffffffu, window, (pair_at >> p.page_shift) - window_first);
    const bool wanted = token + (pair_token & ~15) < keys, good = wanted && static_cast<unsigned>(id) < static_cast<unsigned>(p.pages);
    const uint32_t goods = __ballot_sync(0xffffffffu, good);
    if (__any_sync(0xffffffffu, wanted && !good) && lane == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
    if (!good) id = 0;
    const uint8_t* const pair_src = page_src(id) + pair_offset + 4 * (pair_at & (page - 1));
    const uint32_t dst = lane_code + stage * Cfg::kStageBytes, dst_odd = lane_code_odd + stage * Cfg::kStageBytes;
    const uint32_t to_pair = pair_dst + stage * Cfg::kStageBytes;
    int parts = 0;                                       // of this tile that are there
#pragma unroll
    for (int r = 0; r < kParts; ++r) parts |= (goods >> (4 * r) & 1) << r;
    if (lane == 0) infos[warp][stage] = make_int4(b, head, block, (tile << (kParts + 1)) | (tile == tiles - 1 ? 1 << kParts : 0) | parts);
    const uint8_t* src = page_src(__shfl_sync(0xffffffffu, id, 0)) + (token & (page - 1)) * (kDim / 2) + 16 * lane;
    if (rows == kTile && goods == ~0u) {
      if (pair_side < 2) copy16<0, 0>(to_pair, pair_src);
      if (!small_page) {
        copy_rows<kCopies * kParts, 0>(dst, dst_odd, src);
        copy_rows<kCopies * kParts, kValues>(dst, dst_odd, src + value_offset);
      } else {
#pragma unroll
        for (int r = 0; r < kParts; ++r) {
          const int at = token + 16 * r;
          src = page_src(__shfl_sync(0xffffffffu, window, (at >> p.page_shift) - window_first)) + (at & (page - 1)) * (kDim / 2) + 16 * lane;
          copy_rows<kCopies, 0>(dst + 8 * kDim * r, dst_odd + 8 * kDim * r, src);
          copy_rows<kCopies, kValues>(dst + 8 * kDim * r, dst_odd + 8 * kDim * r, src + value_offset);
        }
      }
    } else {
      // rows behind the last key or on a page that cannot be followed are filled with zeros: scale 0, zero point 0
      // (their source is an address that is not read: a copy of no bytes)
#pragma unroll 1
      for (int r = 0; r < kParts; ++r) {
        const int at = token + 16 * r, part_rows = parts >> r & 1 ? rows - 16 * r : 0;
        src = page_src(__shfl_sync(0xffffffffu, id, 4 * r)) + (at & (page - 1)) * (kDim / 2) + 16 * lane;
        copy_rows<kCopies, 0, kPerCopy>(dst + 8 * kDim * r, dst_odd + 8 * kDim * r, src, part_rows, lane_row);
        copy_rows<kCopies, kValues, kPerCopy>(dst + 8 * kDim * r, dst_odd + 8 * kDim * r, src + value_offset, part_rows, lane_row);
      }
      if (pair_side < 2) copy16<0, 0>(to_pair, pair_src, good ? 4 * max(0, min(4, rows - pair_token)) : 0);
    }
    if (++tile == tiles) {                               // the next block of rows, head or sequence
      tile = 0;
      if (++block * kRows >= seq.rows * group) {
        block = 0;
        if (++head == p.kv_heads) {
          head = 0;
          do {
            if (++b < p.batch) seq = kv4_sequence(p, b);
          } while (b < p.batch && (seq.rows == 0 || seq.rows * group > params.most_rows));
        }
      }
      if (b < p.batch) {
        keys = kv4_block_keys(seq, p.group, kRows, block);
        tiles = kv4_block_tiles<kTile>(keys);
        begin_unit();
      }
    }
    __syncwarp();                                        // the tile's description is there for every lane
  };
  if (count > 0) begin_unit();
  // ---- the consumer's side
  float o[4 * kVWords][kQ][4];
  float m[kQ][2], sum[kQ][2], qscale[kQ][2];
  int qsum[kQ][2];
  // 128 / the power of two above the values' scales that the row has seen so far (a row of its own: large values that are hidden
  // from it must not push its weights out of FP16); before the first scale above 0 2^118, which a weight may be multiplied with.
  // Powers of two, so two rows' fit a register as BF16 numbers.
  uint32_t value_units[kQ] = {};
  constexpr uint32_t kFirstUnits = 0x7a807a80u;
  auto value_unit = [&](int n, int e) { return e ? bf16_hi(value_units[n]) : bf16_lo(value_units[n]); };
  int limit[kQ][2];
  uint32_t q[kKWords][kQ][4];                            // high digits (even, odd components of a word), low digits
  int cur_b = 0, cur_head = 0, cur_block = 0, cur_tile = 0, cur_rows = 0, cur_start = 0, cur_keys = 0, first_tile = 0;
  int least = 0;
  bool fresh = true;
  const int turned = kv4_row<kDim>(g);                   // which token of eight a row of S^T holds
  const int t_even = kv4_row<kDim>(2 * c), t_odd = kv4_row<kDim>(2 * c + 1);
  const int key_at = turned * (kDim / 2) + (kDim == 64 ? 8 * c : 16 * (c ^ kv4_turn<kDim>(turned)));
  auto value_at = [&](int row) {
    return row * (kDim / 2) + (kDim == 64 ? 4 * g : kDim == 128 ? 16 * (g >> 1 ^ kv4_turn<kDim>(row)) + 8 * (g & 1) : 16 * (g ^ kv4_turn<kDim>(row)));
  };
  const int even_at = value_at(t_even), odd_at = value_at(t_odd);
  uint32_t ones;                                         // kept in a register: an immediate would cost a second instruction
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(ones));

  // Leaves this warp's maximum, sum (in piece_m, piece_l) and output of every row. An output is divided by its sum before it
  // leaves the unit it was summed in, here and wherever pieces are joined: sums of large values have no place in FP32.
  auto write_piece = [&](int piece, float* dst) {
#pragma unroll
    for (int n = 0; n < kQ; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * n + 2 * c + e;
        const float inverse = sum[n][e] == 0.f ? 0.f : 1.f / value_unit(n, e) / sum[n][e];   // the unit is a power of two
        if (g == 0) {
          piece_m[piece][row] = m[n][e];
          piece_l[piece][row] = sum[n][e];
        }
#pragma unroll
        for (int k = 0; k < kVWords; ++k) {
          float4* to = reinterpret_cast<float4*>(dst + row * kDim + 8 * (kVWords * g + k));
          to[0] = make_float4(o[4 * k][n][e] * inverse, o[4 * k + 1][n][e] * inverse, o[4 * k + 2][n][e] * inverse, o[4 * k + 3][n][e] * inverse);
          to[1] = make_float4(o[4 * k][n][2 + e] * inverse, o[4 * k + 1][n][2 + e] * inverse, o[4 * k + 2][n][2 + e] * inverse, o[4 * k + 3][n][2 + e] * inverse);
        }
      }
  };
  auto add_sums = [&]() {                                // the lanes' sums over their tokens, joined
#pragma unroll
    for (int n = 0; n < kQ; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 4);
        sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 8);
        sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 16);
      }
  };
  // Queries of a block of rows: lane (g, c) holds row g's words c as digits, in the order of a word's two masks.
  auto load_queries = [&]() {
    const Kv4Sequence s = kv4_sequence(p, cur_b);
    cur_rows = s.rows * group;
    cur_start = s.start;
    cur_keys = kv4_block_keys(s, p.group, kRows, cur_block);
    least = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < kQ; ++n) {
      const int row = cur_block * kRows + 8 * n + g, row_token = p.group.quotient(row);
      const uint16_t* src = p.q + (cur_start + row_token) * p.q_stride + static_cast<int64_t>(cur_head * group + row - row_token * group) * kDim;
      uint4 w[kKWords];
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < kKWords; ++k) {
        const int word = kLoad * c + (k % kLoad) + (k / kLoad) * 4 * kLoad;
        w[k] = make_uint4(0, 0, 0, 0);
        if (row < cur_rows)
          w[k] = *reinterpret_cast<const uint4*>(src + 8 * word);
      }
#pragma unroll
      for (int k = 0; k < kKWords; ++k) {
        float x[8];
        unpack8(w[k], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max_abs_keep_nan(most, x[j]);
      }
      most = fabsf(most);
      most = max_abs_keep_nan(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fabsf(max_abs_keep_nan(most, __shfl_xor_sync(0xffffffffu, most, 2)));
      // 127 * 256 + 127 steps; from 2^-100 on, so that a row of zeros or of the smallest numbers has a finite scale too
      const float largest = fmaxf(most, 0x1p-100f), scale = 32639.f / largest;
      // a row with a NaN or an infinity has NaN scores
      const float unit = most < INFINITY ? largest * (1.f / 32639.f) * p.scale_log2 : __int_as_float(0x7fffffff);
      int digits_sum = 0;
#pragma unroll
      for (int k = 0; k < kKWords; ++k) {
        float x[8];
        unpack8(w[k], x);
        // x * scale rounded to an integer by adding 1.5 * 2^23: its low byte is the low digit; with 128 more, its second
        // byte is the high one
        uint32_t low[8], high[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          low[j] = __float_as_uint(fmaf(x[j], scale, 12582912.f));
          high[j] = __float_as_uint(fmaf(x[j], scale, 12582912.f + 128.f));
        }
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          q[k][n][odd] = __byte_perm(__byte_perm(high[odd], high[2 + odd], 0x0051), __byte_perm(high[4 + odd], high[6 + odd], 0x0051), 0x5410);
          q[k][n][2 + odd] = __byte_perm(__byte_perm(low[odd], low[2 + odd], 0x0040), __byte_perm(low[4 + odd], low[6 + odd], 0x0040), 0x5410);
          digits_sum += 256 * __dp4a(static_cast<int>(q[k][n][odd]), 0x01010101, 0) + __dp4a(static_cast<int>(q[k][n][2 + odd]), 0x01010101, 0);
        }
      }
      digits_sum += __shfl_xor_sync(0xffffffffu, digits_sum, 1);
      digits_sum += __shfl_xor_sync(0xffffffffu, digits_sum, 2);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int column = cur_block * kRows + 8 * n + 2 * c + e;
        qsum[n][e] = __shfl_sync(0xffffffffu, digits_sum, 8 * c + 4 * e);
        qscale[n][e] = __shfl_sync(0xffffffffu, unit, 8 * c + 4 * e);
        limit[n][e] = column < cur_rows ? max(0, s.keys - s.rows + p.group.quotient(column) + 1) : 0x7fffffff;
        least = min(least, limit[n][e]);
        m[n][e] = -INFINITY;
        sum[n][e] = 0.f;
      }
      value_units[n] = kFirstUnits;
#pragma unroll
      for (int k = 0; k < 4 * kVWords; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[k][n][j] = 0.f;
    }
    least = __reduce_min_sync(0xffffffffu, least);
  };
  float* const head_slot = params.slots + (2ll * gridDim.x + static_cast<long long>(blockIdx.x) * kWarps + warp) * Cfg::kPieceFloats;

  int stage = 0;
  // The first kStages rounds only fill the ring. Every round closes one group of copies, empty ones too: the waits count groups.
#pragma unroll 1
  for (int it = -kStages; it < count; ++it) {
    int4 info = make_int4(0, 0, 0, 0);
    if (it >= 0) {
      info = infos[warp][stage];
      cur_tile = info.w >> (kParts + 1);
      if (fresh) {
        fresh = false;
        cur_b = info.x; cur_head = info.y; cur_block = info.z;
        first_tile = cur_tile;
        load_queries();
      }
      copies_wait<kStages - 1>();
      __syncwarp();
      const uint8_t* keys_at = ring + (warp * kStages + stage) * Cfg::kStageBytes;
      const uint8_t* values_at = keys_at + Cfg::kCodeBytes + Cfg::kPairBytes;
      const int first = cur_tile * kTile;
      // not whole: a tile with tokens behind the last one that some row sees, or on a page that could not be followed
      const bool whole = first + kTile <= least && (info.w & ((1 << kParts) - 1)) == (1 << kParts) - 1;
      auto usable = [&](int t) { return (info.w >> (t >> 4)) & 1; };

      // S^T = K Q^T, complete (query unit, then key scale: an integer sum times a key scale may leave FP32's range) before
      // keys are hidden, so that hidden ones count for nothing whatever the unit is
      float s[kParts][kQ][4], top[kQ][2], vscale[kParts][2];
#pragma unroll
      for (int n = 0; n < kQ; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
      for (int m2 = 0; m2 < kParts; m2 += 2) {
        int high[2][kQ][4], low[2][kQ][4];
#pragma unroll
        for (int j = 0; j < kKWords; j += kLoad) {
          uint32_t wa[2][kLoad], wb[2][kLoad];           // two parts side by side: four independent sums
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint8_t* at = keys_at + 16 * (m2 + u) * (kDim / 2) + (key_at ^ 16 * j);
            lds_words(at, wa[u]);
            lds_words(at + 8 * (kDim / 2), wb[u]);
          }
#pragma unroll
          for (int k = 0; k < kLoad; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t a0 = wa[u][k] & 0x0f0f0f0fu, a1 = wb[u][k] & 0x0f0f0f0fu, a2 = (wa[u][k] >> 4) & 0x0f0f0f0fu, a3 = (wb[u][k] >> 4) & 0x0f0f0f0fu;
#pragma unroll
              for (int n = 0; n < kQ; ++n) {
                const uint32_t(&d)[4] = q[j + k][n];
                if (j + k == 0) {
                  mma_u8s8_first(high[u][n], a0, a1, a2, a3, d[0], d[1]);
                  mma_u8s8_first(low[u][n], a0, a1, a2, a3, d[2], d[3]);
                } else {
                  mma_u8s8(high[u][n], a0, a1, a2, a3, d[0], d[1]);
                  mma_u8s8(low[u][n], a0, a1, a2, a3, d[2], d[3]);
                }
              }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int mt = m2 + u, t = 16 * mt + turned + 8 * r;
            const uint32_t key_pair = lds32(keys_at + Cfg::kCodeBytes + 4 * t);
            vscale[mt][r] = bf16_lo(lds32(values_at + Cfg::kCodeBytes + 4 * t));
            const float kscale = bf16_lo(key_pair);
            const int zero = __float2int_rn(bf16_hi(key_pair));
#pragma unroll
            for (int n = 0; n < kQ; ++n) {
              float x[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) x[e] = static_cast<float>(high[u][n][2 * r + e] * 256 + low[u][n][2 * r + e] - zero * qsum[n][e]);
              // two to an instruction, but for dim 256 with sixteen rows, whose registers are all taken (174 us packed, 159 not, for
              // 32 sequences of 8192 keys, 12 query heads on each of 4 key heads; 16 on 4 of dim 128 72 packed, 74 not)
              float2 score = make_float2(x[0] * qscale[n][0] * kscale, x[1] * qscale[n][1] * kscale);
              if constexpr (kDim * kQ < 512)
                score = __fmul2_rn(__fmul2_rn(make_float2(x[0], x[1]), make_float2(qscale[n][0], qscale[n][1])), make_float2(kscale, kscale));
              s[mt][n][2 * r] = score.x;
              s[mt][n][2 * r + 1] = score.y;
            }
          }
      }
      if (!whole) {
#pragma unroll
        for (int mt = 0; mt < kParts; ++mt)
#pragma unroll
          for (int n = 0; n < kQ; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = 16 * mt + turned + 8 * (j / 2);
              if (first + t >= limit[n][j % 2] || !usable(t)) s[mt][n][j] = -INFINITY;
            }
      }
#pragma unroll
      for (int mt = 0; mt < kParts; ++mt)
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) top[n][j % 2] = fmaxf(top[n][j % 2], s[mt][n][j]);
      float tile_scale = 0.f;
#pragma unroll
      for (int mt = 0; mt < kParts; ++mt) tile_scale = fmaxf(tile_scale, fmaxf(vscale[mt][0], vscale[mt][1]));
      tile_scale = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(tile_scale)));
      bool grows = !whole;                               // rows see different scales there: looked at below
#pragma unroll
      for (int n = 0; n < kQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 4));
          top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 8));
          top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 16));
          grows |= top[n][e] > m[n][e] + 8.f || tile_scale * value_unit(n, e) > 128.f;
        }
      // The maximum follows only when it has grown by more than 2^8 (weights up to 256 fit), so that the output is rarely
      // scaled again.
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float seen = tile_scale, turn = 1.f;         // the largest of the values' scales that the row sees
            if (!whole) {
              seen = 0.f;
#pragma unroll
              for (int mt = 0; mt < kParts; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                  if (s[mt][n][2 * r + e] != -INFINITY) seen = fmaxf(seen, vscale[mt][r]);
#pragma unroll
              for (int d = 4; d < 32; d *= 2) seen = fmaxf(seen, __shfl_xor_sync(0xffffffffu, seen, d));
            }
            if (seen * value_unit(n, e) > 128.f) {
              const float unit = 128.f / __uint_as_float((__float_as_uint(seen) + 0x007fffffu) & 0xff800000u);
              turn = unit / value_unit(n, e);
              value_units[n] = __byte_perm(value_units[n], __float_as_uint(unit), e ? 0x7610 : 0x3276);
            }
            const float next = fmaxf(m[n][e], top[n][e]);
            float keep = next == -INFINITY ? 1.f : fast_exp2(m[n][e] - next);
            m[n][e] = next;
            sum[n][e] *= keep;
            keep *= turn;
#pragma unroll
            for (int k = 0; k < 4 * kVWords; ++k) {
              o[k][n][e] *= keep;
              o[k][n][2 + e] *= keep;
            }
          }
      }
      // weights, times the values' scales, transposed into the second product's operand
      uint32_t w[kParts][kQ][2];
      float base[kQ][2];
#pragma unroll
      for (int n = 0; n < kQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) base[n][e] = m[n][e] == -INFINITY ? 0.f : -m[n][e];
#pragma unroll
      for (int mt = 0; mt < kParts; ++mt) {
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float weight[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              weight[e] = fast_exp2(s[mt][n][2 * r + e] + base[n][e]);
              sum[n][e] += weight[e];
            }
            // in this order: a hidden key's weight is 0, and its scale times the row's unit may leave FP32's range
            const float2 x = __fmul2_rn(__fmul2_rn(make_float2(weight[0], weight[1]), make_float2(value_unit(n, 0), value_unit(n, 1))),
                                        make_float2(vscale[mt][r], vscale[mt][r]));
            w[mt][n][r] = transpose8x8(pack_f16(x.x, x.y));
          }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int mt = 0; mt < kParts; ++mt) {
        uint32_t minus_low[2], minus_high[2], v[4][kVWords];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int ta = 16 * mt + 8 * r + t_even, tb = 16 * mt + 8 * r + t_odd;
          const uint32_t pa = lds32(values_at + Cfg::kCodeBytes + 4 * ta), pb = lds32(values_at + Cfg::kCodeBytes + 4 * tb);
          // 128 + zero as BF16 has the zero point in its low bits, which then make -(1024 + zero) as FP16
          uint32_t zeros = __byte_perm(pa, pb, 0x7632);
          asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(zeros) : "r"(0x43004300u));
          minus_low[r] = (zeros & 0x000f000fu) | 0xe400e400u;
          asm("add.rn.f16x2 %0, %1, %2;" : "=r"(minus_high[r]) : "r"(minus_low[r]), "r"(0x63806380u));   // + 960
          lds_words(values_at + (16 * mt + 8 * r) * (kDim / 2) + even_at, v[2 * r]);
          lds_words(values_at + (16 * mt + 8 * r) * (kDim / 2) + odd_at, v[2 * r + 1]);
        }
#pragma unroll
        for (int k = 0; k < kVWords; ++k) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {           // components 0, 1 (4, 5), then 2, 3 (6, 7) of the word
            const uint32_t lo0 = __byte_perm(v[0][k], v[1][k], half ? 0x0501 : 0x0400), hi0 = __byte_perm(v[0][k], v[1][k], half ? 0x0703 : 0x0602);
            const uint32_t lo1 = __byte_perm(v[2][k], v[3][k], half ? 0x0501 : 0x0400), hi1 = __byte_perm(v[2][k], v[3][k], half ? 0x0703 : 0x0602);
            const uint32_t a0 = code_pair<0>(lo0, ones, minus_low[0], minus_high[0]), a1 = code_pair<0>(hi0, ones, minus_low[0], minus_high[0]);
            const uint32_t a2 = code_pair<0>(lo1, ones, minus_low[1], minus_high[1]), a3 = code_pair<0>(hi1, ones, minus_low[1], minus_high[1]);
            const uint32_t b0 = code_pair<1>(lo0, ones, minus_low[0], minus_high[0]), b1 = code_pair<1>(hi0, ones, minus_low[0], minus_high[0]);
            const uint32_t b2 = code_pair<1>(lo1, ones, minus_low[1], minus_high[1]), b3 = code_pair<1>(hi1, ones, minus_low[1], minus_high[1]);
#pragma unroll
            for (int n = 0; n < kQ; ++n) {
              mma_f16(o[4 * k + 2 * half][n], a0, a1, a2, a3, w[mt][n][0], w[mt][n][1]);
              mma_f16(o[4 * k + 2 * half + 1][n], b0, b1, b2, b3, w[mt][n][0], w[mt][n][1]);
            }
          }
        }
      }
      __syncwarp();                                      // every lane has read the stage
    }
    if (it + kStages < count) issue(stage);
    copies_commit();
    if (++stage == kStages) stage = 0;
    if (info.w >> kParts & 1) {                          // the last tile of these rows
      add_sums();
      if (first_tile == 0) {
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = cur_block * kRows + 8 * n + 2 * c + e;
            if (row >= cur_rows) continue;
            const float inverse = sum[n][e] == 0.f ? 0.f : 1.f / value_unit(n, e) / sum[n][e];
            const int row_token = p.group.quotient(row);
            uint16_t* dst = p.out + (static_cast<int64_t>(cur_start + row_token) * p.q_heads + cur_head * group + row - row_token * group) * kDim;
#pragma unroll
            for (int k = 0; k < kVWords; ++k) {
              float x[8];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                x[j] = o[4 * k + j][n][e] * inverse;
                x[4 + j] = o[4 * k + j][n][2 + e] * inverse;
              }
              *reinterpret_cast<uint4*>(dst + 8 * (kVWords * g + k)) = pack8(x);
            }
          }
      } else {
        write_piece(2 * warp, head_slot);                // only the first sequence of a range can have begun before it
        if (lane == 0)
          pieces[2 * warp] = Kv4Piece{1, 0, range + it - cur_tile, cur_tile + 1u, cur_start, cur_block * kRows,
                                      min(kRows, cur_rows - cur_block * kRows), cur_head};
      }
      fresh = true;
    }
  }
  if (!fresh) {                                          // the range ends inside a sequence: kept in the ring, which is idle now
    add_sums();
    write_piece(2 * warp + 1, reinterpret_cast<float*>(ring + warp * kStages * Cfg::kStageBytes));
    if (lane == 0)
      pieces[2 * warp + 1] = Kv4Piece{2, first_tile == 0, range + count - 1 - cur_tile, static_cast<unsigned>(kv4_block_tiles<kTile>(cur_keys)),
                                      cur_start, cur_block * kRows, min(kRows, cur_rows - cur_block * kRows), cur_head};
  }
  __syncthreads();

  // ---- the warps' pieces, in order: an open piece belongs with those behind it up to the one that ends the sequence.
  // Groups of pieces as bit masks, the same in every warp.
  const int kind = lane < 2 * kWarps ? pieces[lane].kind : 0;
  const uint32_t present = __ballot_sync(0xffffffffu, kind != 0), ends = __ballot_sync(0xffffffffu, kind == 1);
  if (!present) return;
  const uint32_t last_end = ends ? 31 - __clz(ends) : 0;
  const int groups = __popc(ends) + ((ends ? present >> last_end >> 1 : present) != 0 ? 1 : 0);
  auto group_mask = [&](int piece) {                     // the pieces of this piece's group
    const uint32_t below = (1u << piece) - 1, before = ends & below, behind = ends & ~below;
    const uint32_t low = before ? ~((2u << (31 - __clz(before))) - 1) : ~0u;
    const uint32_t high = behind ? (2u << (__ffs(behind) - 1)) - 1 : ~0u;
    return present & low & high;
  };
  for (int i = thread; i < 2 * kWarps * kRows; i += kThreads) {
    const int piece = i / kRows, row = i % kRows;
    if (!(present >> piece & 1)) continue;
    const uint32_t mask = group_mask(piece);
    float most = -INFINITY, all = 0.f;
    for (uint32_t rest = mask; rest; rest &= rest - 1) most = fmaxf(most, piece_m[__ffs(rest) - 1][row]);
    auto part = [&](int other) {
      const float l = piece_l[other][row];
      return l == 0.f ? 0.f : fast_exp2(piece_m[other][row] - most) * l;     // 0: saw no key (a NaN score makes the sum NaN, which is kept)
    };
    for (uint32_t rest = mask; rest; rest &= rest - 1) all += part(__ffs(rest) - 1);
    if (piece == __ffs(mask) - 1) {
      group_m[piece][row] = most;
      group_l[piece][row] = all;
    }
    weights[piece][row] = all == 0.f ? 0.f : part(piece) / all;
  }
  __syncthreads();
  auto write_out = [&](const Kv4Piece& unit, int row, int column, const float4& x) {
    const int r = unit.row + row, row_token = p.group.quotient(r);
    uint16_t* dst = p.out + (static_cast<int64_t>(unit.start + row_token) * p.q_heads + unit.head * group + r - row_token * group) * kDim + column;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
  };
  const float* const head_slots = params.slots + (2ll * gridDim.x + static_cast<long long>(blockIdx.x) * kWarps) * Cfg::kPieceFloats;
  constexpr int kColumns = kDim / 4;
  for (int i = thread; i < groups * kRows * kColumns; i += kThreads) {
    const int column = i % kColumns * 4, row = i / kColumns % kRows;
    uint32_t rest = present;                             // the group's first piece: the first behind the last end before it
    for (int skip = i / (kColumns * kRows), n = 0; n < skip; ++n) rest &= ~((2u << (__ffs(rest & ends) - 1)) - 1);
    const int piece = __ffs(rest) - 1;
    const Kv4Piece unit = pieces[piece];
    if (row >= unit.rows) continue;
    const uint32_t mask = group_mask(piece);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (rest = mask; rest; rest &= rest - 1) {
      const int other = __ffs(rest) - 1;
      const float* from = other & 1 ? reinterpret_cast<const float*>(ring + (other / 2) * kStages * Cfg::kStageBytes)
                                    : head_slots + (other / 2) * Cfg::kPieceFloats;
      const float weight = weights[other][row];
      if (weight == 0.f) continue;
      const float4 y = *reinterpret_cast<const float4*>(from + row * kDim + column);
      x.x += weight * y.x; x.y += weight * y.y; x.z += weight * y.z; x.w += weight * y.w;
    }
    if (unit.starts && (mask & ends)) {
      write_out(unit, row, column, x);
    } else {
      float* slot = params.slots + (2ll * blockIdx.x + (unit.starts ? 1 : 0)) * Cfg::kPieceFloats;
      if (column == 0) {
        slot[row] = group_m[piece][row];
        slot[kRows + row] = group_l[piece][row];
        if (row == 0) shared_units[unit.starts ? 1 : 0] = unit;
      }
      *reinterpret_cast<float4*>(slot + 2 * kRows + row * kDim + column) = x;
    }
  }
  __syncthreads();

  // ---- sequences shared by several CTAs: the last to arrive joins the CTAs' slots in order and leaves the counter at zero
  auto cta_of = [&](unsigned place) -> int {
    const unsigned of_longer = longer * (per_cta + 1);
    return place < of_longer ? place / (per_cta + 1) : longer + (place - of_longer) / per_cta;
  };
  if (thread < 2 && shared_units[thread].kind) {
    const Kv4Piece& unit = shared_units[thread];
    const int from = cta_of(unit.first), to = cta_of(unit.first + unit.tiles - 1);
    __threadfence();
    if (atomicAdd(params.counters + from, 1u) == static_cast<unsigned>(to - from)) {
      params.counters[from] = 0;
      comes_last[thread] = 1;
    }
    __threadfence();
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    if (!comes_last[which]) continue;
    const Kv4Piece unit = shared_units[which];
    const int from = cta_of(unit.first), count_ctas = cta_of(unit.first + unit.tiles - 1) - from + 1;
    const int rows = unit.rows;
    const float* slots = params.slots + 2ll * from * Cfg::kPieceFloats;   // slot 1 of the first CTA, slot 0 of the others
    auto slot_of = [&](int i) { return slots + (2ll * i + (i == 0 ? 1 : 0)) * Cfg::kPieceFloats; };
    float* cta_weights = reinterpret_cast<float*>(ring);                  // [CTA][row]; the pieces in the ring are done with
    for (int row = warp; row < rows; row += kWarps) {
      float most = -INFINITY, all = 0.f;
      for (int i = lane; i < count_ctas; i += 32) most = fmaxf(most, __ldcg(slot_of(i) + row));
#pragma unroll
      for (int d = 16; d; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      for (int i = lane; i < count_ctas; i += 32) {
        const float part_sum = __ldcg(slot_of(i) + kRows + row);
        const float part = part_sum == 0.f ? 0.f : fast_exp2(__ldcg(slot_of(i) + row) - most) * part_sum;
        cta_weights[i * kRows + row] = part;
        all += part;
      }
#pragma unroll
      for (int d = 16; d; d /= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
      if (all != 0.f)
        for (int i = lane; i < count_ctas; i += 32) cta_weights[i * kRows + row] /= all;
    }
    __syncthreads();
    for (int e = thread; e < rows * (kDim / 4); e += kThreads) {
      const int row = e / (kDim / 4), column = e % (kDim / 4) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < count_ctas; ++i) {
        const float weight = cta_weights[i * kRows + row];
        const float4 y = __ldcg(reinterpret_cast<const float4*>(slot_of(i) + 2 * kRows + row * kDim + column));
        x.x += weight * y.x; x.y += weight * y.y; x.z += weight * y.z; x.w += weight * y.w;
      }
      write_out(unit, row, column, x);
    }
    __syncthreads();
  }
}

}  // namespace ci8
