// Attention of few query rows per sequence (generated tokens) over the 4-bit key/value cache: bound by reading the
// cache, dim / 2 + 4 bytes per token and side.
//
// Work is cut into tiles of 32 tokens of one (sequence, key head, block of query rows) and the tiles of all of them,
// laid end to end, are dealt to the warps in equal contiguous ranges, so that ragged batches fill the GPU evenly and
// a long history is split as far as there are warps. Every warp runs on its own: its ring of tiles is filled by bulk
// copies it issues itself, and it keeps its own running maximum, sum and output. Ranges begin and end inside a
// sequence; what a warp has of such a sequence is joined with its neighbours' inside the CTA at the end, and across
// CTAs by whichever of them comes last, in the order of the CTAs (so the bits do not depend on the timing).
//
// The products run transposed on the tensor cores with register-fed operands: S^T[token, query] = K Q^T and
// O^T[component, query] = V^T P^T (mma.sync m16n8k16), so that eight query rows fill an instruction and the cache is
// the operand that is unpacked on the way, straight from its packed words: four bits become the BF16 number
// 128 + code by one mask-and-or. Keys keep the 128 (it is taken out of the score, exactly scaled, as
// (128 + zero) * sum of q); values are made exact small integers code - zero by one packed subtraction, because
// their products are summed over the whole history. The values' scales go into the weights before they are rounded
// to BF16 for the second product (2^-9 relative each, the size of the output's own rounding); all else is FP32.
#pragma once
#include "kv4_attention.cuh"

namespace ci8 {

constexpr int kKv4Tile = 32;                                    // tokens per ring stage
constexpr int kKv4CounterBytes = 4096;                          // arrival counters at the head of the workspace
constexpr int kKv4MaxCtas = kKv4CounterBytes / 4;

template <int kDim, int kQ>                                     // kQ: groups of eight query rows per warp
struct Kv4SingleConfig {
  static constexpr int kRows = 8 * kQ;
  static constexpr int kWarps = kDim * kQ <= 128 ? 16 : 8;      // registers: output and queries take kDim * kQ * 3 / 8 each thread
  static constexpr int kCodeBytes = kKv4Tile * kDim / 2;
  static constexpr int kPairBytes = kKv4Tile * 4;
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

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two four-bit codes, at bits 4 * i and 16 + 4 * i of w, as the BF16 numbers 128 + code.
template <int i>
__device__ __forceinline__ uint32_t codes_pair(uint32_t w) {
  return ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&w)[1]) { w[0] = lds32(at); }
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&w)[2]) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&w)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Number of keys the last row of a block of query rows sees, and the tiles they make (one at least: rows that see
// nothing have to be written too).
__device__ __forceinline__ int kv4_block_keys(const Kv4Sequence& s, int group, int rows_per_block, int block) {
  const int last = min(s.rows * group, (block + 1) * rows_per_block) - 1;
  return max(0, s.keys - s.rows + last / group + 1);
}
__device__ __forceinline__ int kv4_block_tiles(int keys) { return max(1, (keys + kKv4Tile - 1) / kKv4Tile); }
// Tiles of one key head of a sequence.
__device__ __forceinline__ long long kv4_head_tiles(const Kv4Sequence& s, int group, int rows_per_block, int most_rows) {
  const int rows = s.rows * group;
  if (rows == 0 || rows > most_rows) return 0;
  long long tiles = 0;
  for (int block = 0; block * rows_per_block < rows; ++block) tiles += kv4_block_tiles(kv4_block_keys(s, group, rows_per_block, block));
  return tiles;
}

// What a warp leaves of a sequence it shares with a neighbour.
struct Kv4Piece {
  int b, head, block, kind;       // kind: 0 none, 1 ends the sequence's tiles (in the workspace), 2 open at its end (in the ring)
  int starts;                     // it holds the first tile
  long long first, tiles;         // place of the first tile among all, number of tiles
};

template <int kDim, int kQ>
__global__ void __launch_bounds__(Kv4SingleConfig<kDim, kQ>::kWarps * 32, 1) kv4_single_kernel(const Kv4SingleParams params) {
  using Cfg = Kv4SingleConfig<kDim, kQ>;
  constexpr int kWarps = Cfg::kWarps, kThreads = kWarps * 32, kStages = Cfg::kStages, kRows = Cfg::kRows;
  constexpr int kKWords = kDim / 32;                     // a lane's words of a key row
  constexpr int kVWords = kDim / 64;                     // a lane's words of a value row
  constexpr int kLoad = kKWords > 4 ? 4 : kKWords;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];
  __shared__ int4 infos[kWarps][kStages];
  __shared__ long long prefix[kThreads + 1];
  __shared__ Kv4Piece pieces[2 * kWarps];
  __shared__ Kv4Piece shared_units[2];                   // sequences shared with the CTA before [0] and behind [1]
  __shared__ float inverse_sums[kRows];
  __shared__ int abort_flag, comes_last[2];
  const Kv4AttendParams& p = params.a;
  const int thread = threadIdx.x, warp = thread / 32, lane = thread % 32, g = lane / 4, c = lane % 4;
  const int group = p.q_heads / p.kv_heads;

  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&bars[warp][s]), 1);
  }
  if (thread == 0) abort_flag = 0;
  if (thread < 2 * kWarps) pieces[thread].kind = 0;
  if (thread < 2) shared_units[thread].kind = comes_last[thread] = 0;
  fence_barrier_init();
  pdl_wait();
  pdl_launch_dependents();

  // ---- every tile's place: thread t sums the sequences of its share, then a scan over the threads
  const int share = (p.batch + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int b = thread * share; b < min(p.batch, (thread + 1) * share); ++b)
    mine += kv4_head_tiles(kv4_sequence(p, b), group, kRows, params.most_rows) * p.kv_heads;
  long long scan = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long other = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += other;
  }
  __shared__ long long warp_sums[kWarps];
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  long long before = 0;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
  prefix[thread + 1] = before + scan;
  if (thread == 0) prefix[0] = 0;
  __syncthreads();
  const long long total = prefix[kThreads];
  if (total == 0) return;
  // as many CTAs as give every warp a few tiles: below that, joining costs more than the tiles
  constexpr int kLeast = 2;
  long long ctas = (total + kWarps * kLeast - 1) / (kWarps * kLeast);
  if (ctas > gridDim.x) ctas = gridDim.x;
  if (blockIdx.x >= ctas) return;
  const long long workers = ctas * kWarps;
  const long long worker = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const long long range = worker * total / workers, range_end = (worker + 1) * total / workers;
  const int count = static_cast<int>(range_end - range);

  // ---- where this warp's range begins
  int b = 0, head = 0, block = 0, tile = 0, keys = 0, tiles = 0;
  Kv4Sequence seq{};
  if (count > 0) {
    int low = 0, high = kThreads;                        // the thread whose share holds the first tile
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (prefix[mid] <= range) low = mid; else high = mid;
    }
    long long rest = range - prefix[low], per_head = 0;
    for (b = low * share;; ++b) {
      seq = kv4_sequence(p, b);
      per_head = kv4_head_tiles(seq, group, kRows, params.most_rows);
      if (rest < per_head * p.kv_heads) break;
      rest -= per_head * p.kv_heads;
    }
    head = static_cast<int>(rest / per_head);
    rest -= head * per_head;
    for (block = 0;; ++block) {
      keys = kv4_block_keys(seq, group, kRows, block);
      tiles = kv4_block_tiles(keys);
      if (rest < tiles) break;
      rest -= tiles;
    }
    tile = static_cast<int>(rest);
  }

  // ---- the loader's side of the ring: tiles of the range in order, one ahead of what it has issued (page numbers are
  // fetched one tile early)
  const int page = 1 << p.page_shift;
  const int64_t block_bytes = kv4_block_bytes(page, kDim);
  const uint32_t ring_base = smem_u32(ring) + warp * kStages * Cfg::kStageBytes;
  const int part_rows = page < kKv4Tile ? page : kKv4Tile, parts = kKv4Tile / part_rows;
  const int part = lane >> 2, piece_of = lane & 3;       // lanes 0..4 * parts - 1 issue a copy each
  int page_id = -1;
  auto fetch_page = [&]() {
    const int token = tile * kKv4Tile + part * part_rows;
    page_id = -1;
    if (part < parts && token < keys) page_id = p.block_table[static_cast<int64_t>(b) * p.width + (token >> p.page_shift)];
  };
  auto issue = [&](int stage) {
    const int token = tile * kKv4Tile + part * part_rows;
    const int rows = part < parts ? min(part_rows, max(0, keys - token)) : 0;
    const bool wanted = rows > 0, good = wanted && page_id >= 0 && page_id < p.pages;
    if (wanted && !good && piece_of == 0) atomicOr(&g_ci8_status, kStatusBadIndex);
    const int copied = good ? (rows + 3) & ~3 : 0;       // rows in fours: 16-byte multiples
    const uint32_t bytes = piece_of & 1 ? copied * 4 : copied * (kDim / 2);
    const uint32_t goods = __ballot_sync(0xffffffffu, good);
    const uint32_t sum = __reduce_add_sync(0xffffffffu, bytes);
    const uint32_t bar = smem_u32(&bars[warp][stage]);
    if (lane == 0) {
      const int flags = (goods & 1u ? 1 : 0) | (goods & 16u ? 2 : 0) | (tile == tiles - 1 ? 4 : 0);
      infos[warp][stage] = make_int4(b, head, block, (tile << 3) | flags);
      mbar_arrive_expect_tx(bar, sum);
    }
    __syncwarp();
    if (bytes) {
      const uint8_t* src = p.cache + ((static_cast<int64_t>(page_id) * kKv4Side + (piece_of >> 1)) * p.kv_heads + head) * block_bytes;
      const int row = token & (page - 1);
      src += piece_of & 1 ? page * (kDim / 2) + 4 * row : row * (kDim / 2);
      const uint32_t dst = ring_base + stage * Cfg::kStageBytes + (piece_of >> 1) * (Cfg::kCodeBytes + Cfg::kPairBytes) +
                           (piece_of & 1 ? Cfg::kCodeBytes + part * part_rows * 4 : part * part_rows * (kDim / 2));
      bulk_load(dst, src, bytes, bar);
    }
    // the next tile
    if (++tile == tiles) {
      tile = 0;
      if (++block * kRows >= seq.rows * group) {
        block = 0;
        if (++head == p.kv_heads) {
          head = 0;
          do {
            ++b;
            if (b < p.batch) seq = kv4_sequence(p, b);
          } while (b < p.batch && (seq.rows == 0 || seq.rows * group > params.most_rows));
        }
      }
      if (b < p.batch) {
        keys = kv4_block_keys(seq, group, kRows, block);
        tiles = kv4_block_tiles(keys);
      }
    }
    if (b < p.batch) fetch_page();
  };
  int issued = 0;
  if (count > 0) fetch_page();
  for (; issued < min(count, kStages); ++issued) issue(issued);

  // ---- the consumer's side
  float o[4 * kVWords][kQ][4];
  float m[kQ][2], sum[kQ][2], qsum[kQ][2];
  int limit[kQ][2];
  uint32_t q[2 * kKWords][kQ][2];
  int cur_b = 0, cur_head = 0, cur_block = 0, cur_tile = 0, cur_rows = 0, cur_start = 0, cur_keys = 0, unit_first_tile = 0;
  int least = 0;
  bool fresh = true, open = false;
  const int turned = g ^ ((g >> 1) & 1);                 // which token of eight a row of S^T holds: spreads the reads over the banks
  const int t_even = 2 * c ^ (c & 1), t_odd = (2 * c + 1) ^ (c & 1);

  // Writes this warp's maximum, sum and output of every row: [maximum][sum][output].
  auto write_piece = [&](float* dst) {
#pragma unroll
    for (int n = 0; n < kQ; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * n + 2 * c + e;
        if (g == 0) {
          dst[row] = m[n][e];
          dst[kRows + row] = sum[n][e];
        }
#pragma unroll
        for (int k = 0; k < kVWords; ++k) {
          float4* to = reinterpret_cast<float4*>(dst + 2 * kRows + row * kDim + 8 * (kVWords * g + k));
          to[0] = make_float4(o[4 * k][n][e], o[4 * k + 1][n][e], o[4 * k + 2][n][e], o[4 * k + 3][n][e]);
          to[1] = make_float4(o[4 * k][n][2 + e], o[4 * k + 1][n][2 + e], o[4 * k + 2][n][2 + e], o[4 * k + 3][n][2 + e]);
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
  float* const head_slot = params.slots + (2ll * gridDim.x + worker) * Cfg::kPieceFloats;

  for (int it = 0; it < count; ++it) {
    const int stage = it % kStages;
    if (!mbar_wait(smem_u32(&bars[warp][stage]), (it / kStages) & 1, &abort_flag)) {
      int gave_up = 0;                                   // the copies in flight still write here: wait for them, with the same limit
      for (int k = it; k < issued && !gave_up; ++k) mbar_wait(smem_u32(&bars[warp][k % kStages]), (k / kStages) & 1, &gave_up);
      break;
    }
    const int4 info = infos[warp][stage];
    cur_tile = info.w >> 3;
    if (fresh) {
      fresh = false;
      open = true;
      cur_b = info.x; cur_head = info.y; cur_block = info.z;
      unit_first_tile = cur_tile;
      const Kv4Sequence s = kv4_sequence(p, cur_b);
      cur_rows = s.rows * group;
      cur_start = s.start;
      cur_keys = kv4_block_keys(s, group, kRows, cur_block);
      least = 0x7fffffff;
#pragma unroll
      for (int n = 0; n < kQ; ++n) {
        // queries: lane (g, c) holds row g's words c, in the order in which the keys' codes come out of a word
        const int row = cur_block * kRows + 8 * n + g;
        float part_sum = 0.f;
#pragma unroll
        for (int k = 0; k < kKWords; ++k) {
          const int word = kLoad * c + (k % kLoad) + (k / kLoad) * 4 * kLoad;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (row < cur_rows)
            w = *reinterpret_cast<const uint4*>(p.q + (cur_start + row / group) * p.q_stride +
                                                static_cast<int64_t>(cur_head * group + row % group) * kDim + 8 * word);
          float x[8];
          unpack8(w, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) part_sum += x[j];
          q[2 * k][n][0] = __byte_perm(w.x, w.z, 0x5410);
          q[2 * k][n][1] = __byte_perm(w.x, w.z, 0x7632);
          q[2 * k + 1][n][0] = __byte_perm(w.y, w.w, 0x5410);
          q[2 * k + 1][n][1] = __byte_perm(w.y, w.w, 0x7632);
        }
        part_sum += __shfl_xor_sync(0xffffffffu, part_sum, 1);
        part_sum += __shfl_xor_sync(0xffffffffu, part_sum, 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int column = cur_block * kRows + 8 * n + 2 * c + e;
          qsum[n][e] = __shfl_sync(0xffffffffu, part_sum, 8 * c + 4 * e);
          limit[n][e] = column < cur_rows ? max(0, s.keys - s.rows + column / group + 1) : 0x7fffffff;
          least = min(least, limit[n][e]);
          m[n][e] = -INFINITY;
          sum[n][e] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 4 * kVWords; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[k][n][j] = 0.f;
      }
      least = __reduce_min_sync(0xffffffffu, least);
    }
    const uint32_t keys_at = ring_base + stage * Cfg::kStageBytes, values_at = keys_at + Cfg::kCodeBytes + Cfg::kPairBytes;
    const int first = cur_tile * kKv4Tile;
    // a tile with tokens behind the last one some row sees, or on a page that could not be followed
    const bool whole = first + kKv4Tile <= least && (info.w & 3) == (parts == 2 ? 3 : 1);
    auto usable = [&](int t) { return (info.w >> (parts == 2 ? t >> 4 : 0)) & 1; };

    // S^T = K Q^T
    float s[2][kQ][4];
    float kscale[2][2], kzero[2][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int n = 0; n < kQ; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[mt][n][j] = 0.f;
      const int t0 = 16 * mt + turned;
#pragma unroll
      for (int j = 0; j < kKWords; j += kLoad) {
        uint32_t wa[kLoad], wb[kLoad];
        const uint32_t at = keys_at + t0 * (kDim / 2) + 4 * (kLoad * c + j * 4);
        lds_words(at, wa);
        lds_words(at + 8 * (kDim / 2), wb);
#pragma unroll
        for (int k = 0; k < kLoad; ++k) {
#pragma unroll
          for (int n = 0; n < kQ; ++n)
            mma_bf16(s[mt][n], codes_pair<0>(wa[k]), codes_pair<0>(wb[k]), codes_pair<1>(wa[k]), codes_pair<1>(wb[k]),
                     q[2 * (j + k)][n][0], q[2 * (j + k)][n][1]);
#pragma unroll
          for (int n = 0; n < kQ; ++n)
            mma_bf16(s[mt][n], codes_pair<2>(wa[k]), codes_pair<2>(wb[k]), codes_pair<3>(wa[k]), codes_pair<3>(wb[k]),
                     q[2 * (j + k) + 1][n][0], q[2 * (j + k) + 1][n][1]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t pair = lds32(keys_at + Cfg::kCodeBytes + 4 * (t0 + 8 * r));
        kscale[mt][r] = bf16_lo(pair) * p.scale_log2;
        kzero[mt][r] = -128.f - bf16_hi(pair);
      }
    }
    float top[kQ][2];
#pragma unroll
    for (int n = 0; n < kQ; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int n = 0; n < kQ; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = fmaf(kzero[mt][j / 2], qsum[n][j % 2], s[mt][n][j]) * kscale[mt][j / 2];
          if (!whole) {
            const int t = 16 * mt + turned + 8 * (j / 2);
            if (first + t >= limit[n][j % 2] || !usable(t)) x = -INFINITY;
          }
          s[mt][n][j] = x;
          top[n][j % 2] = fmaxf(top[n][j % 2], x);
        }
    bool grows = false;
#pragma unroll
    for (int n = 0; n < kQ; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 4));
        top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 8));
        top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(0xffffffffu, top[n][e], 16));
        grows |= top[n][e] > m[n][e] + 8.f;
      }
    // The maximum follows only when it has grown by more than 2^8: weights up to 256 cost nothing in FP32 or BF16, and
    // the output is rarely scaled again.
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int n = 0; n < kQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float next = fmaxf(m[n][e], top[n][e]);
          const float keep = next == -INFINITY ? 1.f : fast_exp2(m[n][e] - next);
          m[n][e] = next;
          sum[n][e] *= keep;
#pragma unroll
          for (int k = 0; k < 4 * kVWords; ++k) {
            o[k][n][e] *= keep;
            o[k][n][2 + e] *= keep;
          }
        }
    }
    // weights, times the values' scales, transposed into the second product's operand
    uint32_t w[2][kQ][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      float vscale[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int t = 16 * mt + turned + 8 * r;
        uint32_t pair = lds32(values_at + Cfg::kCodeBytes + 4 * t);
        if (!whole && (first + t >= cur_keys || !usable(t))) pair = 0;
        vscale[r] = bf16_lo(pair);
      }
#pragma unroll
      for (int n = 0; n < kQ; ++n) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float base = m[n][j % 2] == -INFINITY ? 0.f : m[n][j % 2];
          const float weight = fast_exp2(s[mt][n][j] - base);
          sum[n][j % 2] += weight;
          x[j] = weight * vscale[j / 2];
        }
        w[mt][n][0] = transpose8x8(pack2(x[0], x[1]));
        w[mt][n][1] = transpose8x8(pack2(x[2], x[3]));
      }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t zero[2];
      uint32_t v[4][kVWords];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int ta = 16 * mt + 8 * r + t_even, tb = 16 * mt + 8 * r + t_odd;
        uint32_t pa = lds32(values_at + Cfg::kCodeBytes + 4 * ta), pb = lds32(values_at + Cfg::kCodeBytes + 4 * tb);
        if (!whole) {
          if (first + ta >= cur_keys || !usable(ta)) pa = 0;
          if (first + tb >= cur_keys || !usable(tb)) pb = 0;
        }
        zero[r] = add_bf16x2(__byte_perm(pa, pb, 0x7632), 0x43004300u);
        lds_words(values_at + ta * (kDim / 2) + 4 * kVWords * g, v[2 * r]);
        lds_words(values_at + tb * (kDim / 2) + 4 * kVWords * g, v[2 * r + 1]);
      }
#pragma unroll
      for (int k = 0; k < kVWords; ++k) {
        const uint32_t lo0 = __byte_perm(v[0][k], v[1][k], 0x5410), hi0 = __byte_perm(v[0][k], v[1][k], 0x7632);
        const uint32_t lo1 = __byte_perm(v[2][k], v[3][k], 0x5410), hi1 = __byte_perm(v[2][k], v[3][k], 0x7632);
        auto step = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
          a0 = sub_bf16x2(a0, zero[0]);
          a1 = sub_bf16x2(a1, zero[0]);
          a2 = sub_bf16x2(a2, zero[1]);
          a3 = sub_bf16x2(a3, zero[1]);
#pragma unroll
          for (int n = 0; n < kQ; ++n) mma_bf16(o[4 * k + i][n], a0, a1, a2, a3, w[mt][n][0], w[mt][n][1]);
        };
        step(0, codes_pair<0>(lo0), codes_pair<0>(hi0), codes_pair<0>(lo1), codes_pair<0>(hi1));
        step(1, codes_pair<1>(lo0), codes_pair<1>(hi0), codes_pair<1>(lo1), codes_pair<1>(hi1));
        step(2, codes_pair<2>(lo0), codes_pair<2>(hi0), codes_pair<2>(lo1), codes_pair<2>(hi1));
        step(3, codes_pair<3>(lo0), codes_pair<3>(hi0), codes_pair<3>(lo1), codes_pair<3>(hi1));
      }
    }
    __syncwarp();                                        // every lane has read the stage
    if (issued < count) {
      issue(stage);
      ++issued;
    }
    if (info.w & 4) {                                    // the last tile of these rows
      add_sums();
      if (unit_first_tile == 0) {
#pragma unroll
        for (int n = 0; n < kQ; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = cur_block * kRows + 8 * n + 2 * c + e;
            if (row >= cur_rows) continue;
            const float inverse = sum[n][e] == 0.f ? 0.f : 1.f / sum[n][e];
            uint16_t* dst = p.out + (static_cast<int64_t>(cur_start + row / group) * p.q_heads + cur_head * group + row % group) * kDim;
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
        write_piece(head_slot);
        if (lane == 0) {
          // only the first sequence of a range can have begun before it
          pieces[2 * warp] = Kv4Piece{cur_b, cur_head, cur_block, 1, 0, range + it - cur_tile, cur_tile + 1};
        }
      }
      fresh = true;
      open = false;
    }
  }
  if (open) {                                            // the range ends inside a sequence: kept in the ring, which is idle now
    add_sums();
    write_piece(reinterpret_cast<float*>(ring + warp * kStages * Cfg::kStageBytes));
    if (lane == 0) {
      const Kv4Sequence s = kv4_sequence(p, cur_b);
      const int all = kv4_block_tiles(kv4_block_keys(s, group, kRows, cur_block));
      pieces[2 * warp + 1] = Kv4Piece{cur_b, cur_head, cur_block, 2, unit_first_tile == 0, range_end - 1 - cur_tile, all};
    }
  }
  __syncthreads();

  // ---- the warps' pieces, in order: an open piece belongs with those behind it up to the one that ends the sequence
  auto piece_at = [&](int i) {
    return pieces[i].kind == 1 ? params.slots + (2ll * gridDim.x + static_cast<long long>(blockIdx.x) * kWarps + i / 2) * Cfg::kPieceFloats
                               : reinterpret_cast<const float*>(ring + (i / 2) * kStages * Cfg::kStageBytes);
  };
  auto write_out = [&](const Kv4Sequence& s, const Kv4Piece& unit, int row, int column, const float4& x) {
    const int r = unit.block * kRows + row;
    uint16_t* dst = p.out + (static_cast<int64_t>(s.start + r / group) * p.q_heads + unit.head * group + r % group) * kDim + column;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
  };
  for (int at = 0; at < 2 * kWarps;) {
    if (pieces[at].kind == 0) { ++at; continue; }
    const int begin = at;
    while (pieces[at].kind != 1 && ++at < 2 * kWarps) {}
    const bool ends = at < 2 * kWarps;                   // else it goes on in the next CTA
    const int end = ends ? ++at : at;
    const Kv4Piece unit = pieces[begin];
    const Kv4Sequence s = kv4_sequence(p, unit.b);
    const int rows = min(kRows, s.rows * group - unit.block * kRows);
    const bool closed = ends && unit.starts;
    float* slot = params.slots + (2ll * blockIdx.x + (unit.starts ? 1 : 0)) * Cfg::kPieceFloats;
    for (int e = thread; e < rows * (kDim / 4); e += kThreads) {
      const int row = e / (kDim / 4), column = e % (kDim / 4) * 4;
      float most = -INFINITY, all = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = begin; i < end; ++i)
        if (pieces[i].kind) most = fmaxf(most, piece_at(i)[row]);
      for (int i = begin; i < end; ++i) {
        if (!pieces[i].kind) continue;
        const float* from = piece_at(i);
        const float part_sum = from[kRows + row];
        if (part_sum == 0.f) continue;                   // saw no key (a NaN score makes its sum NaN, which is kept)
        const float weight = fast_exp2(from[row] - most);
        const float4 y = *reinterpret_cast<const float4*>(from + 2 * kRows + row * kDim + column);
        all += weight * part_sum;
        x.x += weight * y.x; x.y += weight * y.y; x.z += weight * y.z; x.w += weight * y.w;
      }
      if (closed) {
        const float inverse = all == 0.f ? 0.f : 1.f / all;
        write_out(s, unit, row, column, make_float4(x.x * inverse, x.y * inverse, x.z * inverse, x.w * inverse));
      } else {
        if (column == 0) { slot[row] = most; slot[kRows + row] = all; }
        *reinterpret_cast<float4*>(slot + 2 * kRows + row * kDim + column) = x;
      }
    }
    if (!closed && thread == 0) shared_units[unit.starts ? 1 : 0] = unit;
  }
  __syncthreads();

  // ---- sequences shared by several CTAs: the last to arrive joins the CTAs' slots in order and leaves the counter at zero
  auto cta_of = [&](long long place) { return static_cast<int>(((place + 1) * workers - 1) / total / kWarps); };
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
    const Kv4Sequence s = kv4_sequence(p, unit.b);
    const int rows = min(kRows, s.rows * group - unit.block * kRows);
    const float* slots = params.slots + 2ll * from * Cfg::kPieceFloats;   // slot 1 of the first CTA, slot 0 of the others
    auto slot_of = [&](int i) { return slots + (2ll * i + (i == 0 ? 1 : 0)) * Cfg::kPieceFloats; };
    float* weights = reinterpret_cast<float*>(ring);                      // [CTA][row]; the pieces in the ring are done with
    for (int row = warp; row < rows; row += kWarps) {
      float most = -INFINITY, all = 0.f;
      for (int i = lane; i < count_ctas; i += 32) most = fmaxf(most, __ldcg(slot_of(i) + row));
#pragma unroll
      for (int d = 16; d; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      for (int i = lane; i < count_ctas; i += 32) {
        const float part_sum = __ldcg(slot_of(i) + kRows + row);
        const float weight = part_sum == 0.f ? 0.f : fast_exp2(__ldcg(slot_of(i) + row) - most);
        weights[i * kRows + row] = weight;
        all += weight * part_sum;
      }
#pragma unroll
      for (int d = 16; d; d /= 2) all += __shfl_xor_sync(0xffffffffu, all, d);
      if (lane == 0) inverse_sums[row] = all == 0.f ? 0.f : 1.f / all;
    }
    __syncthreads();
    for (int e = thread; e < rows * (kDim / 4); e += kThreads) {
      const int row = e / (kDim / 4), column = e % (kDim / 4) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < count_ctas; ++i) {
        const float weight = weights[i * kRows + row];
        const float4 y = __ldcg(reinterpret_cast<const float4*>(slot_of(i) + 2 * kRows + row * kDim + column));
        x.x += weight * y.x; x.y += weight * y.y; x.z += weight * y.z; x.w += weight * y.w;
      }
      const float inverse = inverse_sums[row];
      write_out(s, unit, row, column, make_float4(x.x * inverse, x.y * inverse, x.z * inverse, x.w * inverse));
    }
    __syncthreads();
  }
}

}  // namespace ci8
