// Attention of many query rows per sequence (prompts, chunks of prompts) over the 4-bit key/value cache, on tcgen05.
//
// A CTA takes up to 256 query rows of one key head (a row is a token and one of the query heads that share the key
// head, so their keys are unpacked once), as tiles of 128: two for dim 64 and 128, one for dim 256 (512 TMEM columns
// hold the scores and outputs of no more). It walks the keys in tiles of 128 (64 for dim 256):
//   unpack warps   codes from global memory (a half-step ahead, in registers) -> BF16 code - zero, exact small integers,
//                  into the 128-byte-swizzled operand tiles; scales beside them as FP32
//   MMA warp       S = Q K^T (Q from TMEM where it has room, from shared memory for dim 128), O += P V (P from TMEM)
//   softmax warps  32 rows each: S * key scale (times the softmax scale), running maximum and sum, weights * value scale
//                  rounded to BF16 into the columns of S. The output is scaled only when a row's maximum has grown by more than 2^8.
// The components of a word come out of the unpacking as 0 4 1 5 2 6 3 7; the queries are stored in that order and the
// output is put back.
//
// What bounds it is not the tensor pipe (37 to 40 % busy) but what feeds it. Dim 256, where a tile of keys serves 128 rows
// only: the unpacking (11 instructions and one 16-byte store for eight components), ahead of the shared memory's bandwidth.
// Dim 128: the chain scores -> softmax -> product -> next scores of each query tile, of which two run at a time, with 37 %
// of the cycles taken by the exponentials. Measured (32 query heads and 8 key heads of 128, 8192 new tokens): 748 us,
// 735 TFLOP/s; 24 and 4 heads of 256, 4096 tokens behind 4096: 762 us, 812 TFLOP/s, where queries in shared memory and lanes
// that load from eight rows at a time took 1020; 32 and 8 heads of 64, 8192 tokens: 636 us. Tried and slower: tiles of 64 keys
// with two score buffers for dim 128 (792), the tiles of keys dealt to two softmax warpgroups in turn (831; dim 256 880
// against 876 then), four unpacking warpgroups for dim 256 (917 against 876), more registers for the softmax (782 to 821).
#pragma once
#include "kv4_attention.cuh"

namespace ci8 {

template <int kDim>
struct Kv4PromptConfig {
  static constexpr int kQTiles = kDim == 256 ? 1 : 2;
  static constexpr int kRows = 128 * kQTiles;            // query rows of a CTA
  static constexpr int kKeys = kDim == 256 ? 64 : 128;   // keys of a tile
  static constexpr int kUnpackGroups = kDim == 256 ? 2 : 1;
  static constexpr int kThreads = 512;                   // softmax, unpack and MMA warpgroups
  static constexpr int kQBytes = 128 * kDim * 2;
  static constexpr int kTileBytes = kKeys * kDim * 2;
  // TMEM columns: two score buffers, the outputs from 256 on, and where they leave room the queries, which the score
  // products then need not read from shared memory for every tile of keys.
  static constexpr bool kQInTmem = kDim != 128;
  static constexpr int kScoreColumns = kDim == 256 ? 64 : 128;
  static constexpr int kQColumn = kDim == 256 ? 128 : 384;
  static constexpr int kStages = kDim == 256 ? 3 : 2;
  static constexpr int kSmemBytes = (kQInTmem ? 0 : kQTiles * kQBytes) + 2 * kStages * kTileBytes + 1024;
  // registers per thread after the hand-over; together 512 * 128
  static constexpr int kSoftmaxRegs = 192;
  static constexpr int kUnpackRegs = kDim == 256 ? 120 : 88;
  static constexpr int kMmaRegs = 40;
  static_assert(kQTiles * kSoftmaxRegs + kUnpackGroups * kUnpackRegs + kMmaRegs <= 512 && kSoftmaxRegs > 128 && kUnpackRegs < 128 && kMmaRegs < 128,
                "what is taken has been given back, and only a smaller number is a giving back");
};

struct Kv4PromptParams {
  Kv4AttendParams a;
  float* partial;             // [tile][key head][split][maximum, sum, output of every row] where there are several splits
  int splits;
  int most_rows;              // sequences with no more query rows than this belong to another kernel
};

// Scales are read by the softmax warps, some tiles behind the unpacking: the keys of tile j + kStages are unpacked when the
// scores of tile j are complete, and those were issued behind a product with the weights of tile j - 2 (or j - 1), whose
// scales were read then. So tile j may take the slot of tile j - 8 as long as kStages + 2 <= 8; the marks of tile j + 8 are
// cleared while those of tile j are set.
constexpr int kKv4ScaleSlots = 8;
constexpr int kKv4MarkSlots = 2 * kKv4ScaleSlots;

// Outputs are sums of weights (up to 2^8) times values (up to 2^127) over up to 2^30 keys until they are divided by the weights'
// sum. They are kept in units of 2^40, as the values' scales are: 2^125 at most, and the least scale, 2^-66, leaves weights down
// to 2^-20 normal.
constexpr float kKv4ValueUnit = 0x1p40f;

__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n, bool b_transposed) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_transposed ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// Operand tiles are stored as segments of 64 components: rows of 128 bytes, swizzled (the descriptor's upper word says
// so). The same tile serves as keys (K-major: components along K) and as values (components along N: `segment` is the
// distance between segments, in the lower word beside the address). A step of n bytes adds n / 16 to the lower word. The
// issuing warp shares its scheduler with three busy ones, so an MMA must cost it few instructions: one addition a
// descriptor.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr, uint32_t segment) { return ((smem_addr & 0x3FFFFu) >> 4) | ((segment >> 4) << 16); }
__device__ __forceinline__ void mma_bf16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
// 16 rows x 64 columns: lane 4 g + c holds columns 8 i + 2 c and 8 i + 2 c + 1 of row g in v[4 i], v[4 i + 1] and of row
// g + 8 in v[4 i + 2], v[4 i + 3].
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_16x64(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// 32 rows, one to a lane, x 32 columns.
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// 16 rows x 32 columns: column 4 i + c of row g in v[2 i], of row g + 8 in v[2 i + 1].
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The sequence and the place in it of row tile `index` (tiles of `rows` query rows, counted over the sequences that have
// more than most_rows); all lanes of a warp together. Returns the number of tiles there are.
struct Kv4PromptTile {
  int b, tile;
};
__device__ __forceinline__ int kv4_prompt_tile(const Kv4AttendParams& p, int rows, int most_rows, int index, Kv4PromptTile& found) {
  const int lane = threadIdx.x % 32;
  found = {-1, 0};
  int before = 0;
  for (int base = 0; base < p.batch; base += 32) {
    const int b = base + lane;
    int tiles = 0;
    if (b < p.batch) {
      const int q_rows = kv4_sequence(p, b).rows * static_cast<int>(p.group.d);
      if (q_rows > most_rows) tiles = (q_rows + rows - 1) / rows;
    }
    int scan = tiles;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += other;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, index >= before + scan - tiles && index < before + scan);
    if (hit) {
      const int from = __ffs(hit) - 1;
      found = {base + from, index - (before + __shfl_sync(0xffffffffu, scan - tiles, from))};
    }
    before += __shfl_sync(0xffffffffu, scan, 31);
  }
  return before;
}

// A bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, int parity, int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abort));
}

// kSplit: a row tile's keys are split over gridDim.z CTAs, whose parts the kernel below joins. (In one kernel for both, the
// loops' values got worse registers: 8192 tokens of 32 and 8 heads of 128 took 775 us, 747 in the one without splits.)
template <int kDim, bool kSplit>
__global__ void __launch_bounds__(512, 1) kv4_prompt_kernel(const Kv4PromptParams params) {
  using Cfg = Kv4PromptConfig<kDim>;
  constexpr int kQTiles = Cfg::kQTiles, kKeys = Cfg::kKeys, kStages = Cfg::kStages;
  constexpr int kSegments = kDim / 64;                   // of 64 components, 128 bytes a row
  constexpr int kSoftmaxGroups = kQTiles;
  constexpr uint32_t kOutputColumn = 256;
  static_assert(kStages + 2 <= kKv4ScaleSlots, "a slot's scales have been read when it is filled again");
  extern __shared__ uint8_t dynamic_smem[];
  __shared__ __align__(8) uint64_t bar_q, bar_s[2], bar_p[2][2], bar_done[2], bar_k[kStages], bar_k_free[kStages], bar_v[kStages], bar_v_free[kStages];
  __shared__ __align__(8) uint64_t bar_scale_k[kKv4ScaleSlots], bar_scale_v[kKv4ScaleSlots];
  __shared__ __align__(16) float scale_k[kKv4ScaleSlots][kKeys], scale_v[kKv4ScaleSlots][kKeys];
  __shared__ uint32_t hidden[kKv4MarkSlots][kKeys / 32];   // keys of the tile on a page that could not be followed
  __shared__ int any_hidden[kKv4MarkSlots];
  __shared__ float row_max[2][128], row_sum[2][128];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag, tile_info[2];
  const Kv4AttendParams& p = params.a;
  const int thread = threadIdx.x, warp = thread / 32, lane = thread % 32, warpgroup = warp / 4;
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dynamic_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* const q_smem = smem;
  uint8_t* const k_smem = smem + (Cfg::kQInTmem ? 0 : kQTiles * Cfg::kQBytes);
  uint8_t* const v_smem = k_smem + kStages * Cfg::kTileBytes;

  if (warp == 0) {
    if (lane == 0) {
      mbar_init(smem_u32(&bar_q), 128 * kQTiles);
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&bar_s[i]), 1);
        mbar_init(smem_u32(&bar_p[i][0]), 128);
        mbar_init(smem_u32(&bar_p[i][1]), 128);
        mbar_init(smem_u32(&bar_done[i]), 1);
      }
      for (int i = 0; i < kStages; ++i) {
        mbar_init(smem_u32(&bar_k[i]), 128);
        mbar_init(smem_u32(&bar_k_free[i]), 1);
        mbar_init(smem_u32(&bar_v[i]), 128);
        mbar_init(smem_u32(&bar_v_free[i]), 1);
      }
      for (int i = 0; i < kKv4ScaleSlots; ++i) {
        mbar_init(smem_u32(&bar_scale_k[i]), 128);
        mbar_init(smem_u32(&bar_scale_v[i]), 128);
      }
      abort_flag = 0;
    }
    if (lane < kKv4MarkSlots) {
      any_hidden[lane] = 0;
      for (int c = 0; c < kKeys / 32; ++c) hidden[lane][c] = 0;
    }
    __syncwarp();
    fence_barrier_init();
    tmem_alloc<1>(smem_u32(&tmem_base), 512);
    tmem_relinquish<1>();
  }
  pdl_wait();
  pdl_launch_dependents();
  if (warp == 1) {
    // the last row tiles see the most keys: they go first
    Kv4PromptTile found;
    const int all = kv4_prompt_tile(p, Cfg::kRows, params.most_rows, -1, found);
    const int index = all - 1 - static_cast<int>(blockIdx.x);
    if (index >= 0) kv4_prompt_tile(p, Cfg::kRows, params.most_rows, index, found);
    if (lane == 0) {
      tile_info[0] = index >= 0 ? found.b : -1;
      tile_info[1] = found.tile;
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_base;
  const int b = tile_info[0], first_row = tile_info[1] * Cfg::kRows, head = blockIdx.y, split = kSplit ? blockIdx.z : 0;
  const int group = p.group.d;

  if (b >= 0) {
    const Kv4Sequence seq = kv4_sequence(p, b);
    const int all_rows = seq.rows * group;
    const int last_row = min(all_rows, first_row + Cfg::kRows) - 1;
    const int keys = max(0, seq.keys - seq.rows + p.group.quotient(last_row) + 1);   // that the CTA's last row sees
    const int all_tiles = (keys + kKeys - 1) / kKeys;
    const int begin = kSplit ? static_cast<int>(static_cast<long long>(all_tiles) * split / params.splits) : 0;
    const int end = kSplit ? static_cast<int>(static_cast<long long>(all_tiles) * (split + 1) / params.splits) : all_tiles;
    const int tiles = end - begin;

    if (warpgroup < kSoftmaxGroups) {
      // ================================================================ softmax
      setmaxnreg_inc<Cfg::kSoftmaxRegs>();
      const int t = warpgroup, row_in_tile = thread % 128, row = first_row + 128 * t + row_in_tile;
      if constexpr (Cfg::kQInTmem) {
        // the thread's query row, in the unpacked codes' order
        const int token = p.group.quotient(row);
        const uint16_t* src = p.q + (seq.start + token) * p.q_stride + static_cast<int64_t>(head * group + row - token * group) * kDim;
#pragma unroll 1
        for (int base = 0; base < kDim; base += 64) {
          uint4 w[8];
#pragma unroll
          for (int n = 0; n < 8; ++n) w[n] = row < all_rows ? *reinterpret_cast<const uint4*>(src + base + 8 * n) : make_uint4(0, 0, 0, 0);
          uint32_t x[32];
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            x[4 * n] = __byte_perm(w[n].x, w[n].z, 0x5410);
            x[4 * n + 1] = __byte_perm(w[n].x, w[n].z, 0x7632);
            x[4 * n + 2] = __byte_perm(w[n].y, w[n].w, 0x5410);
            x[4 * n + 3] = __byte_perm(w[n].y, w[n].w, 0x7632);
          }
          tmem_st_32x32(tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + Cfg::kQColumn + (t * kDim + base) / 2, x);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        mbar_arrive(smem_u32(&bar_q));
      } else {
        // the tile's queries, in the unpacked codes' order
        constexpr int kPieces = kDim / 8;
        uint8_t* const tile = q_smem + t * Cfg::kQBytes;
#pragma unroll 1
        for (int base = row_in_tile; base < 128 * kPieces; base += 8 * 128) {
          uint4 w[8];                                    // eight loads in flight
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const int i = base + 128 * n, q_row = first_row + 128 * t + i / kPieces;
            w[n] = make_uint4(0, 0, 0, 0);
            if (q_row < all_rows) {
              const int token = p.group.quotient(q_row);
              w[n] = *reinterpret_cast<const uint4*>(p.q + (seq.start + token) * p.q_stride +
                                                     static_cast<int64_t>(head * group + q_row - token * group) * kDim + 8 * (i % kPieces));
            }
          }
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const int i = base + 128 * n, r = i / kPieces, piece = i % kPieces;
            *reinterpret_cast<uint4*>(tile + (piece / 8) * (128 * 128) + r * 128 + ((piece % 8) ^ (r & 7)) * 16) =
                make_uint4(__byte_perm(w[n].x, w[n].z, 0x5410), __byte_perm(w[n].x, w[n].z, 0x7632), __byte_perm(w[n].y, w[n].w, 0x5410),
                           __byte_perm(w[n].y, w[n].w, 0x7632));
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&bar_q));
      }
      constexpr int kRuns = kKeys / 64;
      // A warp's 32 rows as TMEM hands them out: lane 4 g + c works on rows g, g + 8, g + 16, g + 24 and on the keys 8 i + 2 c
      // and 8 i + 2 c + 1 of each. A lane then needs the scales of 16 keys of 64; with a whole row to a lane the scales'
      // broadcasts took as much of the shared memory's bandwidth as the MMAs' operands.
      const int g = lane / 4, c = lane % 4;
      int limit[4], least = 0x7fffffff;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int q_row = first_row + 128 * t + 32 * (warp % 4) + 8 * r + g;
        limit[r] = q_row < all_rows ? max(0, seq.keys - seq.rows + p.group.quotient(q_row) + 1) : 0;
        least = min(least, limit[r]);
      }
      least = __reduce_min_sync(0xffffffffu, least);
      const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16, half = 16u << 16;   // rows 16 .. 31 of the warp
      const uint32_t output = tmem + lanes + kOutputColumn + t * kDim;
      float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      float2 sum2[4] = {};
      bool fine = true;
      for (int j = 0; j < tiles && fine; ++j) {
        const int buffer = kQTiles == 2 ? t : j & 1;
        const uint32_t scores = tmem + lanes + Cfg::kScoreColumns * buffer;
        const int slot = j % kKv4ScaleSlots, slot_parity = j / kKv4ScaleSlots & 1;
        fine = warp_wait(&bar_s[buffer], kQTiles == 2 ? j & 1 : j >> 1 & 1, &abort_flag) && warp_wait(&bar_scale_k[slot], slot_parity, &abort_flag);
        if (!fine) break;
        tcgen05_fence_after();
        uint32_t s[kRuns][2][32];                        // [64 keys][rows g and g + 8, rows g + 16 and g + 24]
        const int first_key = (begin + j) * kKeys;
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        tmem_ld_16x64(scores, s[0][0]);
        tmem_ld_16x64(scores + half, s[0][1]);
#pragma unroll
        for (int h = 0; h < kRuns; ++h) {
          tmem_ld_wait_for(s[h][0]);
          tmem_ld_wait_for(s[h][1]);
          if (h + 1 < kRuns) {                           // the next keys' scores are on their way while these are in work
            tmem_ld_16x64(scores + 64 * (h + 1), s[h + 1][0]);
            tmem_ld_16x64(scores + 64 * (h + 1) + half, s[h + 1][1]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 k = *reinterpret_cast<const float2*>(&scale_k[slot][64 * h + 8 * i + 2 * c]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              uint32_t* at = &s[h][r / 2][4 * i + 2 * (r & 1)];
              const float2 x = __fmul2_rn(make_float2(__uint_as_float(at[0]), __uint_as_float(at[1])), k);
              at[0] = __float_as_uint(x.x);
              at[1] = __float_as_uint(x.y);
              top[r] = max3(top[r], x.x, x.y);
            }
          }
        }
        if (first_key + kKeys > least || any_hidden[j % kKv4MarkSlots]) {
#pragma unroll
          for (int r = 0; r < 4; ++r) top[r] = -INFINITY;
#pragma unroll
          for (int i = 0; i < 8 * kRuns; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = 8 * i + 2 * c + e;
              const bool marked = hidden[j % kKv4MarkSlots][key / 32] >> (key % 32) & 1;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                uint32_t& x = s[i / 8][r / 2][4 * (i % 8) + 2 * (r & 1) + e];
                if (marked || first_key + key >= limit[r]) x = 0xff800000u;
                top[r] = fmaxf(top[r], __uint_as_float(x));
              }
            }
        }
        bool grows = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          grows |= top[r] > m[r] + 8.f;
        }
        if (__any_sync(0xffffffffu, grows)) {
          float keep[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float next = fmaxf(m[r], top[r]);
            keep[r] = next == -INFINITY ? 1.f : fast_exp2(m[r] - next);
            m[r] = next;
            sum2[r].x *= keep[r];
            sum2[r].y *= keep[r];
          }
          if (j > 0) {
            // Two query tiles: these scores were issued behind the product that last wrote the output, which is
            // complete. One: that product may still be running.
            if (kQTiles == 1) {
              fine = warp_wait(&bar_done[1], (j - 1) & 1, &abort_flag);
              if (!fine) break;
              tcgen05_fence_after();
            }
#pragma unroll 1
            for (int part = 0; part < 2 * (kDim / 64); ++part) {
              const uint32_t at = output + 64 * (part / 2) + (part & 1 ? half : 0);
              const float low = part & 1 ? keep[2] : keep[0], high = part & 1 ? keep[3] : keep[1];
              uint32_t o[32];
              tmem_ld_16x64(at, o);
              tmem_ld_wait_for(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * (i & 2 ? high : low));
              tmem_st_16x64(at, o);
            }
          }
        }
        fine = warp_wait(&bar_scale_v[slot], slot_parity, &abort_flag);
        if (!fine) break;
        float2 base2[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) base2[r].x = base2[r].y = m[r] == -INFINITY ? 0.f : -m[r];
#pragma unroll
        for (int h = 0; h < kRuns; ++h) {
          uint32_t packed[2][16];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 v = *reinterpret_cast<const float2*>(&scale_v[slot][64 * h + 8 * i + 2 * c]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t* at = &s[h][r / 2][4 * i + 2 * (r & 1)];
              float2 x = __fadd2_rn(make_float2(__uint_as_float(at[0]), __uint_as_float(at[1])), base2[r]);
              x = make_float2(fast_exp2(x.x), fast_exp2(x.y));
              sum2[r] = __fadd2_rn(sum2[r], x);
              x = __fmul2_rn(x, v);
              packed[r / 2][2 * i + (r & 1)] = pack2(x.x, x.y);
            }
          }
          tmem_st_16x32(scores + 32 * h, packed[0]);
          tmem_st_16x32(scores + 32 * h + half, packed[1]);
          tmem_st_wait();
          tcgen05_fence_before();
          mbar_arrive(smem_u32(&bar_p[buffer][h]));      // the product may begin on the first half of the keys
        }
      }
      // the rows' maxima and sums, for the lanes that hold them in the output's layout (one row to a lane)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float all = sum2[r].x + sum2[r].y;
        all += __shfl_xor_sync(0xffffffffu, all, 1);
        all += __shfl_xor_sync(0xffffffffu, all, 2);
        if (c == 0) {
          row_max[t][32 * (warp % 4) + 8 * r + g] = m[r];
          row_sum[t][32 * (warp % 4) + 8 * r + g] = all;
        }
      }
      __syncwarp();
      const int token = p.group.quotient(row);
      const float sum = row_sum[t][row_in_tile];
      // ---- output
      if (fine && tiles > 0) fine = warp_wait(&bar_done[t], 0, &abort_flag);
      tcgen05_fence_after();
      if constexpr (kSplit) {
        float* slot = params.partial + (((static_cast<int64_t>(blockIdx.x) * p.kv_heads + head) * params.splits + split) * Cfg::kRows + 128 * t) * (kDim + 2);
        slot[row_in_tile] = row_max[t][row_in_tile];       // [128 maxima][128 sums][128 outputs]
        slot[128 + row_in_tile] = sum;
        float* dst = slot + 256 + row_in_tile * kDim;
        if (tiles > 0 && fine) {
#pragma unroll 1
          for (int c = 0; c < kDim; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32(output + c, o);
            tmem_ld_wait_for(o);
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(o[i], o[i + 2], o[i + 4], o[i + 6]);
              *reinterpret_cast<uint4*>(dst + c + i + 4) = make_uint4(o[i + 1], o[i + 3], o[i + 5], o[i + 7]);
            }
          }
        }
      } else {
        const float inverse = sum == 0.f ? 0.f : kKv4ValueUnit / sum;
        uint16_t* dst = p.out + (static_cast<int64_t>(seq.start + token) * p.q_heads + head * group + row - token * group) * kDim;
#pragma unroll 1
        for (int c = 0; c < kDim; c += 32) {
          uint32_t o[32];
          if (tiles > 0 && fine) {
            tmem_ld_32x32(output + c, o);
            tmem_ld_wait_for(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (row < all_rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(o[i + e]) * inverse;
              *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(pack2(x[0], x[2]), pack2(x[4], x[6]), pack2(x[1], x[3]), pack2(x[5], x[7]));
            }
          }
        }
      }
    } else if (warpgroup < 3) {
      // ================================================================ unpacking
      setmaxnreg_dec<Cfg::kUnpackRegs>();
      // One group unpacks keys and values in turn; two groups take one each.
      const int side_first = Cfg::kUnpackGroups == 2 ? warpgroup - kSoftmaxGroups : 0;
      constexpr int kSteps = Cfg::kUnpackGroups == 2 ? 1 : 2;          // half-steps (sides) per tile of keys
      // Eight neighbouring lanes load pieces of 16 code bytes and store 16 bytes of components together. Both want different
      // banks: four rows of two pieces for dim 64 and 128, and for dim 256 one row, whose words the lanes then store in an
      // order of their own (word ^ turn), at the cost of the selections.
      constexpr int kPieces = kDim / 32, kPassRows = 128 / kPieces, kPasses = kKeys / kPassRows;
      const int lane_row = kPassRows / 4 * (warp % 4) + (kDim == 128 ? lane / 2 % 4 + lane / 16 * 4 : lane / kPieces);
      const int lane_piece = kDim == 128 ? lane % 2 + lane / 8 % 2 * 2 : lane % kPieces;
      const int turn = kDim == 256 ? lane_piece / 2 : 0;
      const int page = 1 << p.page_shift;
      const unsigned block_bytes = page * (kDim / 2 + 4), page_bytes = block_bytes * kKv4Side * p.kv_heads;   // at most 70 MB
      const uint8_t* const head_src = p.cache + static_cast<uint64_t>(head) * block_bytes;
      const int32_t* const table = p.block_table + static_cast<int64_t>(b) * p.width;
      // A run of 16 keys lies on one page, and a warp's rows of a pass in one run. Page numbers are loaded a tile ahead of the
      // codes: lane l holds the one of the tile's run l.
      constexpr int kRunsOfTile = kKeys / 16;
      auto load_ids = [&](int j) { return table[min((begin + j) * kKeys + 16 * lane, keys - 1) >> p.page_shift]; };
      const int lane_code = lane_row % 16 * (kDim / 2) + 16 * lane_piece, lane_pair = page * (kDim / 2) + 4 * (lane_row % 16);
      int ids = -1, ids_ahead = tiles > 0 ? load_ids(0) : -1;
      uint4 codes[kPasses];
      uint32_t pairs[kPasses];                           // (nothing may touch what is loaded before the next half-step)
      uint32_t live = 0, marks = 0;                      // runs whose keys are there, that lie on a page that cannot be followed
      auto load = [&](int step) {
        const int j = step / kSteps, side = kSteps == 2 ? step & 1 : side_first, first = (begin + j) * kKeys;
        const uint8_t* const side_src = head_src + side * p.kv_heads * block_bytes;
        if (kSteps == 1 || side == 0) {
          ids = ids_ahead;
          ids_ahead = load_ids(j + 1);
        }
        const bool wanted = lane < kRunsOfTile && first + 16 * lane < keys, good = wanted && static_cast<unsigned>(ids) < static_cast<unsigned>(p.pages);
        live = __ballot_sync(0xffffffffu, good);
        marks = __ballot_sync(0xffffffffu, wanted && !good);
        const unsigned id = good ? ids : 0u;             // a run that is not there reads the cache's first page and is made zero when it is used
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          const int run = (kPassRows * i + lane_row) / 16, at = (first + 16 * run) & (page - 1);
          const uint8_t* src = side_src + static_cast<uint64_t>(__shfl_sync(0xffffffffu, id, run)) * page_bytes;
          if (p.pages > 0) {
            pairs[i] = __ldcg(reinterpret_cast<const unsigned*>(src + (4 * at + lane_pair)));
            codes[i] = __ldcg(reinterpret_cast<const uint4*>(src + (at * (kDim / 2) + lane_code)));
          }
        }
      };
      const int steps = tiles * kSteps;
      bool fine = true;
      if (steps > 0) load(0);
      for (int step = 0; step < steps; ++step) {
        const int j = step / kSteps, side = kSteps == 2 ? step & 1 : side_first;
        const int stage = j % kStages, slot = j % kKv4ScaleSlots;
        uint64_t* const full = side ? bar_v : bar_k;
        uint64_t* const empty = side ? bar_v_free : bar_k_free;
        uint4 now[kPasses];
        uint32_t now_pairs[kPasses];
        const uint32_t now_marks = marks, now_live = live;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          now_pairs[i] = pairs[i];
          now[i] = codes[i];
        }
        if (step + 1 < steps) load(step + 1);
        if (j >= kStages) fine = warp_wait(&empty[stage], (j / kStages - 1) & 1, &abort_flag);
        if (!fine) break;
        if (now_live != (1u << kRunsOfTile) - 1 || (begin + j + 1) * kKeys > keys) {
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const int row = kPassRows * i + lane_row;
            if ((now_live >> (row / 16) & 1) && (begin + j) * kKeys + row < keys) continue;
            now_pairs[i] = 0;
            now[i] = make_uint4(0, 0, 0, 0);
          }
        }
        uint8_t* const tile = (side ? v_smem : k_smem) + stage * Cfg::kTileBytes;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          const int row = kPassRows * i + lane_row;
          const float zero = 128.f + bf16_hi(now_pairs[i]);
          const uint32_t zeros = pack2(zero, zero);
          // the softmax scale comes with the keys': a score and the maximum are then one rounded number, and their difference
          // is exact where the score is the maximum, however large
          if (lane_piece == 0) (side ? scale_v : scale_k)[slot][row] = bf16_lo(now_pairs[i]) * (side ? 1.f / kKv4ValueUnit : p.scale_log2);
          uint32_t words[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
#pragma unroll
          for (int bit = 1; kDim == 256 && bit < 4; bit *= 2)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if (w & bit) continue;
              const uint32_t first = words[w], second = words[w ^ bit];
              words[w] = turn & bit ? second : first;
              words[w ^ bit] = turn & bit ? first : second;
            }
          uint8_t* const segment = tile + (lane_piece / 2) * (kKeys * 128) + row * 128;
          const int chunk = (lane_piece % 2 * 4) ^ turn ^ (row & 7);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[e] = ((words[w] >> (4 * e)) & 0x000f000fu) | 0x43004300u;
              asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(v[e]) : "r"(zeros));
            }
            *reinterpret_cast<uint4*>(segment + (chunk ^ w) * 16) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        if (side == 0) {
          if (warp % 4 == 0) {
            const int clear = (j + kKv4ScaleSlots) % kKv4MarkSlots;
            if (lane < kKeys / 32) hidden[clear][lane] = 0;
            if (lane == 0) any_hidden[clear] = 0;
          }
          if (now_marks) {
            any_hidden[j % kKv4MarkSlots] = 1;
            atomicOr(&g_ci8_status, kStatusBadIndex);
            if (now_marks >> lane & 1) atomicOr(&hidden[j % kKv4MarkSlots][lane / 2], 0xffffu << (lane % 2 * 16));
          }
          mbar_arrive(smem_u32(&bar_scale_k[slot]));
        } else {
          mbar_arrive(smem_u32(&bar_scale_v[slot]));
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&full[stage]));
      }
    } else {
      setmaxnreg_dec<Cfg::kMmaRegs>();
      if (warp == 12 && tiles > 0) {
        // ================================================================ MMA issue
        constexpr uint32_t kIdescS = idesc_bf16(128, kKeys, false), kIdescO = idesc_bf16(128, kDim, true);
        const uint32_t q_desc = desc_low(smem_u32(q_smem), 16), k_desc = desc_low(smem_u32(k_smem), 16);
        const uint32_t v_desc = desc_low(smem_u32(v_smem), kKeys * 128);
        constexpr uint32_t kTileStep = Cfg::kTileBytes / 16, kQStep = Cfg::kQBytes / 16;
        auto scores = [&](int t, int buffer, int stage) {
          const uint32_t d = tmem + Cfg::kScoreColumns * buffer, b = k_desc + stage * kTileStep;
          const uint32_t a = Cfg::kQInTmem ? tmem + Cfg::kQColumn + t * (kDim / 2) : q_desc + t * kQStep;
          if (elect_one()) {
#pragma unroll
            for (int s = 0; s < kSegments; ++s)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if constexpr (Cfg::kQInTmem)
                  mma_bf16_ts(d, a + 32 * s + 8 * k, b + s * (kKeys * 128 / 16) + 2 * k, kIdescS, s + k > 0);
                else
                  mma_bf16_ss(d, a + s * (128 * 128 / 16) + 2 * k, b + s * (kKeys * 128 / 16) + 2 * k, kIdescS, s + k > 0);
              }
            mma_commit(smem_u32(&bar_s[buffer]));
          }
          __syncwarp();
        };
        auto outputs = [&](int t, int buffer, int stage, int parity, bool accumulate) {   // waits for the weights, 64 keys at a time
          for (int h = 0; h < kKeys / 64; ++h) {
            if (!warp_wait(&bar_p[buffer][h], parity, &abort_flag)) return false;
            tcgen05_fence_after();
            const uint32_t d = tmem + kOutputColumn + t * kDim, a = tmem + Cfg::kScoreColumns * buffer + 32 * h, b = v_desc + stage * kTileStep + h * (8192 / 16);
            if (elect_one()) {
              mma_bf16_ts(d, a, b, kIdescO, accumulate || h > 0);
#pragma unroll
              for (int k = 1; k < 4; ++k) mma_bf16_ts(d, a + 8 * k, b + k * (2048 / 16), kIdescO, 1);
            }
            __syncwarp();
          }
          return true;
        };
        auto commit = [&](uint64_t* bar) {
          if (elect_one()) mma_commit(smem_u32(bar));
          __syncwarp();
        };
        bool fine = warp_wait(&bar_q, 0, &abort_flag);
        tcgen05_fence_after();
        if constexpr (kQTiles == 2) {
          for (int j = 0; j <= tiles && fine; ++j) {
            for (int t = 0; t < 2 && fine; ++t) {
              if (j > 0) {
                const int stage = (j - 1) % kStages;
                if (t == 0) fine = warp_wait(&bar_v[stage], (j - 1) / kStages & 1, &abort_flag);
                fine = fine && outputs(t, t, stage, (j - 1) & 1, j > 1);
                if (!fine) break;
                if (t == 1) commit(&bar_v_free[stage]);
                if (j == tiles) commit(&bar_done[t]);
              }
              if (j < tiles) {
                const int stage = j % kStages;
                if (t == 0) {
                  fine = warp_wait(&bar_k[stage], j / kStages & 1, &abort_flag);
                  if (!fine) break;
                  tcgen05_fence_after();
                }
                scores(t, t, stage);
                if (t == 1) commit(&bar_k_free[stage]);
              }
            }
          }
        } else {
          for (int j = 0; j <= tiles && fine; ++j) {
            if (j < tiles) {
              const int stage = j % kStages;
              fine = warp_wait(&bar_k[stage], j / kStages & 1, &abort_flag);
              if (!fine) break;
              tcgen05_fence_after();
              scores(0, j & 1, stage);
              commit(&bar_k_free[stage]);
            }
            if (j > 0) {
              const int stage = (j - 1) % kStages, buffer = (j - 1) & 1;
              fine = warp_wait(&bar_v[stage], (j - 1) / kStages & 1, &abort_flag) && outputs(0, buffer, stage, (j - 1) >> 1 & 1, j > 1);
              if (!fine) break;
              commit(&bar_v_free[stage]);
              commit(&bar_done[j == tiles ? 0 : 1]);
            }
          }
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc<1>(tmem, 512);
}

// Joins the splits of a row tile: grid (row tiles, key heads, shares), in the order of the splits. Bound by the latency of its
// loads: a thread takes one group of four components where the grid allows, and the loads of several splits are in
// flight together (3 splits of 128 rows of 256: 7 us, 17 with four groups a thread and one load at a time).
template <int kDim>
__global__ void __launch_bounds__(256) kv4_prompt_join_kernel(const Kv4PromptParams params) {
  using Cfg = Kv4PromptConfig<kDim>;
  __shared__ int tile_info[2];
  const Kv4AttendParams& p = params.a;
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < 32) {
    Kv4PromptTile found;
    const int all = kv4_prompt_tile(p, Cfg::kRows, params.most_rows, -1, found);
    const int index = all - 1 - static_cast<int>(blockIdx.x);
    if (index >= 0) kv4_prompt_tile(p, Cfg::kRows, params.most_rows, index, found);
    if (threadIdx.x == 0) {
      tile_info[0] = index >= 0 ? found.b : -1;
      tile_info[1] = found.tile;
    }
  }
  __syncthreads();
  const int b = tile_info[0], first_row = tile_info[1] * Cfg::kRows, head = blockIdx.y, group = p.group.d;
  if (b < 0) return;
  const Kv4Sequence seq = kv4_sequence(p, b);
  const int rows = min(Cfg::kRows, seq.rows * group - first_row);
  const float* base = params.partial + (static_cast<int64_t>(blockIdx.x) * p.kv_heads + head) * params.splits * Cfg::kRows * (kDim + 2);
  for (int e = threadIdx.x + 256 * blockIdx.z; e < rows * (kDim / 4); e += 256 * gridDim.z) {
    const int row = e / (kDim / 4), column = e % (kDim / 4) * 4;
    auto piece = [&](int s) { return base + (static_cast<int64_t>(s) * Cfg::kRows + row / 128 * 128) * (kDim + 2); };
    float most = -INFINITY, all = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < params.splits; ++s) most = fmaxf(most, __ldcg(piece(s) + row % 128));
#pragma unroll 4
    for (int s = 0; s < params.splits; ++s) {
      const float sum = __ldcg(piece(s) + 128 + row % 128), top = __ldcg(piece(s) + row % 128);
      float4 y = __ldcg(reinterpret_cast<const float4*>(piece(s) + 256 + row % 128 * kDim + column));
      // a part that saw no key has sum 0 and left its output unwritten (a NaN score makes its sum NaN, which is kept)
      const float weight = sum == 0.f ? 0.f : fast_exp2(top - most);
      if (sum == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
      all += weight * sum;
      x.x += weight * y.x; x.y += weight * y.y; x.z += weight * y.z; x.w += weight * y.w;
    }
    const float inverse = all == 0.f ? 0.f : kKv4ValueUnit / all;
    const int r = first_row + row, token = p.group.quotient(r);
    uint16_t* dst = p.out + (static_cast<int64_t>(seq.start + token) * p.q_heads + head * group + r - token * group) * kDim + column;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(x.x * inverse, x.y * inverse), pack2(x.z * inverse, x.w * inverse));
  }
}

}  // namespace ci8
