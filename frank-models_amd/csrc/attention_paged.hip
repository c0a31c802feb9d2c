// Attention of a sequence's new tokens over a paged cache of e4m3 codes with
// one scale for each (page, K/V head):
//   score_j = (q . K_j) SK[page(j)] * scale,  out = sum_j softmax(score)_j SV[page(j)] V_j
// over the positions j below the context's length and, causal, up to the
// query's own.  Table entries outside the pool are rows of zeros, as in
// kvcache_gather; a query that attends nothing gives zeros.
//
// Query rows of a K/V head are its (token, query head) pairs, token-major:
// row r is token r / G, query head kvh * G + r % G, for G query heads per
// K/V head, so that one read of K and V serves the group and the tokens.
#include <algorithm>
#include <atomic>

#include "common.h"
#include "launch.h"

namespace fmoe {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// What exponents are taken against: the maximum, or 0 where every score is
// minus infinity, so that such positions weigh 0 and not NaN.
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ f32x4_t mfma16(const u32x4_t a, const u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                0, 0, 0);
}

__device__ __forceinline__ void load_lds16(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 16, 0, kNonTemporal);
}
__device__ __forceinline__ void load_lds16_cached(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
}
__device__ __forceinline__ void load_lds4(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0);
}

// Eight codes of one column from eight rows of a tile in LDS: the lanes
// 2k and 2k + 1 of a group of 16 name row k's 8 low and 8 high columns, and
// lane c of the group gets column c, row k in byte k.  Several at once and
// waited for together, in assembly: before the compiler's own reads of this
// kind it waits for every load to LDS in flight, the next tiles' too, which
// cost a decode step of 61 x 1000 positions 27.4 us instead of 25.3.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

template <int N>
__device__ __forceinline__ void read_columns(const uint32_t (&at)[N], u32x2_t (&w)[N]) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "one column piece per 16 dimensions");
  if constexpr (N == 1) {
    asm volatile("ds_read_b64_tr_b8 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(w[0]) : "v"(at[0]) : "memory");
  } else if constexpr (N == 2) {
    asm volatile(
        "ds_read_b64_tr_b8 %0, %2\n\tds_read_b64_tr_b8 %1, %3\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1])
        : "v"(at[0]), "v"(at[1])
        : "memory");
  } else if constexpr (N == 4) {
    asm volatile(
        "ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\t"
        "ds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\t"
        "ds_read_b64_tr_b8 %2, %10\n\tds_read_b64_tr_b8 %3, %11\n\t"
        "ds_read_b64_tr_b8 %4, %12\n\tds_read_b64_tr_b8 %5, %13\n\t"
        "ds_read_b64_tr_b8 %6, %14\n\tds_read_b64_tr_b8 %7, %15\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7])
        : "memory");
  }
}

// The same for four steps of kStep bytes from each address.
template <int kStep, int N>
__device__ __forceinline__ void read_columns4(const uint32_t (&at)[N], u32x2_t (&w)[4][N]) {
  static_assert(N == 2 || N == 4, "32 columns each");
  if constexpr (N == 2) {
    asm volatile(
        "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\t"
        "ds_read_b64_tr_b8 %2, %8 offset:%10\n\tds_read_b64_tr_b8 %3, %9 offset:%10\n\t"
        "ds_read_b64_tr_b8 %4, %8 offset:%11\n\tds_read_b64_tr_b8 %5, %9 offset:%11\n\t"
        "ds_read_b64_tr_b8 %6, %8 offset:%12\n\tds_read_b64_tr_b8 %7, %9 offset:%12\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(w[0][0]), "=&v"(w[0][1]), "=&v"(w[1][0]), "=&v"(w[1][1]), "=&v"(w[2][0]), "=&v"(w[2][1]),
          "=&v"(w[3][0]), "=&v"(w[3][1])
        : "v"(at[0]), "v"(at[1]), "i"(kStep), "i"(2 * kStep), "i"(3 * kStep)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b8 %0, %16\n\tds_read_b64_tr_b8 %1, %17\n\t"
        "ds_read_b64_tr_b8 %2, %18\n\tds_read_b64_tr_b8 %3, %19\n\t"
        "ds_read_b64_tr_b8 %4, %16 offset:%20\n\tds_read_b64_tr_b8 %5, %17 offset:%20\n\t"
        "ds_read_b64_tr_b8 %6, %18 offset:%20\n\tds_read_b64_tr_b8 %7, %19 offset:%20\n\t"
        "ds_read_b64_tr_b8 %8, %16 offset:%21\n\tds_read_b64_tr_b8 %9, %17 offset:%21\n\t"
        "ds_read_b64_tr_b8 %10, %18 offset:%21\n\tds_read_b64_tr_b8 %11, %19 offset:%21\n\t"
        "ds_read_b64_tr_b8 %12, %16 offset:%22\n\tds_read_b64_tr_b8 %13, %17 offset:%22\n\t"
        "ds_read_b64_tr_b8 %14, %18 offset:%22\n\tds_read_b64_tr_b8 %15, %19 offset:%22\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(w[0][0]), "=&v"(w[0][1]), "=&v"(w[0][2]), "=&v"(w[0][3]), "=&v"(w[1][0]), "=&v"(w[1][1]),
          "=&v"(w[1][2]), "=&v"(w[1][3]), "=&v"(w[2][0]), "=&v"(w[2][1]), "=&v"(w[2][2]), "=&v"(w[2][3]),
          "=&v"(w[3][0]), "=&v"(w[3][1]), "=&v"(w[3][2]), "=&v"(w[3][3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "i"(kStep), "i"(2 * kStep), "i"(3 * kStep)
        : "memory");
  }
}

// 0x80 in each byte that is a NaN code (0x7F, 0xFF).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// x as a sum of kTerms bf16 values, eight at a time, each rounded to nearest:
// one term holds a bf16 value exactly, three an fp32 value to 2^-24 or better.
template <int kTerms>
__device__ __forceinline__ void split8(const float* x, u32x4_t* t) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
    for (int k = 0; k < kTerms; ++k) {
      const uint32_t w = pack_bf16x2(a, b);
      t[k][e] = w;
      if (k + 1 < kTerms) {
        a -= bf16_lo(w);
        b -= bf16_hi(w);
      }
    }
  }
}

// One sequence's tokens, context and limits.
struct Span {
  int len;      // new tokens that are not padding
  int64_t pos;  // position of token 0 (negative: the context is shorter than the tokens)
  int cut;      // positions that exist: min(context, max_ctx)
};

__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, int b) {
  Span s;
  s.len = a.lens ? min(max(a.lens[b], 0), a.seq_len) : a.seq_len;
  const int ctx = max(a.ctx_lens[b], 0);
  s.pos = static_cast<int64_t>(ctx) - s.len;
  s.cut = min(ctx, a.max_ctx);
  return s;
}

// Positions that token t attends: those below the result.
__device__ __forceinline__ int limit_of(const PagedAttnArgs& a, const Span& s, int t) {
  if (t >= s.len) return 0;
  return a.causal ? static_cast<int>(min(max(s.pos + t + 1, int64_t{0}), static_cast<int64_t>(s.cut))) : s.cut;
}

// The n lowest bits.
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n > 0 ? (1ull << n) - 1 : 0ull; }

// Four values from element i on (a multiple of 4) of the output.
__device__ __forceinline__ void store4(const PagedAttnArgs& a, int64_t i, f32x4_t v) {
  if (a.dtype == DT_F32)
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + i) = v;
  else
    *reinterpret_cast<u32x2_t*>(static_cast<bf16_t*>(a.out) + i) =
        u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// Four values from element i on of a tensor in dtype.
__device__ __forceinline__ f32x4_t load4(const void* p, int dtype, int64_t i) {
  if (dtype == DT_F32) return *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(p) + i);
  const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const bf16_t*>(p) + i);
  return f32x4_t{bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
}

// Over lanes l and l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// How a call is cut (plan_of): splits of split_len positions; few rows: the
// waves that share a row tile, a power of two.
struct Plan {
  bool big, aligned, join;  // aligned: four neighbouring positions share a page
  int n_split, split_len, waves_per_tile;
  int group, tile_groups;  // query heads per K/V head; blocks that a sequence's rows take in a split
  Div batch_div, split_div, kv_div, group_div, block_div, head_div, len_div;  // batch, n_split, n_head_kv, group, block_size, n_head, split_len
};

// ------------------------------------------------------------------ few rows
// A wave takes one row tile of 16 and, of its context split, every
// waves_per_tile-th chunk of 64 positions, through a ring of its own in LDS;
// the waves of a tile are merged at the end.  K and V codes pass through the
// ring once, by global_load_lds, in tiles that are refilled with the next
// chunk's as soon as they are read, so that 16 KiB a wave (head_dim 128) stay
// in flight through the arithmetic, and a wave's first K and V arrive
// together; the page table runs two chunks ahead, rows and scales one.
// Scores: v_mfma_f32_16x16x32_bf16 with A = 16 positions x 32 dimensions of
// K (codes are exact in bf16), B = the 16 query rows: a lane then holds, for
// row l % 16, positions 4 (l / 16) + i of each 16.  That is the B operand of
// the second product as it stands, with A = V transposed (ds_read_b64_tr_b8)
// taken in the same order of positions.  fp32 activations: q and the weights
// as three bf16 terms.
// A chunk that not every row attends in full takes the masked path: scores
// replaced by selects, and V codes that are NaN kept from the rows that do
// not attend them (0 * NaN is NaN) by a product of indicators of its own.
// Bound by memory: 16 x 4096 positions of 32/8 heads x 128, 134 MB, 26.4 us
// (5.1 TB/s; a copy reaches 5.2) and 4.1 for the join; 61 of 1000 and fewer, 95
// MB, 22.7 us; 64 x 8192, 1.07 GB, 171 us; 1 x 8192 8.2 and 3.6 us, the latency
// of a table entry, rows, K and V one after another.  fp32 activations are
// bound by the products of their terms: 3 x 701 tokens, causal, 56.5 us, 120
// TFLOP/s where a library's fp32 product reaches 154.
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kRows = 16;
constexpr int kChunk = 64;
constexpr int kSub = kChunk / 16;  // groups of 16 positions

// The running maximum is raised, and the sums rescaled, only when a row's has
// grown by more than 2^kLazy: weights are then at most 2^kLazy, which fp32
// sums and bf16 operands hold as well.
constexpr float kLazy = 8.f;
// The same of a lane's 32 weights together where the maximum is not looked
// for: wider, since to look costs what was saved (with 2^8, 4 x 1021 tokens 62.6 us
// instead of 55.1), and as far from fp32's limits.
constexpr float kMaxSum = 65536.f;

template <int D>
struct Stream {
  static constexpr int kRowsPerLoad = 1024 / D;                        // a load is 64 lanes x 16 bytes
  static constexpr int kTile = kRowsPerLoad > 32 ? kRowsPerLoad : 32;  // positions
  static constexpr int kLoads = kTile / kRowsPerLoad;
  static constexpr int kTiles = kChunk / kTile;  // of K, and of V
  static constexpr int kTileB = kTile * D;
  static constexpr int kRing = 2 * kTiles * kTileB;
  static constexpr int kWaveB = kRing + 6 * kChunk * 4;  // + table, rows, and K and V scales of two chunks
  static constexpr int kPieces = D / 16;                 // 16-byte pieces of a row
  static constexpr int kSteps = D >= 32 ? D / 32 : 1;    // products over the dimensions
  static constexpr int kLds = kWaves * kWaveB + 2 * kWaves * kRows * 4;
  static_assert(kTiles <= 2, "the waits count at most two tiles");
  static_assert(kRows * D * 4 <= kRing, "a wave's partial output fits its ring");
};

// Where piece c of row r of a tile lies among the row's 16-byte pieces: the
// rows that an operand read touches together spread over the banks.
template <int D>
__device__ __forceinline__ int k_place(int r) {  // rows r .. r + 15
  return D == 128 ? (r >> 1) & 7 : D == 64 ? (r >> 2) & 3 : D == 32 ? (r >> 3) & 1 : 0;
}
template <int D>
__device__ __forceinline__ int v_place(int r) {  // rows 0-7 and 16-23, or 8-15 and 24-31
  return D == 128 ? ((r >> 1) & 3) | ((r >> 4) & 1) << 2
         : D == 64 ? ((r >> 2) & 1) | ((r >> 4) & 1) << 1
         : D == 32 ? (r >> 4) & 1
                   : 0;
}

// Over lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float max_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_quarters(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

template <int D, int kTerms>
__global__ __launch_bounds__(kThreads, 2) void paged_stream_kernel(PagedAttnArgs a, Plan plan) {
  using R = Stream<D>;
  constexpr int kL = R::kLoads, kT = R::kTiles;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int q4 = lane >> 4, col = lane & 15;
  const int wpt = plan.waves_per_tile, part_wave = wave & (wpt - 1), tiles_log2 = __builtin_ctz(kWaves / wpt);
  const int x = plan.split_div(blockIdx.x), split = blockIdx.x - x * plan.n_split;
  const int g = plan.batch_div(x), b = x - g * a.batch;
  // Row tiles by (rows, K/V head), heads fastest: a block's waves read
  // neighbouring heads' parts of the same pool rows, 512 bytes together.  The
  // tiles of the last tokens, which attend most, go first.
  const int tile = ((plan.tile_groups - 1 - g) << tiles_log2) + (wave >> (2 - tiles_log2));
  const int row_tile = plan.kv_div(tile), kvh = tile - row_tile * a.n_head_kv;
  const int row0 = row_tile * kRows;
  const int j0 = split * plan.split_len;

  unsigned char* ring = lds + wave * R::kWaveB;
  int* table = reinterpret_cast<int*>(ring + R::kRing);
  int* rows = table + kChunk;
  float* ks = reinterpret_cast<float*>(rows + kChunk);  // [2][kChunk]
  float* vs = ks + 2 * kChunk;                          // [2][kChunk]
  float* stat = reinterpret_cast<float*>(lds + kWaves * R::kWaveB);  // [waves][16] maxima, then sums

  // Chunk c of this wave: its first position within the sequence.
  auto chunk_at = [&](int c) __attribute__((always_inline)) { return j0 + (c * wpt + part_wave) * kChunk; };
  const int* seq_table = a.tables + static_cast<int64_t>(b) * a.max_blocks;
  // The page table entries of a chunk's positions, into LDS.
  auto load_table = [&](int c) __attribute__((always_inline)) {
    load_lds4(seq_table + min(plan.block_div(chunk_at(c) + lane), a.max_blocks - 1), table);
  };
  load_table(0);  // needs no length, so it is asked for beside them

  // This lane's query row (column `col` of the products).
  const int G = plan.group;
  const Span span = span_of(a, b);
  const int token = plan.group_div(row0 + col), head = kvh * G + row0 + col - token * G;
  const int limit = limit_of(a, span, token);
  const int first_token = plan.group_div(row0);
  const int first_limit = limit_of(a, span, first_token);  // 0: the tile is padding
  const int end = first_token < span.len ? limit_of(a, span, min(plan.group_div(row0 + kRows - 1), span.len - 1)) : 0;
  const int len = min(plan.split_len, end - j0);  // positions of this tile in the split
  const int n_all = len > 0 ? (len + kChunk - 1) / kChunk : 0;
  const int n = n_all > part_wave ? (n_all - part_wave + wpt - 1) >> __builtin_ctz(wpt) : 0;  // this wave's chunks
  const uint32_t row_b = static_cast<uint32_t>(a.n_head_kv) * D;
  const uint8_t* kp = a.k_pool + kvh * D;
  const uint8_t* vp = a.v_pool + kvh * D;

  // Query operand: step s of lane (q4, col) holds 8 dimensions of row `col`,
  // in the order in which a lane's bytes of a K row come.
  u32x4_t q[kTerms][R::kSteps];
  {
    const int64_t at = (static_cast<int64_t>(b) * a.seq_len + token) * a.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int s = 0; s < R::kSteps; ++s) {
      const int d = D >= 64 ? 16 * (q4 + 4 * (s / 2)) + 8 * (s % 2) : 8 * q4;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (token < span.len && d < D) {
        if (kTerms == 1 && !a.k_new) {
          const u32x4_t w = *reinterpret_cast<const u32x4_t*>(static_cast<const bf16_t*>(a.q) + at + d);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[2 * e] = bf16_lo(w[e]);
            x[2 * e + 1] = bf16_hi(w[e]);
          }
        } else {
          const float* p = static_cast<const float*>(a.q) + at + d;
          const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(p), hi = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = lo[e];
            x[4 + e] = hi[e];
          }
        }
      }
      u32x4_t t[kTerms];
      split8<kTerms>(x, t);
#pragma unroll
      for (int k = 0; k < kTerms; ++k) q[k][s] = t[k];
    }
#pragma unroll
    for (int k = 0; k < kTerms; ++k)
#pragma unroll
      for (int s = 0; s < R::kSteps; ++s) asm volatile("" : "+v"(q[k][s]));  // loaded here, not between the tiles
  }

  float m = -INFINITY, l = 0.f;  // l: of this lane's positions
  f32x4_t acc[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float c2 = a.scale * kLog2e;

  // Bits of a chunk's positions: a page of the pool, and a row of zeros.
  uint64_t valid = 0, zero = 0;
  // Pool rows of the chunk, unusable ones replaced by a usable one, and its
  // scales' loads.
  auto load_rows = [&](int c) __attribute__((always_inline)) {
    const int t = chunk_at(c) + lane, lb = plan.block_div(t);
    const int pb = table[lane];
    const bool in = t < j0 + len, ok = in && lb < a.max_blocks && pb >= 0 && pb < a.n_blocks;
    const int r = ok ? pb * a.block_size + (t - lb * a.block_size) : -1;
    valid = __ballot(ok);
    zero = __ballot(in && !ok);
    const int first = valid ? __builtin_amdgcn_readlane(r, __builtin_ctzll(valid)) : 0;
    rows[lane] = ok ? r : first;
    const int64_t at = static_cast<int64_t>(ok ? pb : plan.block_div(first)) * a.n_head_kv + kvh;
    load_lds4(a.k_scales + at, ks + (c & 1) * kChunk);
    load_lds4(a.v_scales + at, vs + (c & 1) * kChunk);
  };
  const int lr = lane / R::kPieces, lc = lane % R::kPieces;  // this lane's row and piece of a load
  auto load_tile = [&](int it, bool v) __attribute__((always_inline)) {
    uint32_t r[kL];
#pragma unroll
    for (int i = 0; i < kL; ++i) r[i] = rows[it * R::kTile + i * R::kRowsPerLoad + lr];
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      const int tr = i * R::kRowsPerLoad + lr;
      const int piece = lc ^ (v ? v_place<D>(tr) : k_place<D>(tr));
      load_lds16((v ? vp : kp) + piece * 16 + static_cast<uint64_t>(r[i]) * row_b, ring + ((v ? kT : 0) + it) * R::kTileB + i * 1024);
    }
  };

  if (n > 0) {
    __builtin_amdgcn_s_waitcnt(wait_vm(0, true));
    asm volatile("" ::: "memory");
    load_rows(0);
    load_table(1);
    __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
    asm volatile("" ::: "memory");
#pragma unroll
    for (int it = 0; it < kT; ++it) load_tile(it, false);
#pragma unroll
    for (int it = 0; it < kT; ++it) load_tile(it, true);
  }
  for (int c = 0; c < n; ++c) {
    const bool more = c + 1 < n;
    const int at = chunk_at(c);
    const bool full = valid == ~0ull && at + kChunk <= first_limit;
    // Positions that this lane's row attends: rows of the pool, and rows of
    // zeros; bit 16 st + i belongs to score i of sc[st].
    uint64_t on = ~0ull, nil = 0ull;
    if (!full) {
      const uint64_t below = low_bits(limit - at);
      on = (valid & below) >> (4 * q4);
      nil = (zero & below) >> (4 * q4);
    }
    auto attends = [&](int st, int i) __attribute__((always_inline)) { return (on >> (16 * st + i) & 1) != 0; };
    const float* ks_now = ks + (c & 1) * kChunk;
    const float* vs_now = vs + (c & 1) * kChunk;

    // ---- scores.  In flight behind K tile `it`, with another chunk to come:
    // 2 kT - 1 tiles, and from the first on the next chunk's scales and the
    // table after it (three loads)
    f32x4_t sc[kSub];
#pragma unroll
    for (int it = 0; it < kT; ++it) {
      if (it == 0)
        __builtin_amdgcn_s_waitcnt(wait_vm((2 * kT - 1) * kL, false));
      else if (more)
        __builtin_amdgcn_s_waitcnt(wait_vm((2 * kT - 1) * kL + 3, false));
      else
        __builtin_amdgcn_s_waitcnt(wait_vm((2 * kT - 2) * kL, false));
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      if (it == 0 && more) {
        load_rows(c + 1);  // the table came before this tile
        load_table(c + 2);
      }
      constexpr int kSt = R::kTile / 16;
      u32x4_t w[kSt][D >= 64 ? D / 64 : 1];
#pragma unroll
      for (int u = 0; u < kSt; ++u) {
        const int r = 16 * u + col;
        const unsigned char* p = ring + it * R::kTileB + r * D;
        if constexpr (D >= 64) {
#pragma unroll
          for (int s = 0; s < D / 64; ++s)
            w[u][s] = *reinterpret_cast<const u32x4_t*>(p + (((q4 + 4 * s) ^ k_place<D>(r)) << 4));
        } else {
          const u32x2_t h =
              *reinterpret_cast<const u32x2_t*>(p + ((((q4 >> 1) ^ k_place<D>(r)) & (R::kPieces - 1)) << 4) + 8 * (q4 & 1));
          w[u][0] = D == 16 && q4 >= 2 ? u32x4_t{0u, 0u, 0u, 0u} : u32x4_t{h[0], h[1], 0u, 0u};
        }
      }
      f32x4_t kscale[kSt];
#pragma unroll
      for (int u = 0; u < kSt; ++u) kscale[u] = *reinterpret_cast<const f32x4_t*>(ks_now + (it * kSt + u) * 16 + 4 * q4);
      // the slot is refilled after its reads have returned
      __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_tile(it, false);
#pragma unroll
      for (int u = 0; u < kSt; ++u) {
        f32x4_t d{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < R::kSteps; ++s) {
          const u32x4_t kv = f8x8_to_bf16x8(w[u][s / 2][2 * (s % 2)], w[u][s / 2][2 * (s % 2) + 1]);
#pragma unroll
          for (int k = 0; k < kTerms; ++k) d = mfma16(kv, q[k][s], d);
        }
        const int st = it * kSt + u;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] *= kscale[u][i];
        if (!full) {
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = attends(st, i) ? d[i] : nil >> (16 * st + i) & 1 ? 0.f : -INFINITY;
        }
        sc[st] = d;
      }
    }

    // ---- softmax over the wave's positions so far
    float mx = -INFINITY;
#pragma unroll
    for (int st = 0; st < kSub; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[st][i]);
    mx = max_quarters(mx);
    if (__any((mx - m) * c2 > kLazy)) {
      const float top = fmaxf(m, mx);
      const float f = __builtin_amdgcn_exp2f((m - finite_base(top)) * c2);
      m = top;
      l *= f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] *= f;
    }
    const float base = finite_base(m) * c2;
    u32x4_t p[kTerms][kSub / 2];
#pragma unroll
    for (int g = 0; g < kSub / 2; ++g) {
      float w[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int st = 2 * g + u;
        const f32x4_t vscale = *reinterpret_cast<const f32x4_t*>(vs_now + st * 16 + 4 * q4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(sc[st][i], c2, -base));
          l += e;
          w[4 * u + i] = e * vscale[i];
        }
      }
      if (!full) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!attends(2 * g + e / 4, e % 4)) w[e] = 0.f;  // 0 times a scale that is not finite
      }
      // bf16 activations: the weights rounded to bf16, which the output's own
      // rounding matches
      u32x4_t t[kTerms];
      split8<kTerms>(w, t);
#pragma unroll
      for (int k = 0; k < kTerms; ++k) p[k][g] = t[k];
    }

    // ---- values
#pragma unroll
    for (int it = 0; it < kT; ++it) {
      if (more)
        __builtin_amdgcn_s_waitcnt(wait_vm((2 * kT - 1) * kL + 3, false));
      else if (it == 0)
        __builtin_amdgcn_s_waitcnt(wait_vm((kT - 1) * kL, false));
      else
        __builtin_amdgcn_s_waitcnt(wait_vm(0, false));
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      constexpr int kPg = R::kTile / 32;
      u32x2_t w[kPg][D / 16];
#pragma unroll
      for (int g = 0; g < kPg; ++g) {
        const int k = (lane & 15) >> 1, r = 16 * (k >> 2) + 4 * q4 + (k & 3);
        const uint32_t tile = lds_address(ring + (kT + it) * R::kTileB + (32 * g + r) * D + 8 * (lane & 1));
        uint32_t from[D / 16];
#pragma unroll
        for (int t = 0; t < D / 16; ++t) from[t] = tile + ((t ^ v_place<D>(r)) << 4);
        read_columns(from, w[g]);
      }
      __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_tile(it, true);
#pragma unroll
      for (int g = 0; g < kPg; ++g) {
        const int pg = it * kPg + g;
        bool bad = false;
        if (!full) {
          uint32_t any = 0;
#pragma unroll
          for (int t = 0; t < D / 16; ++t) any |= nan_bytes(w[g][t][0]) | nan_bytes(w[g][t][1]);
          bad = __any(any != 0);
        }
        if (__builtin_expect(bad, 0)) {
          float y[8];  // 1 where this lane's row attends the position
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = attends(2 * pg + e / 4, e % 4) ? 1.f : 0.f;
          u32x4_t one[1];
          split8<1>(y, one);
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            const uint32_t n0 = (nan_bytes(w[g][t][0]) >> 7) * 0xFFu, n1 = (nan_bytes(w[g][t][1]) >> 7) * 0xFFu;
            w[g][t][0] &= ~n0;
            w[g][t][1] &= ~n1;
            const f32x4_t hit = mfma16(f8x8_to_bf16x8(n0 & 0x38383838u, n1 & 0x38383838u), one[0],
                                       f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (hit[i] > 0.f) acc[t][i] = __builtin_nanf("");
          }
        }
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          const u32x4_t v = f8x8_to_bf16x8(w[g][t][0], w[g][t][1]);
#pragma unroll
          for (int k = 0; k < kTerms; ++k) acc[t] = mfma16(v, p[k][pg], acc[t]);
        }
      }
    }
  }
  // nothing of the wave is in flight beyond a table
  __builtin_amdgcn_s_waitcnt(wait_vm(0, true));
  asm volatile("" ::: "memory");

  // ---- the tile's waves merged in order
  float* o = reinterpret_cast<float*>(ring) + col * D;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4_t*>(o + 16 * t + 4 * q4) = acc[t];
  l = sum_quarters(l);
  if (lane < kRows) {
    stat[wave * kRows + lane] = m;
    stat[(kWaves + wave) * kRows + lane] = l;
  }
  __syncthreads();
  if (len <= 0 && plan.join) return;  // the join reads only the splits with positions
  const int64_t n_rows = static_cast<int64_t>(a.batch) * a.seq_len * a.n_head;
  for (int i = part_wave * kWave + lane; i < kRows * D / 4; i += wpt * kWave) {
    const int r = i / (D / 4), d = i % (D / 4) * 4, t = plan.group_div(row0 + r), h = kvh * G + row0 + r - t * G;
    if (t >= a.seq_len) break;
    const int w0 = wave - part_wave;
    float M = stat[w0 * kRows + r];
    for (int w = 1; w < wpt; ++w) M = fmaxf(M, stat[(w0 + w) * kRows + r]);
    const float base = finite_base(M) * c2;
    f32x4_t x{0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    for (int w = 0; w < wpt; ++w) {
      const float f = __builtin_amdgcn_exp2f(fmaf(stat[(w0 + w) * kRows + r], c2, -base));  // 0 without positions
      const f32x4_t y = *reinterpret_cast<const f32x4_t*>(lds + (w0 + w) * R::kWaveB + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(f, y[e], x[e]);
      L = fmaf(f, stat[(kWaves + w0 + w) * kRows + r], L);
    }
    const int64_t row = (static_cast<int64_t>(b) * a.seq_len + t) * a.n_head + h;
    if (!plan.join) {
      const bool none = t >= span.len || L == 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : x[e] / L;
      store4(a, row * D + d, x);
    } else {
      *reinterpret_cast<f32x4_t*>(a.part + (row * plan.n_split + split) * D + d) = x;
      if (d == 0)
        *reinterpret_cast<float2*>(a.part + n_rows * plan.n_split * D + (row * plan.n_split + split) * 2) = float2{M, L};
    }
  }
}

// ------------------------------------------------------------------ many rows
// Block (row tile of 128, K/V head, context split; sequence): wave w has 32
// rows, and the four share tiles of 128 positions, two in LDS: while one is
// computed the next is in flight (global_load_lds; one block barrier a tile).
// Scores: v_mfma_scale_f32_32x32x64_f8f6f4 with A = the K codes as they lie
// and B = q as two e4m3 terms under a power of two of the row: hi = e4m3(q/s),
// lo = e4m3(q/s - hi), exact for bf16 values down to s/4 and within s/1024
// below.  Two fp8 products cost what one bf16 product does and spare the
// conversion of K.  A lane holds, for row l % 32, positions 8 i + 4 (l / 32)
// + 0..3, which serve as the B operand of the second product in bf16
// (32x32x16) with A = V transposed, converted as it is read.  The denominator
// adds the weights before they are rounded to bf16 (2^-8 of each, at most,
// goes into the numerator); adding them as rounded, in v_dot2, waited for
// every product in flight, which the other vector instructions pass by.
// Bound by the matrix cores and the vector unit under the card's power: 64
// positions of 32 rows are 1024 cycles of products and about 900 of vector
// instructions at head_dim 128, which two waves overlap, but with every CU at
// it the clock falls to 1.7 - 1.95 GHz (products alone: 1.75).  8192 tokens
// of 8192, 32/8 heads x 128, causal: 503 to 535 us, 1.03 to 1.09 PFLOP/s where
// a library's bf16 product of 8192^3 reaches 1.2; without the interleaving of
// products and softmax 605.
constexpr int kBigRows = 128;
constexpr int kWaveRows = 32;
constexpr int kBigTile = 128;
constexpr int kStages = 2;

typedef __attribute__((ext_vector_type(8))) int i32x8_t;

__device__ __forceinline__ f32x16_t mfma32(const u32x4_t a, const u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                0, 0, 0);
}

// a times 2^(scale - 127), one scale for each lane's part of a row.
__device__ __forceinline__ f32x16_t mfma32_f8(const i32x8_t a, int scale, const i32x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, scale, 0, 127);
}

// Four codes times s (a power of two), then four times t, in bf16.
__device__ __forceinline__ u32x4_t scaled_bf16x8(uint32_t a, float s, uint32_t b, float t) {
  return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, t, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, t, true))};
}

template <int D>
struct Big {
  static constexpr int kPieces = D / 16;
  static constexpr int kRowsPerLoad = 1024 / D;
  static constexpr int kLoads = kBigTile / kRowsPerLoad / kWaves;  // of K, and of V, per wave and tile
  static constexpr int kTileB = kBigTile * D;
  static constexpr int kScaleB = kWaves * kWave * 4;
  static constexpr int kStageB = 2 * kTileB + kScaleB;
  static constexpr int kLds = kStages * kStageB + kThreads * 4 + kStages * kWaves * 8;
  static constexpr int kWaveTileRows = kBigTile / kWaves;
  static_assert(kLoads * kRowsPerLoad == kWaveTileRows, "a wave loads whole rows");
};

// As v_place, for the rows that one read of 32 columns touches: bits 0, 1 and
// 3 vary, and the piece's lowest bit.
template <int D>
__device__ __forceinline__ int v_place32(int r) {
  return D == 128 ? ((r >> 1) & 1) << 1 | ((r >> 3) & 1) << 2 : ((r >> 3) & 1) << 1;
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void paged_tile_kernel(PagedAttnArgs a, Plan plan) {
  using R = Big<D>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int n_split = plan.n_split, split_len = plan.split_len;
  uint32_t* flags = reinterpret_cast<uint32_t*>(lds + kStages * R::kStageB + kThreads * 4);  // [stage]: valid by wave, zero by wave
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane >> 5, col = lane & 31;
  const int G = plan.group;
  const int x = plan.split_div(blockIdx.x), split = blockIdx.x - x * n_split;
  const int g = plan.batch_div(x), b = x - g * a.batch;
  // the tiles of the last tokens, which attend most, go first, in every sequence
  const int tile = plan.tile_groups - 1 - g, row_tile = plan.kv_div(tile), kvh = tile - row_tile * a.n_head_kv;
  const int row0 = row_tile * kBigRows;
  const Span span = span_of(a, b);

  const int wave_row0 = row0 + wave * kWaveRows;
  const int token = plan.group_div(wave_row0 + col), head = kvh * G + wave_row0 + col - token * G;
  const int limit = limit_of(a, span, token);
  auto end_of = [&](int first, int n) {  // positions that rows [first, first + n) attend
    return plan.group_div(first) < span.len ? limit_of(a, span, min(plan.group_div(first + n - 1), span.len - 1)) : 0;
  };
  const int j0 = split * split_len;
  const int end = min(end_of(row0, kBigRows), j0 + split_len);  // of this block
  const int wave_end = min(end_of(wave_row0, kWaveRows), j0 + split_len);
  const int first_limit = limit_of(a, span, plan.group_div(wave_row0));
  const int n = end > j0 ? (end - j0 + kBigTile - 1) / kBigTile : 0;
  if (n == 0 && n_split > 1) return;  // the combine reads only the splits with positions

  const int* seq_table = a.tables + static_cast<int64_t>(b) * a.max_blocks;
  const uint32_t row_b = static_cast<uint32_t>(a.n_head_kv) * D;
  const uint8_t* kp = a.k_pool + kvh * D;
  const uint8_t* vp = a.v_pool + kvh * D;

  // ---- loads.  Lanes l and l % 32 stand for position 32 wave + l % 32 of a
  // tile.  All of them go to LDS, the table entries of the tile after it too,
  // where the compiler does not wait for a register.
  const int wp = wave * R::kWaveTileRows + (lane & 31);
  int next_j = j0 + wp, next_page = plan.block_div(next_j), next_off = next_j - next_page * a.block_size;
  const int page_step = plan.block_div(kBigTile), off_step = kBigTile - page_step * a.block_size;
  int* entries = reinterpret_cast<int*>(lds + kStages * R::kStageB) + wave * kWave;
  auto load_entries = [&]() __attribute__((always_inline)) {
    load_lds4(seq_table + min(next_page, a.max_blocks - 1), entries);
  };
  const int lr = lane / R::kPieces, lc = lane % R::kPieces;
  const float* scales_of = (lane & 32 ? a.v_scales : a.k_scales) + kvh;
  // The places of a wave's loads repeat every 16 rows.
  constexpr int kPlaces = 16 / R::kRowsPerLoad;
  const uint8_t *k_at[kPlaces], *v_at[kPlaces];
#pragma unroll
  for (int i = 0; i < kPlaces; ++i) {
    k_at[i] = kp + ((lc ^ k_place<D>(i * R::kRowsPerLoad + lr)) << 4);
    v_at[i] = vp + ((lc ^ v_place32<D>(i * R::kRowsPerLoad + lr)) << 4);
  }
  // A tile's loads: its rows (every lane's own position, then of each load),
  // the entries of the tile after it and this one's scales, and load i.
  struct Rows {
    int page;
    uint32_t r[R::kLoads];
  };
  auto load_rows = [&](int stage, Rows& rows) __attribute__((always_inline)) {
    const int entry = entries[lane];
    const bool in = next_j < end;
    const bool ok = (next_page < a.max_blocks) & (static_cast<uint32_t>(entry) < static_cast<uint32_t>(a.n_blocks)) & in;
    const uint32_t valid = static_cast<uint32_t>(__ballot(ok)), zero = static_cast<uint32_t>(__ballot(in & !ok));
    // unusable rows load a usable one (row 0 is there)
    const int from = __builtin_ctz(valid | 1u << 31);
    const int some_page = valid ? __builtin_amdgcn_readlane(entry, from) : 0;
    const int some_off = valid ? __builtin_amdgcn_readlane(next_off, from) : 0;
    rows.page = ok ? entry : some_page;
    const int use = rows.page * a.block_size + (ok ? next_off : some_off);
    if (lane < 2) flags[stage * 2 * kWaves + kWaves * lane + wave] = lane ? zero : valid;
#pragma unroll
    for (int i = 0; i < R::kLoads; ++i) rows.r[i] = __shfl(use, i * R::kRowsPerLoad + lr, kWave);
  };
  auto load_scales = [&](int stage, const Rows& rows) __attribute__((always_inline)) {
    next_j += kBigTile;
    next_page += page_step;
    next_off += off_step;
    const bool wrap = next_off >= a.block_size;
    next_off -= wrap ? a.block_size : 0;
    next_page += wrap ? 1 : 0;
    load_entries();
    load_lds4(scales_of + static_cast<uint64_t>(static_cast<uint32_t>(rows.page)) * static_cast<uint32_t>(a.n_head_kv),
              lds + stage * R::kStageB + 2 * R::kTileB + wave * kWave * 4);
  };
  auto load_part = [&](int stage, const Rows& rows, int i) __attribute__((always_inline)) {
    unsigned char* base = lds + stage * R::kStageB + (wave * R::kLoads + i) * 1024;
    const uint64_t off = static_cast<uint64_t>(rows.r[i]) * row_b;
    load_lds16_cached(k_at[i % kPlaces] + off, base);
    load_lds16_cached(v_at[i % kPlaces] + off, base + R::kTileB);
  };
  auto load_tile = [&](int stage) __attribute__((always_inline)) {
    Rows rows;
    load_rows(stage, rows);
    load_scales(stage, rows);
#pragma unroll
    for (int i = 0; i < R::kLoads; ++i) load_part(stage, rows, i);
  };

  // ---- q as two terms: lane (half, col) holds dimensions 64 s + 32 half + 0..31
  // of row col.  Asked for beside the first tile's table entries, and
  // converted (some 500 instructions) while that tile is loaded.
  if (n > 0) load_entries();
  i32x8_t qh[D / 64], ql[D / 64];
  float c2, q_scale;
  {
    const int64_t at = (static_cast<int64_t>(b) * a.seq_len + token) * a.q_stride + static_cast<int64_t>(head) * D;
    u32x4_t w[D / 64][4];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < D / 64; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[s][i] = u32x4_t{0u, 0u, 0u, 0u};
    if (token < span.len) {
#pragma unroll
      for (int s = 0; s < D / 64; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[s][i] = *reinterpret_cast<const u32x4_t*>(static_cast<const bf16_t*>(a.q) + at + 64 * s + 32 * half + 8 * i);
    }
    __builtin_amdgcn_s_waitcnt(wait_vm(0, true));
    asm volatile("" ::: "memory");
    if (n > 0) load_tile(0);
#pragma unroll
    for (int s = 0; s < D / 64; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(w[s][i][e] << 16 & 0x7FFFFFFFu, w[s][i][e] & 0x7FFF0000u));
    top = __float_as_uint(max_halves(__uint_as_float(min(top, 0x7F800000u))));
    float inv = 1.f;
    q_scale = pow2_scale(__uint_as_float(min(top, 0x7F7F0000u)), &inv);
#pragma unroll
    for (int s = 0; s < D / 64; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x2_t hi, lo;
        e4m3_codes8_x2(w[s][i], inv, hi, lo);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qh[s][2 * i + e] = static_cast<int>(hi[e]);
          ql[s][2 * i + e] = static_cast<int>(lo[e]);
        }
      }
    // a row that is not finite has scores that are NaN
    c2 = top >= 0x7F800000u ? __builtin_nanf("") : a.scale * kLog2e * q_scale;
#pragma unroll
    for (int s = 0; s < D / 64; ++s) asm volatile("" : "+v"(qh[s]), "+v"(ql[s]));  // loaded here, not between the tiles
  }

  float m = -INFINITY, l = 0.f;
  f32x16_t acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;

  // K of 64 positions of a stage, by (32 positions, 64 dimensions), and the
  // products of one, in both terms, times 2^(e8m0 - 127)
  auto keys = [&](const unsigned char* base, int h64, i32x8_t (&k)[2][D / 64]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < D / 64; ++s)
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        u32x4_t w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          w[e] = *reinterpret_cast<const u32x4_t*>(base + (64 * h64 + 32 * pt + col) * D +
                                                   (((4 * s + 2 * half + e) ^ k_place<D>(col)) << 4));
        k[pt][s] = __builtin_bit_cast(i32x8_t, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
      }
  };
  // V columns of 64 positions: v[s][d], 8 codes of positions 16 s + ...
  auto columns = [&](const unsigned char* base, int h64, u32x2_t (&v)[4][D / 32]) __attribute__((always_inline)) {
    const int k = (lane & 15) >> 1, r = 8 * (k >> 2) + 4 * half + (k & 3);  // and 16 s
    const uint32_t row = lds_address(base + R::kTileB + (64 * h64 + r) * D + 8 * (lane & 1));
    uint32_t from[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) from[d] = row + (((2 * d + (lane >> 4 & 1)) ^ v_place32<D>(r)) << 4);
    read_columns4<16 * D>(from, v);
  };
  int nan_from = INT32_MAX, nan_to = 0;  // positions among which V codes that are NaN were left out
  for (int t = 0; t < n; ++t) {
    // This wave's part of tile t is there, and the next tile's table entries,
    // and so is everyone's part after the barrier, which no wave passes
    // before all have read tile t - 1: its stage is free.
    __builtin_amdgcn_s_waitcnt(wait_vm(0, true));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    const bool more = t + 1 < n;
    const int at = j0 + t * kBigTile, other = ~t & 1;
    if (at >= wave_end) {  // none of this wave's rows
      if (more) load_tile(other);
      continue;
    }
    const unsigned char* base = lds + (t & 1) * R::kStageB;
    const float* scales = reinterpret_cast<const float*>(base + 2 * R::kTileB);  // by wave: 32 of K, 32 of V
    const uint32_t* fl = flags + (t & 1) * 2 * kWaves;
    i32x8_t k0[2][D / 64];
    keys(base, 0, k0);
    float ks[kWaves];  // of position col of each 32
    uint32_t su[kWaves], all = ~0u;  // scales of this lane's positions, K's and V's
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      ks[w] = scales[w * kWave + col];
      su[w] = __float_as_uint(scales[w * kWave + lane]);
      all &= __builtin_amdgcn_readfirstlane(static_cast<int>(fl[w]));
    }
    const bool full = all == ~0u && at + kBigTile <= first_limit;
    // Scales that are powers of two, V's one for four neighbouring positions,
    // cost nothing: the products take K's, the conversion of V takes V's.
    // Others multiply scores and weights.
    const bool pow2 = plan.aligned && !__any(((su[0] | su[1] | su[2] | su[3]) & 0x7FFFFFu) |
                                             (min(min(su[0], su[1]), min(su[2], su[3])) < 0x800000u) |
                                             (max(max(su[0], su[1]), max(su[2], su[3])) >= 0x7F800000u));
    // Tiles that every row attends, with scales that are powers of two: 64
    // positions' products run beside the other 64's softmax, and the first
    // 64's beside the next tile's loads.  Weights are taken against the maximum
    // as it stands, at first 0; where a lane's sum says that it has to be
    // raised, or lowered at first, the 64 positions are done again below.
    int done = 0;
    if (full && pow2) {
      const float mc = finite_base(m) * c2;
      int e8m0[4];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) e8m0[w] = static_cast<int>(__float_as_uint(ks[w]) >> 23);
      f32x16_t sc[2][2];
      u32x4_t p[2][4];
      u32x2_t v[4][D / 32];
      float w[2], vs[8], sums[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
      auto score = [&](int h64, const i32x8_t (&k)[2][D / 64], int i) __attribute__((always_inline)) {
        const int pt = i & 1, s = i >> 2;
        sc[h64][pt] = mfma32_f8(k[pt][s], e8m0[2 * h64 + pt], i & 2 ? ql[s] : qh[s], sc[h64][pt]);
      };
      // Weights 2 i and 2 i + 1 of 64 positions, after those before are added
      // to the sums and rounded to bf16.
      auto weigh = [&](int h64, int i) __attribute__((always_inline)) {
        float next[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (i < 16) next[e] = __builtin_amdgcn_exp2f(fmaf(sc[h64][i >> 3][2 * (i & 7) + e], c2, -mc));
        if (i > 0) {
          p[h64][(i - 1) >> 2][(i - 1) & 3] = pack_bf16x2(w[0], w[1]);
          sums[h64][0] += w[0];
          sums[h64][1] += w[1];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (i < 16) w[e] = next[e];
      };
      auto load_values = [&](int h64) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < 8; ++g) vs[g] = scales[(2 * h64 + (g >> 2)) * kWave + 32 + 8 * (g & 3) + 4 * half];
        columns(base, h64, v);
      };
      auto convert = [&](int i) __attribute__((always_inline)) {
        const int s = i / (D / 32), d = i % (D / 32);
        return scaled_bf16x8(v[s][d][0], vs[2 * s], v[s][d][1], vs[2 * s + 1]);
      };
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[h][0][i] = sc[h][1][i] = 0.f;
      Rows rows;
      constexpr int kProducts = D / 16;
#pragma unroll
      for (int i = 0; i < kProducts; ++i) {
        score(0, k0, i);
        __builtin_amdgcn_sched_barrier(0);
        // (behind the last tile, rows that nothing reads)
        if (i == 0) load_rows(other, rows);
        if (i == 1) load_scales(other, rows);
        if (i >= 2 && i - 2 < R::kLoads) load_part(other, rows, i - 2);
        __builtin_amdgcn_sched_barrier(0);
      }
      static_assert(kProducts - 2 >= R::kLoads, "every load has a product");
      i32x8_t k1[2][D / 64];
      keys(base, 1, k1);
      asm volatile("" : "+v"(sc[0][0]), "+v"(sc[0][1]));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (i % (256 / D) == 0) score(1, k1, i / (256 / D));
        weigh(0, i);
        __builtin_amdgcn_sched_barrier(0);
      }
      weigh(0, 16);
      load_values(0);
      // not moved behind the branch
      asm volatile("" : "+v"(sc[1][0]), "+v"(sc[1][1]), "+v"(p[0][0]), "+v"(p[0][1]), "+v"(p[0][2]), "+v"(p[0][3]));
      const float sum0 = sums[0][0] + sums[0][1];
      if (!__any(sum0 > kMaxSum || (m == -INFINITY && sum0 < 1.f / kMaxSum))) {
        l += sum0;
        m = finite_base(m);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const u32x4_t c = convert(i % (D / 8));
          weigh(1, i);
          if (i < D / 8) acc[i % (D / 32)] = mfma32(c, p[0][i / (D / 32) % 4], acc[i % (D / 32)]);
          __builtin_amdgcn_sched_barrier(0);
        }
        weigh(1, 16);
        done = 1;
        if (!__any(sums[1][0] + sums[1][1] > kMaxSum)) {
          l += sums[1][0] + sums[1][1];
          load_values(1);
#pragma unroll
          for (int i = 0; i < D / 8; ++i) acc[i % (D / 32)] = mfma32(convert(i), p[1][i / (D / 32)], acc[i % (D / 32)]);
          done = 2;
        }
      }
    } else if (more) {
      load_tile(other);
    }
#pragma unroll 1
    for (int h64 = done; h64 < 2; ++h64) {  // 64 positions at a time
      const int half_at = at + 64 * h64;
      if (half_at >= wave_end) break;
      float vs[8];  // of positions 8 g + 4 half + 0..3
#pragma unroll
      for (int g = 0; g < 8; ++g) vs[g] = 1.f;
      if (pow2) {
#pragma unroll
        for (int g = 0; g < 8; ++g) vs[g] = scales[(2 * h64 + (g >> 2)) * kWave + 32 + 8 * (g & 3) + 4 * half];
      }
      // Positions that this lane's row attends: rows of the pool, and rows of
      // zeros; bit 8 (i / 4) + i % 4 of word pt belongs to score i of sc[pt].
      uint32_t on[2] = {~0u, ~0u}, nil[2] = {0u, 0u};
      if (!full) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt) {
          const uint32_t below = static_cast<uint32_t>(low_bits(min(limit - half_at - 32 * pt, 32)));
          on[pt] = (fl[2 * h64 + pt] & below) >> (4 * half);
          nil[pt] = (fl[kWaves + 2 * h64 + pt] & below) >> (4 * half);
        }
      }

      // ---- scores
      f32x16_t sc[2];
      int e8m0[2];
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
        e8m0[pt] = pow2 ? static_cast<int>(__float_as_uint(scales[(2 * h64 + pt) * kWave + col]) >> 23) : 127;
      i32x8_t k[2][D / 64];
      keys(base, h64, k);
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[0][i] = sc[1][i] = 0.f;
#pragma unroll
      for (int s = 0; s < D / 64; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[i & 1] = mfma32_f8(k[i & 1][s], e8m0[i & 1], i & 2 ? ql[s] : qh[s], sc[i & 1]);
      if (!pow2) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[pt][i] *= scales[(2 * h64 + pt) * kWave + 8 * (i >> 2) + 4 * half + (i & 3)];
      }
      if (!full) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t bit = 1u << (8 * (i >> 2) + (i & 3));
            sc[pt][i] = on[pt] & bit ? sc[pt][i] : nil[pt] & bit ? 0.f : -INFINITY;
          }
      }
      float top4[4];  // four chains
#pragma unroll
      for (int g = 0; g < 4; ++g) top4[g] = sc[g >> 1][8 * (g & 1)];
#pragma unroll
      for (int i = 1; i < 8; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) top4[g] = fmaxf(top4[g], sc[g >> 1][8 * (g & 1) + i]);
      const float mx = max_halves(fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])));
      __builtin_amdgcn_sched_barrier(0);
      // ---- softmax
      if (__any((mx - m) * c2 > kLazy)) {
        const float top = fmaxf(m, mx);
        const float f = __builtin_amdgcn_exp2f((m - finite_base(top)) * c2);
        m = top;
        l *= f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= f;
      }
      const float mc = finite_base(m) * c2;
      u32x4_t p[4];
      float sums[2] = {0.f, 0.f};
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          w[i] = __builtin_amdgcn_exp2f(fmaf(sc[pt][i], c2, -mc));
          sums[i & 1] += w[i];
        }
        if (!pow2) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            w[i] *= scales[(2 * h64 + pt) * kWave + 32 + 8 * (i >> 2) + 4 * half + (i & 3)];
            if (!(on[pt] & 1u << (8 * (i >> 2) + (i & 3)))) w[i] = 0.f;  // 0 times a scale that is not finite
          }
        }
        split8<1>(w, &p[2 * pt]);
        split8<1>(w + 8, &p[2 * pt + 1]);
        if (pow2 && !full) {  // a row of zeros has its weight and no value
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t bits = on[pt] >> (8 * (2 * g + (e >> 1)) + 2 * (e & 1));
              p[2 * pt + g][e] &= (bits & 1 ? 0xFFFFu : 0u) | (bits & 2 ? 0xFFFF0000u : 0u);
            }
        }
      }
      l += sums[0] + sums[1];
      __builtin_amdgcn_sched_barrier(0);

      // ---- values
      u32x2_t v[4][D / 32];
      columns(base, h64, v);
      if (!full) {
        uint32_t any = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int d = 0; d < D / 32; ++d) any |= nan_bytes(v[s][d][0]) | nan_bytes(v[s][d][1]);
        if (__builtin_expect(__any(any != 0), 0)) {
          // for the rows that do not attend them: 0 * NaN is NaN; the others get theirs at the end
          nan_from = min(nan_from, half_at);
          nan_to = half_at + 64;
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
              v[s][d][0] &= ~((nan_bytes(v[s][d][0]) >> 7) * 0xFFu);
              v[s][d][1] &= ~((nan_bytes(v[s][d][1]) >> 7) * 0xFFu);
            }
        }
      }
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
          acc[d] = mfma32(scaled_bf16x8(v[s][d][0], vs[2 * s], v[s][d][1], vs[2 * s + 1]), p[s], acc[d]);
    }
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(0, true));  // the entries past the end

  // ---- this wave's rows: lane (half, col) holds dimensions 32 d + 8 i + 4 half + 0..3 of row col.
  // V codes that are NaN, in the tiles where they were left out
  for (int j = nan_from; j < min(nan_to, limit); ++j) {
    const int lb = plan.block_div(j), pb = lb < a.max_blocks ? seq_table[lb] : -1;
    if (pb < 0 || pb >= a.n_blocks) continue;
    const uint8_t* row = vp + (static_cast<int64_t>(pb) * a.block_size + j - lb * a.block_size) * row_b + 4 * half;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t nan = nan_bytes(*reinterpret_cast<const uint32_t*>(row + 32 * d + 8 * g));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (nan >> (8 * i) & 0x80u) acc[d][4 * g + i] = __builtin_nanf("");
      }
  }
  l = sum_halves(l);
  if (token >= a.seq_len) return;
  const int64_t row = (static_cast<int64_t>(b) * a.seq_len + token) * a.n_head + head;
  const int64_t n_rows = static_cast<int64_t>(a.batch) * a.seq_len * a.n_head;
  if (n_split == 1) {
    const float f = token >= span.len || l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x2_t w{pack_bf16x2(acc[d][4 * g] * f, acc[d][4 * g + 1] * f),
                        pack_bf16x2(acc[d][4 * g + 2] * f, acc[d][4 * g + 3] * f)};
        *reinterpret_cast<u32x2_t*>(static_cast<bf16_t*>(a.out) + row * D + 32 * d + 8 * g + 4 * half) =
            token >= span.len ? u32x2_t{0u, 0u} : w;
      }
  } else if (limit > j0) {
    float* part = a.part + (row * n_split + split) * D;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t*>(part + 32 * d + 8 * g + 4 * half) =
            f32x4_t{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
    if (half == 0)
      *reinterpret_cast<float2*>(a.part + n_rows * n_split * D + (row * n_split + split) * 2) = float2{m * q_scale, l};
  }
}

// ------------------------------------------------------------------ joining the splits
// D / 4 lanes take four dimensions of an output row each and add the splits
// that hold positions of it in order; with many splits a whole block takes
// the row, its groups of lanes every kGroups-th split, and the groups are
// merged in order.  Bound by latency: the first splits' statistics and
// outputs are asked for beside the lengths that say which of them count (the
// others' memory is there, and not used).  A decode step's own token and its
// positions of zeros (score 0, value 0) are one more split: its key and value
// as they were projected, not yet rounded to codes, against q in fp32.
constexpr int kJoin = 8;  // splits of a round

template <int D, bool kWide, bool kStep>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttnArgs a, Plan plan) {
  constexpr int kLanes = D / 4, kGroups = kWide ? kThreads / kLanes : 1;
  constexpr int kRound = kWide ? 4 : kJoin;
  __shared__ f32x4_t part_o[kWide ? kThreads : 1];
  __shared__ float part_m[kGroups], part_l[kGroups];
  const int n = plan.n_split, d = threadIdx.x % kLanes * 4, g = kWide ? threadIdx.x / kLanes : 0;
  const int i = kWide ? blockIdx.x : blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;  // (token, head)
  const int b = blockIdx.y, in_b = a.seq_len * a.n_head;
  if (i >= in_b) return;  // never with kWide
  const int64_t row = static_cast<int64_t>(b) * in_b + i;
  const float* part = a.part + row * n * D + d;
  const float2* stat = reinterpret_cast<const float2*>(a.part + static_cast<int64_t>(a.batch) * in_b * n * D) + row * n;
  f32x4_t v[kRound];
  float2 st[kRound];
  auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int s = min(s0 + u * kGroups, n - 1);
      st[u] = stat[s];
      v[u] = *reinterpret_cast<const f32x4_t*>(part + static_cast<int64_t>(s) * D);
    }
  };
  load(g);
  const int t = plan.head_div(i);
  const Span span = span_of(a, b);
  const int limit = limit_of(a, span, t), used = limit > 0 ? plan.len_div(limit - 1) + 1 : 0;
  const float c2 = a.scale * kLog2e;
  float M = -INFINITY, L = 0.f;
  f32x4_t o{0.f, 0.f, 0.f, 0.f};
  if (kStep && g == 0) {
    const f32x4_t qv = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(a.q) + row * D + d);
    const int64_t kv = (static_cast<int64_t>(b) * a.n_head_kv + plan.group_div(i)) * D + d;
    const f32x4_t kn = load4(a.k_new, a.dtype, kv), vn = load4(a.v_new, a.dtype, kv);
    float dot = fmaf(qv[3], kn[3], fmaf(qv[2], kn[2], fmaf(qv[1], kn[1], qv[0] * kn[0])));
#pragma unroll
    for (int w = kLanes / 2; w > 0; w /= 2) dot += __shfl_xor(dot, w, kLanes);
    const int zeros = a.max_ctx - span.cut;
    M = zeros > 0 ? fmaxf(dot, 0.f) : dot;
    const float base = finite_base(M) * c2, f = __builtin_amdgcn_exp2f(fmaf(dot, c2, -base));
    L = zeros > 0 ? fmaf(static_cast<float>(zeros), __builtin_amdgcn_exp2f(-base), f) : f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = f * vn[e];
  }
  for (int s0 = g; s0 < used; s0 += kRound * kGroups) {
    if (s0 > g) load(s0);
    float top = M;
#pragma unroll
    for (int u = 0; u < kRound; ++u)
      if (s0 + u * kGroups < used) top = fmaxf(top, st[u].x);
    const float base = finite_base(top) * c2, f = __builtin_amdgcn_exp2f(fmaf(M, c2, -base));
    M = top;
    L *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f;
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      if (s0 + u * kGroups < used) {
        const float w = __builtin_amdgcn_exp2f(fmaf(st[u].x, c2, -base));
        L = fmaf(st[u].y, w, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(v[u][e], w, o[e]);
      }
    }
  }
  if constexpr (kWide) {
    part_o[threadIdx.x] = o;
    if (d == 0) {
      part_m[g] = M;
      part_l[g] = L;
    }
    __syncthreads();
    if (g > 0) return;
#pragma unroll 4
    for (int k = 1; k < kGroups; ++k) M = fmaxf(M, part_m[k]);
    const float base = finite_base(M) * c2;
    L = 0.f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < kGroups; ++k) {
      const float w = __builtin_amdgcn_exp2f(fmaf(part_m[k], c2, -base));
      L = fmaf(part_l[k], w, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(part_o[k * kLanes + threadIdx.x][e], w, o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = L == 0.f ? 0.f : o[e] / L;
  store4(a, row * D + d, o);
}

// Which kernel, and how the context is cut: for two blocks per CU where the
// rows alone do not give them.
// The kernel for many rows where (row, position) pairs are at least 12 M and a
// K/V head has 32 rows: below, most of its 128-row blocks' time is latency,
// and the other's 16-row tiles fill the GPU (4 query heads x 128, 8 K/V heads;
// few rows against many rows: 512 tokens of 512 16.1 against 28.0 us, 128 of 2048
// 26.6 and 25.9, 64 of 8192 41.5 and 32.8, 8 x 256 of 256 34.5 and 22.9, 8 x 8
// of 8192 44.0 and 42.2).
constexpr double kBigPairs = 12 << 20;
constexpr int kBigFrom = 32;

Plan plan_of(int batch, int seq_len, int max_ctx, int n_head, int n_head_kv, int head_dim, int block_size, int dtype,
             bool step) {
  const int64_t rows = static_cast<int64_t>(seq_len) * (n_head / n_head_kv);
  const int64_t pairs = static_cast<int64_t>(batch) * n_head_kv;
  Plan p;
  p.aligned = block_size % 4 == 0;
  p.big = !step && dtype == DT_BF16 && head_dim >= 64 && rows >= kBigFrom &&
          static_cast<double>(pairs) * rows * max_ctx >= kBigPairs;
  int64_t blocks, n;
  int quantum;
  if (p.big) {
    p.waves_per_tile = 1;
    blocks = pairs * ((rows + kBigRows - 1) / kBigRows);
    n = 512 / blocks;
    // Splits of 512 positions at least (256 tokens of 2048 30.0 us with them,
    // 32.0 with shorter ones, 35.8 with 1024; 8 x 128 of 512 23.5 and 36.0), and
    // two only where there is much to halve (8 x 128 of 2048: 53.4 us with one,
    // 61.2 with two; of 8192 165 and 156).
    n = std::min<int64_t>(n, max_ctx / 512);
    if (n == 2 && max_ctx < 4096) n = 1;
    quantum = 2 * kBigTile;
  } else {
    // About 1024 waves, one per SIMD, which keep the memory as busy as twice
    // as many (64 x 8192 positions 176 against 171 us) and spend half the
    // prologues.  Two waves of a tile and two heads per block rather than
    // four and one (64 x 8192: 201 us, 16 x 4096: 30.6 against 33.2 us; half
    // of the pool rows' neighbouring parts are read together), until there
    // are so many splits that joining them costs more (1 x 32768: 27 against
    // 21 us); one where the tiles alone are enough.
    const int64_t tiles = n_head_kv * ((rows + kRows - 1) / kRows);
    p.waves_per_tile = batch * tiles >= 2048 ? 1 : 2;
    n = 512 / (batch * tiles);
    if (n > 16) {
      p.waves_per_tile = 4;
      n /= 2;
    }
    blocks = batch * ((tiles * p.waves_per_tile + kWaves - 1) / kWaves);
    quantum = kChunk * p.waves_per_tile;
  }
  if (n < 1) n = 1;
  int64_t len = (max_ctx + n - 1) / n;
  len = (len + quantum - 1) / quantum * quantum;
  if (len < quantum) len = quantum;
  n = (max_ctx + len - 1) / len;
  p.n_split = static_cast<int>(n < 1 ? 1 : n);
  p.join = step || p.n_split > 1;
  p.split_len = static_cast<int>(len);
  p.group = n_head / n_head_kv;
  p.tile_groups = static_cast<int>(blocks / batch);
  p.batch_div = Div::by(batch);
  p.split_div = Div::by(p.n_split);
  p.kv_div = Div::by(n_head_kv);
  p.group_div = Div::by(p.group);
  p.block_div = Div::by(block_size);
  p.head_div = Div::by(n_head);
  p.len_div = Div::by(p.split_len);
  return p;
}

// More LDS than 64 KiB is asked for once per kernel and device.
template <auto kKernel, int kLds>
hipError_t launch_attn(const PagedAttnArgs& a, const Plan& p, hipStream_t s) {
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(asked.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) return e;
    asked.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t x = static_cast<int64_t>(p.tile_groups) * a.batch * p.n_split;
  if (x > UINT32_MAX / kThreads) return hipErrorInvalidValue;  // a grid counts its threads in 32 bits
  hipLaunchKernelGGL(kKernel, dim3(static_cast<unsigned>(x)), dim3(kThreads), kLds, s, a, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const PagedAttnArgs& a, hipStream_t s) {
  const Plan p = plan_of(a.batch, a.seq_len, a.max_ctx, a.n_head, a.n_head_kv, D, a.block_size, a.dtype,
                         a.k_new != nullptr);
  hipError_t e = hipErrorNotSupported;
  if (p.big) {
    if constexpr (D >= 64) e = launch_attn<paged_tile_kernel<D>, Big<D>::kLds>(a, p, s);
  } else if (a.dtype == DT_F32) {
    e = launch_attn<paged_stream_kernel<D, 3>, Stream<D>::kLds>(a, p, s);
  } else {
    e = launch_attn<paged_stream_kernel<D, 1>, Stream<D>::kLds>(a, p, s);
  }
  if (e != hipSuccess) return e;
  if (p.join) {
    const int rows = a.seq_len * a.n_head, per_block = kThreads / (D / 4);
    const bool wide = p.n_split > kJoin;
    const dim3 grid(wide ? rows : (rows + per_block - 1) / per_block, a.batch);
    if (a.k_new)
      hipLaunchKernelGGL((wide ? paged_join_kernel<D, true, true> : paged_join_kernel<D, false, true>), grid,
                         dim3(kThreads), 0, s, a, p);
    else
      hipLaunchKernelGGL((wide ? paged_join_kernel<D, true, false> : paged_join_kernel<D, false, false>), grid,
                         dim3(kThreads), 0, s, a, p);
  }
  return hipGetLastError();
}

}  // namespace

bool paged_attn_supported(int head_dim) {
  return head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128;
}

size_t paged_attn_workspace_floats(int batch, int seq_len, int max_ctx, int n_head, int n_head_kv, int head_dim,
                                   int dtype, bool step) {
  if (batch == 0 || seq_len == 0) return 0;
  const Plan p = plan_of(batch, seq_len, max_ctx, n_head, n_head_kv, head_dim, 1, dtype, step);
  if (!p.join) return 0;
  return static_cast<size_t>(batch) * seq_len * n_head * p.n_split * (head_dim + 2);
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t s) {
  if (a.batch == 0 || a.seq_len == 0) return hipSuccess;
  switch (a.head_dim) {
    case 16: return launch_dim<16>(a, s);
    case 32: return launch_dim<32>(a, s);
    case 64: return launch_dim<64>(a, s);
    case 128: return launch_dim<128>(a, s);
    default: return hipErrorNotSupported;
  }
}

}  // namespace fmoe
