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
__device__ __forceinline__ void load_lds4(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0);
}

// Eight codes of one column from eight rows of a tile in LDS: the lanes
// 2k and 2k + 1 of a group of 16 name row k's 8 low and 8 high columns, and
// lane c of the group gets column c, row k in byte k.
__device__ __forceinline__ u32x2_t read_columns(const unsigned char* p) {
  typedef __attribute__((ext_vector_type(2))) int i32x2_t;
  const auto v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (__attribute__((address_space(3))) i32x2_t*)(__attribute__((address_space(3))) void*)p);
  return __builtin_bit_cast(u32x2_t, v);
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
  const int64_t ctx = static_cast<int64_t>(max(a.ctx_lens[b], 0)) + a.ctx_add;
  s.pos = ctx - s.len;
  s.cut = static_cast<int>(min(ctx, static_cast<int64_t>(a.max_ctx)));
  return s;
}

// Positions that token t attends: those below the result.
__device__ __forceinline__ int limit_of(const PagedAttnArgs& a, const Span& s, int t) {
  if (t >= s.len) return 0;
  return a.causal ? static_cast<int>(min(max(s.pos + t + 1, int64_t{0}), static_cast<int64_t>(s.cut))) : s.cut;
}

__device__ __forceinline__ void store_out(const PagedAttnArgs& a, int64_t i, float v) {
  if (a.out_dtype == DT_F32)
    static_cast<float*>(a.out)[i] = v;
  else
    static_cast<bf16_t*>(a.out)[i] = f32_to_bf16(v);
}

// ------------------------------------------------------------------ few rows
// Block (row tile of 16, K/V head, context split; sequence): its four waves
// take chunks of 128 positions in turn, each through a ring of its own in
// LDS, and are merged at the end.  K and V codes pass through the ring once,
// by global_load_lds, in tiles that are refilled as soon as they are read, so
// that loads stay in flight through the arithmetic; so do the page table and
// the scales of the next chunk.
// Scores: v_mfma_f32_16x16x32_bf16 with A = 16 positions x 32 dimensions of
// K (codes are exact in bf16), B = the 16 query rows: a lane then holds, for
// row l % 16, positions 4 (l / 16) + i of each 16.  That is the B operand of
// the second product as it stands, with A = V transposed (ds_read_b64_tr_b8)
// taken in the same order of positions.  fp32 activations: q and the weights
// as three bf16 terms.
// A chunk that not every row attends in full takes the masked path: scores
// replaced by selects, and V codes that are NaN kept from the rows that do
// not attend them (0 * NaN is NaN) by a product of indicators of its own.
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kRows = 16;
constexpr int kChunk = 128;
constexpr int kSub = kChunk / 16;  // groups of 16 positions

template <int D>
struct Stream {
  static constexpr int kRowsPerLoad = 1024 / D;                             // a load is 64 lanes x 16 bytes
  static constexpr int kTile = kRowsPerLoad > 32 ? kRowsPerLoad : 32;       // positions
  static constexpr int kLoads = kTile / kRowsPerLoad;
  static constexpr int kTiles = kChunk / kTile;
  static constexpr int kTileB = kTile * D;
  static constexpr int kRing = kTiles * kTileB;
  static constexpr int kWaveB = kRing + 4 * kChunk * 4;  // + table, rows, K and V scales of a chunk
  static constexpr int kChunks16 = D / 16;               // 16-byte pieces of a row
  static constexpr int kSteps = D >= 32 ? D / 32 : 1;    // products over the dimensions
  static constexpr int kLds = kWaves * kWaveB + 2 * kWaves * kRows * 4;
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

template <int D, int kTerms>
__global__ __launch_bounds__(kThreads, 2) void paged_stream_kernel(PagedAttnArgs a, int n_split, int split_len) {
  using R = Stream<D>;
  constexpr int kL = R::kLoads, kT = R::kTiles;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int q4 = lane >> 4, col = lane & 15;
  const int b = blockIdx.y;
  const int split = blockIdx.x % n_split, kvh = blockIdx.x / n_split % a.n_head_kv;
  const int row0 = static_cast<int>(blockIdx.x / n_split / a.n_head_kv) * kRows;
  const int G = a.n_head / a.n_head_kv;
  const Span span = span_of(a, b);

  // This lane's query row (column `col` of the products).
  const int token = (row0 + col) / G, head = kvh * G + (row0 + col) % G;
  const int limit = limit_of(a, span, token);
  const int last_token = min((row0 + kRows - 1) / G, span.len - 1);
  const int first_limit = limit_of(a, span, row0 / G);  // 0: the tile is padding
  const int end = row0 / G < span.len ? limit_of(a, span, last_token) : 0;
  const int j0 = split * split_len;
  const int len = min(split_len, end - j0);  // positions of this block
  if (len <= 0 && n_split > 1) return;       // the combine reads only the splits with positions

  unsigned char* ring = lds + wave * R::kWaveB;
  int* table = reinterpret_cast<int*>(ring + R::kRing);
  int* rows = table + kChunk;
  float* ks = reinterpret_cast<float*>(rows + kChunk);
  float* vs = ks + kChunk;
  float* stat = reinterpret_cast<float*>(lds + kWaves * R::kWaveB);  // [waves][16] maxima, then sums

  const int n_all = len > 0 ? (len + kChunk - 1) / kChunk : 0;
  const int n = n_all > wave ? (n_all - wave + kWaves - 1) / kWaves : 0;  // this wave's chunks
  const int* seq_table = a.tables + static_cast<int64_t>(b) * a.max_blocks;
  const int64_t row_b = static_cast<int64_t>(a.n_head_kv) * D;
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
        if (kTerms == 1) {
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

  float m = -INFINITY, l = 0.f;
  f32x4_t acc[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float c2 = a.scale * kLog2e;

  // Chunk c of this wave: its first position within the sequence.
  auto chunk_at = [&](int c) { return j0 + (c * kWaves + wave) * kChunk; };
  // The chunk's page table entries, into LDS (positions past the split's end
  // read the entry of its last one).
  auto load_table = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = min(chunk_at(c) + h * kWave + lane, j0 + len - 1);
      load_lds4(seq_table + min(j / a.block_size, a.max_blocks - 1), table + h * kWave);
    }
  };
  // Bits of the chunk's positions: a page of the pool, and a row of zeros.
  uint64_t valid[2], zero[2], valid_now[2], zero_now[2];
  // Pool rows of the chunk, unusable ones replaced by a usable one, and its
  // scales' loads.
  auto load_rows = [&](int c) __attribute__((always_inline)) {
    int r[2], pb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = chunk_at(c) + h * kWave + lane;
      const int lb = t / a.block_size;
      pb[h] = table[h * kWave + lane];
      const bool in = t < j0 + len, ok = lb < a.max_blocks && pb[h] >= 0 && pb[h] < a.n_blocks;
      r[h] = in && ok ? pb[h] * a.block_size + (t - lb * a.block_size) : -1;
      valid[h] = __ballot(in && ok);
      zero[h] = __ballot(in && !ok);
    }
    const int first = valid[0]   ? __builtin_amdgcn_readlane(r[0], __builtin_ctzll(valid[0]))
                      : valid[1] ? __builtin_amdgcn_readlane(r[1], __builtin_ctzll(valid[1]))
                                 : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool ok = r[h] >= 0;
      rows[h * kWave + lane] = ok ? r[h] : first;
      const int64_t at = static_cast<int64_t>(ok ? pb[h] : first / a.block_size) * a.n_head_kv + kvh;
      load_lds4(a.k_scales + at, ks + h * kWave);
      load_lds4(a.v_scales + at, vs + h * kWave);
    }
  };
  const int lr = lane / R::kChunks16, lc = lane % R::kChunks16;  // this lane's row and piece of a load
  auto load_tile = [&](const uint8_t* pool, int it, bool v) __attribute__((always_inline)) {
    int r[kL];
#pragma unroll
    for (int i = 0; i < kL; ++i) r[i] = rows[it * R::kTile + i * R::kRowsPerLoad + lr];
#pragma unroll
    for (int i = 0; i < kL; ++i) {
      const int tr = i * R::kRowsPerLoad + lr;
      const int piece = lc ^ (v ? v_place<D>(tr) : k_place<D>(tr));
      load_lds16(pool + r[i] * row_b + piece * 16, ring + it * R::kTileB + i * 1024);
    }
  };

  if (n > 0) {
    load_table(0);
    __builtin_amdgcn_s_waitcnt(wait_vm(0, true));
    asm volatile("" ::: "memory");
    load_rows(0);
    __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
    asm volatile("" ::: "memory");
#pragma unroll
    for (int it = 0; it < kT; ++it) load_tile(kp, it, false);
  }
  for (int c = 0; c < n; ++c) {
    const bool more = c + 1 < n;
    const int at = chunk_at(c);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      valid_now[h] = valid[h];
      zero_now[h] = zero[h];
    }
    const bool full = (valid_now[0] & valid_now[1]) == ~0ull && at + kChunk <= first_limit;
    // Whether this lane's row attends position 16 st + 4 q4 + i of the chunk,
    // a row of the pool.
    auto attends = [&](int st, int i) __attribute__((always_inline)) {
      return (valid_now[st / 4] >> (16 * (st % 4) + 4 * q4 + i) & 1) && at + 16 * st + 4 * q4 + i < limit;
    };
    load_table(min(c + 1, n - 1));  // always two loads, so that the waits below count alike

    // ---- scores.  In flight behind K tile `it`: the tiles after it (K,
    // then V) and the table
    f32x4_t sc[kSub];
#pragma unroll
    for (int it = 0; it < kT; ++it) {
      __builtin_amdgcn_s_waitcnt(wait_vm((kT - 1) * kL + 2, false));
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
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
              *reinterpret_cast<const u32x2_t*>(p + ((((q4 >> 1) ^ k_place<D>(r)) & (R::kChunks16 - 1)) << 4) + 8 * (q4 & 1));
          w[u][0] = D == 16 && q4 >= 2 ? u32x4_t{0u, 0u, 0u, 0u} : u32x4_t{h[0], h[1], 0u, 0u};
        }
      }
      f32x4_t kscale[kSt];
#pragma unroll
      for (int u = 0; u < kSt; ++u) kscale[u] = *reinterpret_cast<const f32x4_t*>(ks + (it * kSt + u) * 16 + 4 * q4);
      // the slot is refilled after its reads have returned
      __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
      __builtin_amdgcn_sched_barrier(0);
      load_tile(vp, it, true);
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
          const uint64_t zm = zero_now[st / 4] >> (16 * (st % 4) + 4 * q4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            d[i] = attends(st, i) ? d[i] : zm >> i & 1 && at + 16 * st + 4 * q4 + i < limit ? 0.f : -INFINITY;
        }
        sc[st] = d;
      }
    }

    // ---- softmax over the wave's positions so far
    float mx = m;
#pragma unroll
    for (int st = 0; st < kSub; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[st][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
    mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
    const float base = finite_base(mx) * c2;
    const float f = __builtin_amdgcn_exp2f(fmaf(m, c2, -base));
    m = mx;
    float sum = 0.f;
    u32x4_t p[kTerms][kSub / 2];
#pragma unroll
    for (int g = 0; g < kSub / 2; ++g) {
      float w[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int st = 2 * g + u;
        const f32x4_t vscale = *reinterpret_cast<const f32x4_t*>(vs + st * 16 + 4 * q4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(sc[st][i], c2, -base));
          sum += e;
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
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    l = fmaf(l, f, sum);
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] *= f;

    // ---- values.  In flight behind V tile `it`: the V tiles after it and,
    // with another chunk, its scales and K tiles
#pragma unroll
    for (int it = 0; it < kT; ++it) {
      if (it == 0)
        __builtin_amdgcn_s_waitcnt(wait_vm((kT - 1) * kL, false));
      else if (more)
        __builtin_amdgcn_s_waitcnt(wait_vm((kT - 1) * kL + 4, false));
      else if (it == 1)
        __builtin_amdgcn_s_waitcnt(wait_vm((kT > 2 ? kT - 2 : 0) * kL, false));
      else if (it == 2)
        __builtin_amdgcn_s_waitcnt(wait_vm((kT > 3 ? kT - 3 : 0) * kL, false));
      else
        __builtin_amdgcn_s_waitcnt(wait_vm(0, false));
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      constexpr int kPg = R::kTile / 32;
      u32x2_t w[kPg][D / 16];
#pragma unroll
      for (int g = 0; g < kPg; ++g) {
        const int k = (lane & 15) >> 1, r = 16 * (k >> 2) + 4 * q4 + (k & 3);
        const unsigned char* tile = ring + it * R::kTileB + (32 * g + r) * D + 8 * (lane & 1);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) w[g][t] = read_columns(tile + ((t ^ v_place<D>(r)) << 4));
      }
      __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
      __builtin_amdgcn_sched_barrier(0);
      if (more) {
        if (it == 0) {
          load_rows(c + 1);  // the table came before this tile
          __builtin_amdgcn_s_waitcnt(wait_vm(63, true));
          asm volatile("" ::: "memory");
        }
        load_tile(kp, it, false);
      }
#pragma unroll
      for (int g = 0; g < kPg; ++g) {
        const int pg = it * kPg + g;
        bool bad = false;
        if (!full) {
          uint32_t any = 0;
#pragma unroll
          for (int t = 0; t < D / 16; ++t) any |= nan_bytes(w[g][t][0]) | nan_bytes(w[g][t][1]);
          bad = __ballot(any != 0) != 0;
        }
        if (__builtin_expect(bad, 0)) {
          // 1 where this lane's row attends the position
          float on[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) on[e] = attends(2 * pg + e / 4, e % 4) ? 1.f : 0.f;
          u32x4_t one[1];
          split8<1>(on, one);
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
  // nothing of the wave is in flight beyond the table of the last chunk
  __builtin_amdgcn_s_waitcnt(wait_vm(0, true));
  asm volatile("" ::: "memory");

  // ---- the waves merged in order
  float* o = reinterpret_cast<float*>(ring) + col * D;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) *reinterpret_cast<f32x4_t*>(o + 16 * t + 4 * q4) = acc[t];
  if (lane < kRows) {
    stat[wave * kRows + lane] = m;
    stat[(kWaves + wave) * kRows + lane] = l;
  }
  __syncthreads();
  for (int i = tid; i < kRows * D; i += kThreads) {
    const int r = i / D, d = i % D, t = (row0 + r) / G, h = kvh * G + (row0 + r) % G;
    if (t >= a.seq_len) break;
    float M = stat[r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, stat[w * kRows + r]);
    const int64_t zeros = n_split == 1 && t < span.len ? max(a.zero_to - span.cut, 0) : 0;
    if (zeros > 0) M = fmaxf(M, 0.f);
    const float base = finite_base(M) * c2;
    float x = 0.f, L = zeros > 0 ? static_cast<float>(zeros) * __builtin_amdgcn_exp2f(-base) : 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(fmaf(stat[w * kRows + r], c2, -base));  // 0 for a wave without positions
      x = fmaf(f, reinterpret_cast<const float*>(lds + w * R::kWaveB)[i], x);
      L = fmaf(f, stat[(kWaves + w) * kRows + r], L);
    }
    const int64_t row = (static_cast<int64_t>(b) * a.seq_len + t) * a.n_head + h;
    if (n_split == 1) {
      store_out(a, row * D + d, t >= span.len || L == 0.f ? 0.f : x / L);
    } else {
      const int64_t n_rows = static_cast<int64_t>(a.batch) * a.seq_len * a.n_head;
      a.part[(row * n_split + split) * D + d] = x;
      if (d < 2) a.part[n_rows * n_split * D + (row * n_split + split) * 2 + d] = d == 0 ? M : L;
    }
  }
}

// ------------------------------------------------------------------ joining the splits
// One wave per output row: the splits that hold positions of it, in order.
constexpr int kJoinUnroll = 8;

template <int D>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(PagedAttnArgs a, int n_split, int split_len) {
  constexpr int kPer = D > kWave ? D / kWave : 1;  // dimensions of a lane
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t n_rows = static_cast<int64_t>(a.batch) * a.seq_len * a.n_head;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
  if (row >= n_rows) return;
  const int t = static_cast<int>(row / a.n_head % a.seq_len);
  const int b = static_cast<int>(row / a.n_head / a.seq_len);
  const Span span = span_of(a, b);
  const int used = (limit_of(a, span, t) + split_len - 1) / split_len;
  const int zeros = t < span.len ? max(a.zero_to - span.cut, 0) : 0;
  const float* part = a.part + row * n_split * D;
  const float2* stat = reinterpret_cast<const float2*>(a.part + n_rows * n_split * D) + row * n_split;
  const float c2 = a.scale * kLog2e;
  float M = zeros > 0 ? 0.f : -INFINITY;
  for (int s = lane; s < used; s += kWave) M = fmaxf(M, stat[s].x);
  M = wave_max(M);
  const float base = finite_base(M) * c2;
  float L = 0.f;
  for (int s = lane; s < used; s += kWave) L = fmaf(stat[s].y, __builtin_amdgcn_exp2f(fmaf(stat[s].x, c2, -base)), L);
  L = wave_sum(L) + (zeros > 0 ? static_cast<float>(zeros) * __builtin_amdgcn_exp2f(-base) : 0.f);
  float o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
  if (lane * kPer < D) {
    for (int s0 = 0; s0 < used; s0 += kJoinUnroll) {
      float v[kJoinUnroll][kPer], m[kJoinUnroll];
#pragma unroll
      for (int u = 0; u < kJoinUnroll; ++u) {
        const int s = min(s0 + u, used - 1);
        m[u] = stat[s].x;
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[u][e] = part[static_cast<int64_t>(s) * D + lane * kPer + e];
      }
#pragma unroll
      for (int u = 0; u < kJoinUnroll; ++u) {
        const float f = s0 + u < used ? __builtin_amdgcn_exp2f(fmaf(m[u], c2, -base)) : 0.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (s0 + u < used) o[e] = fmaf(v[u][e], f, o[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) store_out(a, row * D + lane * kPer + e, L == 0.f ? 0.f : o[e] / L);
  }
}

// How the context is cut: splits of split_len positions, for two blocks per
// CU where the rows alone do not give them.
struct Plan {
  int n_split, split_len;
};

Plan plan_of(int batch, int seq_len, int max_ctx, int n_head, int n_head_kv) {
  const int64_t rows = static_cast<int64_t>(seq_len) * (n_head / n_head_kv);
  const int64_t blocks = static_cast<int64_t>(batch) * n_head_kv * ((rows + kRows - 1) / kRows);
  int64_t n = blocks > 0 ? (512 + blocks - 1) / blocks : 1;
  int64_t len = (max_ctx + n - 1) / n;
  len = (len + 2 * kChunk - 1) / (2 * kChunk) * (2 * kChunk);  // no shorter than two waves' chunks
  if (len < 2 * kChunk) len = 2 * kChunk;
  n = (max_ctx + len - 1) / len;
  return Plan{static_cast<int>(n < 1 ? 1 : n), static_cast<int>(len)};
}

template <int D, int kTerms>
void launch_stream(const PagedAttnArgs& a, const Plan& p, hipStream_t s) {
  constexpr int lds = Stream<D>::kLds;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(paged_stream_kernel<D, kTerms>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  (void)attr;
  const int64_t rows = static_cast<int64_t>(a.seq_len) * (a.n_head / a.n_head_kv);
  const int64_t x = (rows + kRows - 1) / kRows * a.n_head_kv * p.n_split;
  hipLaunchKernelGGL((paged_stream_kernel<D, kTerms>), dim3(static_cast<unsigned>(x), a.batch), dim3(kThreads), lds, s,
                     a, p.n_split, p.split_len);
}

template <int D>
hipError_t launch_dim(const PagedAttnArgs& a, hipStream_t s) {
  const Plan p = plan_of(a.batch, a.seq_len, a.max_ctx, a.n_head, a.n_head_kv);
  if (a.q_dtype == DT_F32)
    launch_stream<D, 3>(a, p, s);
  else
    launch_stream<D, 1>(a, p, s);
  if (p.n_split > 1) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.seq_len * a.n_head;
    hipLaunchKernelGGL((paged_join_kernel<D>), dim3(static_cast<unsigned>((rows + kWaves - 1) / kWaves)),
                       dim3(kThreads), 0, s, a, p.n_split, p.split_len);
  }
  return hipGetLastError();
}

}  // namespace

bool paged_attn_supported(int head_dim) {
  return head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128;
}

size_t paged_attn_workspace_floats(int batch, int seq_len, int max_ctx, int n_head, int n_head_kv, int head_dim, int) {
  const Plan p = plan_of(batch, seq_len, max_ctx, n_head, n_head_kv);
  if (p.n_split <= 1) return 0;
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
