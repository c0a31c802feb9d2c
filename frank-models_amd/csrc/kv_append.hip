// Appending new tokens to a paged K/V cache, with the rotary position applied
// on the way: keys are rotated and written with the values into the pages of
// their sequence, queries are rotated with the same angles.
//
// Pool pages [n_blocks, block_size, n_head_kv, head_dim] hold either the
// activations' type or e4m3 codes with one scale for each (page, head).  With
// codes, the values x of an append to rows [r0, r1) of a page and a head set
//   S' = max(S, s(max |x|)) for r0 > 0 (the page holds earlier rows at S),
//   S' = s(max |x|)         for r0 = 0 (a page begun anew),
// where s(a) is the least power of two with a <= 448 s(a); rows below r0 are
// rounded again from S to S' where S' > S, the new rows are e4m3(x / S').
// Powers of two make the second rounding exact but for what falls below the
// codes' smallest normal value, 2^-15 of the page's largest.
#include "common.h"
#include "launch.h"

namespace fmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxHeadDim = 128;
constexpr int kVec = 8;           // elements of a lane's load
constexpr int kAngleFloats = 8192;  // LDS for (cos, sin): rows of a chunk x head_dim

// Eight elements as they lie.
template <typename T>
struct Vec;
template <>
struct Vec<bf16_t> {
  u32x4_t w;
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
};
template <>
struct Vec<float> {
  f32x4_t a, b;
  __device__ __forceinline__ void get(float* x) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  }
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4_t*>(p) = f32x4_t{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4_t*>(p) = u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                             pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  }
}

// Eight values times inv as codes, round to nearest even; what is not finite
// becomes NaN (v_cvt_pk_fp8_f32 gives NaN beyond 464, and finite values are
// within 448 of the scale that inv inverts).
__device__ __forceinline__ u32x2_t codes8(const float* x, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * d] * inv, x[4 * d + 1] * inv, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * d + 2] * inv, x[4 * d + 3] * inv, c, true);
    w[d] = static_cast<uint32_t>(c);
  }
  return u32x2_t{w[0], w[1]};
}

__device__ __forceinline__ void values8(u32x2_t c, float* x) {
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[d]), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c[d]), true);
    x[4 * d] = lo[0];
    x[4 * d + 1] = lo[1];
    x[4 * d + 2] = hi[0];
    x[4 * d + 3] = hi[1];
  }
}

struct Plan {
  int pages;  // that a sequence's new tokens can touch
  Div page_div, block_div;  // by pages, by block_size
};

// The page of a sequence's first new token, rounded down also for positions
// before the sequence.
__device__ __forceinline__ int first_page(const Plan& p, int start) {
  return start >= 0 ? p.block_div(start) : -1 - p.block_div(-1 - start);
}

// The new tokens [lo, hi) of a sequence from `start` that lie in its page lp.
__device__ __forceinline__ void page_tokens(int64_t lp, int start, int seq_len, int block_size, int& lo, int& hi) {
  const int64_t first = lp * block_size - start;
  lo = static_cast<int>(first > 0 ? min(first, static_cast<int64_t>(seq_len)) : 0);
  hi = static_cast<int>(min(max(first + block_size, static_cast<int64_t>(0)), static_cast<int64_t>(seq_len)));
}

__device__ __forceinline__ double2 cmul(double2 a, double2 b) {
  return double2{a.x * b.x - a.y * b.y, a.x * b.y + a.y * b.x};
}

// Block (page of the new tokens, group of heads, sequence).  An item is one
// K, V or Q head of the page's new tokens; a wave takes an item, so a head's
// maximum needs no barrier.  Bound by memory: 4 x 2048 tokens of 32/8 heads x
// 128 in bf16 to codes in pages of 32, 184 MB, take 37.6 us, 4.9 TB/s where a
// copy reaches 5.2; for a decode step's few tokens by one round trip after
// another: start, table entry, page scale (61 tokens 7.1 us).
// T: activations.  C: codes (the pool holds e4m3), else the pool holds T.
template <typename T, bool C, int kBatch>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendArgs a, Plan plan) {
  extern __shared__ __attribute__((aligned(16))) float2 angles[];  // [rows of a chunk][D / 2]
  __shared__ double2 turns[2][kMaxHeadDim / 2];
  const int b = blockIdx.z, x = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int D = 1 << a.log2_dim, bs = a.block_size;
  const int start = a.start[b];
  const int len = a.lens ? min(max(a.lens[b], 0), a.seq_len) : a.seq_len;  // tokens that are cached
  const int64_t lp = static_cast<int64_t>(first_page(plan, start)) + x;
  int s0, s1;
  page_tokens(lp, start, a.seq_len, bs, s0, s1);
  if (s0 >= s1) return;
  const int n = s1 - s0, n_kv = min(len, s1) - s0;
  const int r0 = static_cast<int>(static_cast<int64_t>(start) + s0 - lp * bs);

  // The page, and whether a later append of this call names it too: then that
  // one alone writes it.
  int64_t page = -1;
  if (n_kv > 0 && lp >= 0 && lp < a.max_blocks) {
    page = a.tables[static_cast<int64_t>(b) * a.max_blocks + lp];
    if (page >= a.n_blocks) page = -1;
  }
  bool later = false;
  if (page >= 0) {
    // (b2, x2): sequence and page, kThreads pages on in each round
    const int on = plan.page_div(kThreads), on_x = kThreads - on * plan.pages, skip = plan.page_div(tid);
    int64_t x2 = static_cast<int64_t>(x) + 1 + tid - static_cast<int64_t>(skip) * plan.pages;
    int b2 = b + skip;
    while (true) {
      if (x2 >= plan.pages) {
        x2 -= plan.pages;
        ++b2;
      }
      if (b2 >= a.batch) break;
      const int st2 = a.start[b2];
      const int64_t lp2 = first_page(plan, st2) + x2;
      int lo, hi;
      page_tokens(lp2, st2, a.seq_len, bs, lo, hi);
      if (lp2 >= 0 && lp2 < a.max_blocks && lo < hi && (!a.lens || lo < a.lens[b2]))
        later |= a.tables[static_cast<int64_t>(b2) * a.max_blocks + lp2] == page;
      x2 += on_x;
      b2 += on;
    }
  }
  const bool write = !__syncthreads_or(later) && page >= 0;

  const int items = 2 * a.n_head_kv + (a.q ? a.n_head : 0);
  const int log2_vecs = a.log2_dim - 3;  // loads of a row
  const int chunk = min(n, kAngleFloats >> a.log2_dim);
  const int64_t row_elems = static_cast<int64_t>(a.n_head_kv) << a.log2_dim;
  bool have_angles = false;

  for (int i0 = blockIdx.y * kWaves; i0 < items; i0 += gridDim.y * kWaves) {
    const int item = i0 + wave;
    const bool active = item < items;
    const int kind = item < a.n_head_kv ? 0 : item < 2 * a.n_head_kv ? 1 : 2;  // k, v, q
    const int head = kind == 0 ? item : kind == 1 ? item - a.n_head_kv : item - 2 * a.n_head_kv;
    const bool turn = a.rope && kind != 1;
    const int rows = !active ? 0 : kind == 2 ? n : write ? n_kv : 0;
    const int64_t stride = kind == 0 ? a.k_stride : kind == 1 ? a.v_stride : a.q_stride;
    const T* src = static_cast<const T*>(kind == 0 ? a.k : kind == 1 ? a.v : a.q) +
                   (static_cast<int64_t>(b) * a.seq_len + s0) * stride + (static_cast<int64_t>(head) << a.log2_dim);
    float amax = 0.f, inv = 0.f;
    Vec<T> raw[kBatch];

    // Two passes over the rows of a K or V item with codes (maximum, then
    // codes), one otherwise.
    for (int pass = C ? 0 : 1; pass < 2; ++pass) {
      for (int c0 = 0; c0 < n; c0 += chunk) {
        const int c1 = min(c0 + chunk, n);
        const int vecs = max(min(c1, rows) - c0, 0) << log2_vecs;
        const bool once = C && rows <= chunk && vecs <= kBatch * kWave;  // raw holds the rows through both passes
        // A lane's load u of a batch from e0 on; lanes behind the last load take it too.
        auto load = [&](int e0) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int e = min(e0 + u * kWave + lane, vecs - 1);
            raw[u] = *reinterpret_cast<const Vec<T>*>(src + (c0 + (e >> log2_vecs)) * stride +
                                                      ((e & ((1 << log2_vecs) - 1)) << 3));
          }
        };
        auto work = [&](int e0) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int e = min(e0 + u * kWave + lane, vecs - 1);
            const int row = c0 + (e >> log2_vecs), col = (e & ((1 << log2_vecs) - 1)) << 3;
            float v[kVec];
            raw[u].get(v);
            if (turn) {
              const float2* cs = angles + 4 * e;  // row e >> log2_vecs, pairs from 4 * (e's load of the row): 4 e in all
#pragma unroll
              for (int p = 0; p < 4; ++p) rope_apply(v[2 * p], v[2 * p + 1], cs[p], v[2 * p], v[2 * p + 1]);
            }
            if (pass == 0) {
#pragma unroll
              for (int k = 0; k < kVec; ++k) {
                const float m = fabsf(v[k]);
                amax = fmaxf(amax, m < INFINITY ? m : 0.f);
              }
            } else if (kind == 2) {
              store8(static_cast<T*>(a.q_out) + (static_cast<int64_t>(b) * a.seq_len + s0 + row) * a.q_out_stride +
                         (static_cast<int64_t>(head) << a.log2_dim) + col,
                     v);
            } else {
              const int64_t at = (page * bs + r0 + row) * row_elems + (static_cast<int64_t>(head) << a.log2_dim) + col;
              void* pool = kind == 0 ? a.k_cache : a.v_cache;
              if constexpr (C)
                *reinterpret_cast<u32x2_t*>(static_cast<f8_t*>(pool) + at) = codes8(v, inv);
              else
                store8(static_cast<T*>(pool) + at, v);
            }
            __builtin_amdgcn_sched_barrier(0);  // four waves a SIMD: one load's values at a time (37.6 us against 42.4)
          }
        };
        if (vecs > 0 && !(once ? pass == 1 : pass == 0 && kind == 2)) load(0);  // before the angles, which take as long
        if (a.rope && (!have_angles || chunk < n)) {  // block-uniform
          if (have_angles) __syncthreads();
          // A thread keeps one pair and steps through rows.  In 64 bits: one
          // sine and cosine a pair for the chunk's first row and one for a
          // row's step, and complex products for the rest.
          const int log2_pairs = a.log2_dim - 1, i = tid & ((1 << log2_pairs) - 1), r = tid >> log2_pairs;
          if (r < 2) {
            const double freq = a.freq_scale * exp2(-static_cast<double>(2 * i) / D * a.log2_base);
            double sn, cs;
            sincos((r ? 1. : static_cast<double>(static_cast<int64_t>(start) + s0 + c0)) * freq, &sn, &cs);
            turns[r][i] = double2{cs, sn};
          }
          __syncthreads();
          double2 z = turns[1][i], w = turns[0][i];
          for (int bit = 1; bit < kThreads >> log2_pairs; bit *= 2) {
            if (r & bit) w = cmul(w, z);
            z = cmul(z, z);
          }
          for (int row = r; row < c1 - c0; row += kThreads >> log2_pairs) {
            angles[(row << log2_pairs) + i] = float2{static_cast<float>(w.x), static_cast<float>(w.y)};
            w = cmul(w, z);
          }
          have_angles = true;
          __syncthreads();
        }
        if (pass == 0 && kind == 2) continue;
        for (int e0 = 0; e0 < vecs; e0 += kBatch * kWave) {
          if (e0 > 0) load(e0);
          work(e0);
        }
      }
      if constexpr (C) {
        if (pass == 0 && kind != 2 && rows > 0) {  // wave-uniform
          amax = wave_max(amax);
          float scale = amax > 0.f ? pow2_scale(amax, &inv) : 0x1p-126f;
          float* at = (kind == 0 ? a.k_scales : a.v_scales) + page * a.n_head_kv + head;
          if (r0 > 0) {
            const float old = *at;
            if (scale > old) {
              const float f = old / scale;
              f8_t* pool = static_cast<f8_t*>(kind == 0 ? a.k_cache : a.v_cache) + page * bs * row_elems +
                           (static_cast<int64_t>(head) << a.log2_dim);
              for (int64_t e = lane; e < static_cast<int64_t>(r0) << log2_vecs; e += kWave) {
                u32x2_t* p = reinterpret_cast<u32x2_t*>(pool + (e >> log2_vecs) * row_elems +
                                                        ((e & ((1 << log2_vecs) - 1)) << 3));
                float y[kVec];
                values8(*p, y);
                *p = codes8(y, f);
              }
            } else {
              scale = old;
            }
          }
          inv = 1.f / scale;
          if (lane == 0) *at = scale;
        }
      }
    }
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, int act, bool codes, hipStream_t s) {
  if (a.batch == 0 || a.seq_len == 0) return hipSuccess;
  // pages that seq_len tokens from any start can touch
  const int64_t pages = (static_cast<int64_t>(a.seq_len) + a.block_size - 2) / a.block_size + 1;
  const Plan plan{static_cast<int>(pages), Div::by(static_cast<uint32_t>(pages)),
                  Div::by(static_cast<uint32_t>(a.block_size))};
  if (pages > UINT32_MAX / kThreads) return hipErrorInvalidValue;  // a grid counts its threads in 32 bits
  const int items = 2 * a.n_head_kv + (a.q ? a.n_head : 0);
  const int groups = (items + kWaves - 1) / kWaves;
  const int rows = min(min(a.block_size, a.seq_len), kAngleFloats >> a.log2_dim);
  const size_t lds = a.rope ? (static_cast<size_t>(rows) << a.log2_dim) * sizeof(float) : 0;
    // About 1024 blocks, each with as many rounds of items: they share the
  // page's angles and the search for later appends (32/8 heads x 128, for 1024
  // blocks, 2048 and one for each group, in us: 4 x 2048 tokens to pages of 32
  // 37.6, 39.6, 41.5; 4 x 509 to bf16 pages of 16 12.3, 13.5, 13.5).
  const int64_t pages_all = pages * a.batch, want = (1024 + pages_all - 1) / pages_all;
  const int rounds = want < groups ? static_cast<int>((groups + want - 1) / want) : 1;
  const int y = (groups + rounds - 1) / rounds;
  const dim3 grid(static_cast<unsigned>(pages), y, a.batch);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), lds, s, a, plan); };
  // Loads of a lane in flight: as many as the rows of a page give it, so that
  // K and V are read once and a page does not take one load's latency after
  // another; no more, since each is computed (61 single tokens 7.1 us with 1,
  // 10.1 with 4, 12.5 with 8; pages of 16 rows 12.0 with 4, 14.7 with 8; pages
  // of 32 37.6 with 8, 45.5 with 4).
  const int loads = ((rows << (a.log2_dim - 3)) + kWave - 1) / kWave;
  if (act == DT_F32 && codes)
    launch(loads <= 1 ? kv_append_kernel<float, true, 1> : kv_append_kernel<float, true, 4>);
  else if (act == DT_F32)
    launch(loads <= 1 ? kv_append_kernel<float, false, 1> : kv_append_kernel<float, false, 4>);
  else if (codes)
    launch(loads <= 1   ? kv_append_kernel<bf16_t, true, 1>
           : loads <= 4 ? kv_append_kernel<bf16_t, true, 4>
                        : kv_append_kernel<bf16_t, true, 8>);
  else
    launch(loads <= 1   ? kv_append_kernel<bf16_t, false, 1>
           : loads <= 4 ? kv_append_kernel<bf16_t, false, 4>
                        : kv_append_kernel<bf16_t, false, 8>);
  return hipGetLastError();
}

}  // namespace fmoe
