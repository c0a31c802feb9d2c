// Attention of a sequence's new tokens over a paged cache of e4m3 codes with
// one scale for each (page, K/V head):
//   score_j = (q . K_j) SK[page(j)] * scale,  out = sum_j softmax(score)_j SV[page(j)] V_j
// over the positions j below the context's length and, causal, up to the
// query's own.  Table entries outside the pool are rows of zeros, as in
// kvcache_gather; a query that attends nothing gives zeros.
#include "common.h"
#include "launch.h"

namespace fmoe {
namespace {

constexpr int kTile = 256;  // positions per step

// One block per (query head, new token, sequence): scores of kTile positions,
// running maximum and sum, values by dimension.
__global__ __launch_bounds__(kTile) void paged_attn_kernel(PagedAttnArgs a) {
  __shared__ float q[128], p[kTile], vs[kTile], red[8];
  __shared__ int rows[kTile];
  const int h = blockIdx.x % a.n_head, s = blockIdx.x / a.n_head, b = blockIdx.y, tid = threadIdx.x, D = a.head_dim;
  const int G = a.n_head / a.n_head_kv, kvh = h / G;
  const int len = a.lens ? min(max(a.lens[b], 0), a.seq_len) : a.seq_len;
  const int64_t ctx = static_cast<int64_t>(max(a.ctx_lens[b], 0)) + a.ctx_add;
  const int64_t pos = ctx - len + s;
  int64_t end = min(ctx, static_cast<int64_t>(a.max_ctx));
  if (a.causal) end = min(end, pos + 1);
  if (s >= len) end = 0;
  const int64_t at = (static_cast<int64_t>(b) * a.seq_len + s);
  if (tid < D)
    q[tid] = a.scale * (a.q_dtype == DT_F32 ? static_cast<const float*>(a.q)[at * a.q_stride + h * D + tid]
                                            : bf16_to_f32(static_cast<const bf16_t*>(a.q)[at * a.q_stride + h * D + tid]));
  __syncthreads();
  const int64_t zeros = s < len ? max(static_cast<int64_t>(a.zero_to) - min(ctx, static_cast<int64_t>(a.max_ctx)), int64_t{0}) : 0;
  float m = zeros > 0 ? 0.f : -INFINITY, l = static_cast<float>(zeros), o = 0.f;
  for (int64_t j0 = 0; j0 < end; j0 += kTile) {
    const int64_t j = j0 + tid;
    float sc = -INFINITY;
    rows[tid] = -1;
    if (j < end) {
      const int64_t lb = j / a.block_size;
      const int pb = lb < a.max_blocks ? a.tables[static_cast<int64_t>(b) * a.max_blocks + lb] : -1;
      sc = 0.f;
      if (pb >= 0 && pb < a.n_blocks) {
        const int row = pb * a.block_size + static_cast<int>(j - lb * a.block_size);
        rows[tid] = row;
        vs[tid] = a.v_scales[static_cast<int64_t>(pb) * a.n_head_kv + kvh];
        const uint8_t* kr = a.k_pool + (static_cast<int64_t>(row) * a.n_head_kv + kvh) * D;
        for (int d = 0; d < D; ++d) sc = fmaf(q[d], e4m3fn_to_f32(kr[d]), sc);
        sc *= a.k_scales[static_cast<int64_t>(pb) * a.n_head_kv + kvh];
      }
    }
    float mx = wave_max(sc);
    if (tid % kWave == 0) red[tid / kWave] = mx;
    __syncthreads();
    mx = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float base = mx == -INFINITY ? 0.f : mx, f = expf(m - base);
    m = mx;
    const float w = j < end ? expf(sc - base) : 0.f;
    p[tid] = w;
    const float sum = wave_sum(w);
    if (tid % kWave == 0) red[4 + tid / kWave] = sum;
    __syncthreads();
    l = l * f + red[4] + red[5] + red[6] + red[7];
    o *= f;
    if (tid < D) {
      for (int t = 0; t < kTile && j0 + t < end; ++t)
        if (rows[t] >= 0)
          o = fmaf(p[t] * vs[t],
                   e4m3fn_to_f32(a.v_pool[(static_cast<int64_t>(rows[t]) * a.n_head_kv + kvh) * D + tid]), o);
    }
    __syncthreads();
  }
  if (tid < D) {
    const float r = l == 0.f ? 0.f : o / l;
    const int64_t i = (at * a.n_head + h) * D + tid;
    if (a.out_dtype == DT_F32)
      static_cast<float*>(a.out)[i] = r;
    else
      static_cast<bf16_t*>(a.out)[i] = f32_to_bf16(r);
  }
}

}  // namespace

bool paged_attn_supported(int head_dim) {
  return head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128;
}

size_t paged_attn_workspace_floats(int, int, int, int, int, int, int) { return 0; }

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t s) {
  if (a.batch == 0 || a.seq_len == 0) return hipSuccess;
  hipLaunchKernelGGL(paged_attn_kernel, dim3(a.n_head * a.seq_len, a.batch), dim3(kTile), 0, s, a);
  return hipGetLastError();
}

}  // namespace fmoe
