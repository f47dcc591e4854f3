// Attention of a step's new tokens over a paged KV cache (include/mimo_moe_paged.h).
#include "common.cuh"
#include "kernels.h"

namespace mimo {

namespace {

// One CTA per (token row, query head): four warps take the visible keys in turn, each with its own running maximum,
// sum and output in float32; the four are joined at the end with the sink.
template <int DQK, int DV>
__global__ void __launch_bounds__(128) paged_attn_kernel(PagedAttnParams p) {
  constexpr int QL = DQK / 32, VL = DV / 32;
  __shared__ float sm_m[4], sm_l[4], sm_o[4][DV];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, h = blockIdx.y, hk = h / (p.nq / p.nkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.cu_q[p.R] > p.T && threadIdx.x == 0) set_status(p.status, MIMO_ERANGE);
  if (t >= p.cu_q[p.R]) return;
  int lo = 0, hi = p.R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_q[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int r = lo, row0 = p.cu_q[r], n = p.cu_q[r + 1] - row0, len = p.seq_lens[r];
  if (row0 < 0 || n < 1 || t < row0 || t >= row0 + n || len < n || row0 + n > p.T ||
      (long long)len > ((long long)p.width << p.page_shift)) {
    if (threadIdx.x == 0) set_status(p.status, MIMO_ERANGE);
    return;
  }
  const int pos = len - n + (t - row0);
  const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
  const int keep = min(p.keep, first), seen = keep + pos - first + 1;
  float q[QL], o[VL];
#pragma unroll
  for (int i = 0; i < QL; ++i) q[i] = bf16_to_f32(p.q[((size_t)t * p.nq + h) * DQK + lane + 32 * i]) * p.scale_log2;
#pragma unroll
  for (int i = 0; i < VL; ++i) o[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int s = warp; s < seen; s += 4) {
    const int j = s < keep ? s : first + (s - keep);
    const int page = p.table[(size_t)r * p.width + (j >> p.page_shift)];
    const bool ok = (unsigned)page < (unsigned)p.num_pages;
    if (!ok && lane == 0) set_status(p.status, MIMO_ERANGE);
    const size_t at = (((size_t)(ok ? page : 0) * p.nkv + hk) << p.page_shift) + (j & ((1 << p.page_shift) - 1));
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < QL; ++i) dot = fmaf(q[i], ok ? bf16_to_f32(p.k[at * DQK + lane + 32 * i]) : 0.f, dot);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, x);
    const float mn = fmaxf(m, dot), a = exp2f(m - mn), w = exp2f(dot - mn);
    l = l * a + w;
#pragma unroll
    for (int i = 0; i < VL; ++i) o[i] = o[i] * a + w * (ok ? bf16_to_f32(p.v[at * DV + lane + 32 * i]) : 0.f);
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < VL; ++i) sm_o[warp][lane + 32 * i] = o[i];
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
  __syncthreads();
  float M = p.sinks ? p.sinks[h] * 1.4426950408889634f : -INFINITY;
  float L = 0.f;
  const float sink = M;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w]);
  if (p.sinks) L = exp2f(sink - M);
  for (int w = 0; w < 4; ++w) L += sm_l[w] * exp2f(sm_m[w] - M);
  for (int d = threadIdx.x; d < DV; d += 128) {
    float a = 0.f;
    for (int w = 0; w < 4; ++w) a += sm_o[w][d] * exp2f(sm_m[w] - M);
    p.out[((size_t)t * p.nq + h) * DV + d] = (uint16_t)f32_to_bf16(a / L);
  }
}

}  // namespace

cudaError_t launch_paged_attention(const PagedAttnParams& p, cudaStream_t st) {
  const dim3 grid(p.T, p.nq);
  if (p.dqk == 192) return launch_k(paged_attn_kernel<192, 128>, grid, dim3(128), 0, st, p);
  if (p.dqk == 128) return launch_k(paged_attn_kernel<128, 128>, grid, dim3(128), 0, st, p);
  return launch_k(paged_attn_kernel<64, 64>, grid, dim3(128), 0, st, p);
}

}  // namespace mimo
