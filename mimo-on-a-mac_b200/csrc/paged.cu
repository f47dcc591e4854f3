// Serving many requests over a paged KV cache: the page plan of a step, the release of finished requests' pages, and
// RoPE + append at a position and slot per token (include/mimo_moe_paged.h).  The attention over the pages is in
// paged_attn.cu.
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace mimo {

namespace {

constexpr int kPlanThreads = 512;

// Exclusive block scan of two 64-bit values per thread (kPlanThreads threads): returns the totals.
__device__ __forceinline__ longlong2 block_scan2(longlong2 v, longlong2* excl, longlong2* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  longlong2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xFFFFFFFFu, x.x, o), b = __shfl_up_sync(0xFFFFFFFFu, x.y, o);
    if (lane >= o) x.x += a, x.y += b;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  longlong2 base = make_longlong2(0, 0), tot = make_longlong2(0, 0);
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const longlong2 s = sh[w];
    if (w < warp) base.x += s.x, base.y += s.y;
    tot.x += s.x, tot.y += s.y;
  }
  *excl = make_longlong2(base.x + x.x - v.x, base.y + x.y - v.y);
  __syncthreads();
  return tot;
}

// Largest r in [0, R) with cu[r] <= t (cu ascending, cu[0] = 0 <= t).
__device__ __forceinline__ int find_row(const int* cu, int R, int t) {
  int lo = 0, hi = R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Every CTA scans the requests' row counts and page needs (R <= 4096: a few values a thread), then takes its share of
// the new pages and of the token rows, each found by a binary search of the offsets in shared memory.  A new page's
// number comes from the free list itself, so no CTA waits for another's table entries.
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PagePlanParams p) {
  extern __shared__ int sm[];
  int* cu = sm;              // [R + 1] row offsets
  int* off = sm + p.R + 1;   // [R + 1] new pages before request r
  __shared__ longlong2 sh[kPlanThreads / 32];
  pdl_wait();  // the lengths come from the preceding kernel (programmatic dependent launch)
  pdl_launch_dependents();
  const int tid = threadIdx.x, shift = p.page_shift, page = 1 << shift;
  const long long longest = (long long)p.width << shift;
  const int nfree = *p.n_free;
  bool bad = nfree < 0 || nfree > p.num_pages;
  const int per = (p.R + kPlanThreads - 1) / kPlanThreads, r0 = min(tid * per, p.R), r1 = min(r0 + per, p.R);
  longlong2 mine = make_longlong2(0, 0);
  for (int r = r0; r < r1; ++r) {
    const int len = p.lens[r], n = p.new_lens[r];
    if (len < 0 || n < 0 || (long long)len + n > longest) {
      bad = true;
      continue;
    }
    mine.x += n;
    mine.y += (((long long)len + n + page - 1) >> shift) - (((long long)len + page - 1) >> shift);
  }
  longlong2 ex;
  const longlong2 tot = block_scan2(mine, &ex, sh);
  bad = __syncthreads_or(bad || tot.x > p.tokens || tot.y > nfree);
  if (bad) {
    if (blockIdx.x == 0) {
      if (tid == 0) {
        set_status(p.status, MIMO_ERANGE);
        *p.n_free_out = nfree;
      }
      for (int r = tid; r <= p.R; r += kPlanThreads) p.cu_q[r] = 0;
      for (int r = tid; r < p.R; r += kPlanThreads) p.seq_lens[r] = p.lens[r];
    }
    for (int t = blockIdx.x * kPlanThreads + tid; t < p.tokens; t += gridDim.x * kPlanThreads)
      p.positions[t] = -1, p.slots[t] = -1;
    return;
  }
  int a = (int)ex.x, b = (int)ex.y;
  for (int r = r0; r < r1; ++r) {
    const int len = p.lens[r], n = p.new_lens[r];
    cu[r] = a, off[r] = b;
    a += n;
    b += (int)((((long long)len + n + page - 1) >> shift) - (((long long)len + page - 1) >> shift));
    if (blockIdx.x == 0) p.cu_q[r] = a - n, p.seq_lens[r] = len + n;
  }
  const int rows = (int)tot.x, fresh = (int)tot.y;
  if (tid == 0) {
    cu[p.R] = rows, off[p.R] = fresh;
    if (blockIdx.x == 0) p.cu_q[p.R] = rows, *p.n_free_out = nfree - fresh;
  }
  __syncthreads();
  const int first = blockIdx.x * kPlanThreads + tid, stride = gridDim.x * kPlanThreads;
  for (int k = first; k < fresh; k += stride) {
    const int r = find_row(off, p.R, k);
    const int old = (int)(((long long)p.lens[r] + page - 1) >> shift);
    const int pg = p.free_pages[nfree - 1 - k];
    if ((unsigned)pg >= (unsigned)p.num_pages) set_status(p.status, MIMO_ERANGE);
    p.table[(size_t)r * p.width + old + (k - off[r])] = pg;
  }
  for (int t = first; t < p.tokens; t += stride) {
    int pos = -1, slot = -1;
    if (t < rows) {
      const int r = find_row(cu, p.R, t);
      const int len = p.lens[r];
      pos = len + (t - cu[r]);
      const int j = pos >> shift, old = (int)(((long long)len + page - 1) >> shift);
      const int pg = j < old ? p.table[(size_t)r * p.width + j] : p.free_pages[nfree - 1 - (off[r] + j - old)];
      if ((unsigned)pg < (unsigned)p.num_pages)
        slot = (pg << shift) + (pos & (page - 1));
      else
        set_status(p.status, MIMO_ERANGE);
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// One CTA (it updates lens, the table and the free list in place): scan of the finished rows' page counts, a check of
// every page, then the move.
__global__ void __launch_bounds__(kPlanThreads) page_release_kernel(PageReleaseParams p) {
  extern __shared__ int sm[];
  int* off = sm;  // [R + 1] released pages before row r
  __shared__ longlong2 sh[kPlanThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, shift = p.page_shift, page = 1 << shift;
  const long long longest = (long long)p.width << shift;
  const int nfree = *p.n_free;
  bool bad = nfree < 0 || nfree > p.num_pages;
  const int per = (p.R + kPlanThreads - 1) / kPlanThreads, r0 = min(tid * per, p.R), r1 = min(r0 + per, p.R);
  longlong2 mine = make_longlong2(0, 0);
  for (int r = r0; r < r1; ++r) {
    if (!p.done[r]) continue;
    const int len = p.lens[r];
    if (len < 0 || len > longest) bad = true;
    else mine.x += ((long long)len + page - 1) >> shift;
  }
  longlong2 ex;
  const longlong2 tot = block_scan2(mine, &ex, sh);
  bad = __syncthreads_or(bad || nfree + tot.x > p.num_pages);
  if (!bad) {
    int a = (int)ex.x;
    for (int r = r0; r < r1; ++r) {
      off[r] = a;
      if (p.done[r]) a += (int)(((long long)p.lens[r] + page - 1) >> shift);
    }
    if (tid == 0) off[p.R] = (int)tot.x;
  }
  __syncthreads();
  const int n = (int)tot.x;
  if (!bad)
    for (int k = tid; k < n; k += kPlanThreads) {
      const int r = find_row(off, p.R, k);
      bad |= (unsigned)p.table[(size_t)r * p.width + (k - off[r])] >= (unsigned)p.num_pages;
    }
  bad = __syncthreads_or(bad);
  if (bad) {
    if (tid == 0) set_status(p.status, MIMO_ERANGE);
    return;
  }
  for (int k = tid; k < n; k += kPlanThreads) {
    const int r = find_row(off, p.R, k);
    int32_t* e = p.table + (size_t)r * p.width + (k - off[r]);
    p.free_pages[nfree + k] = *e;
    *e = -1;
  }
  for (int r = tid; r < p.R; r += kPlanThreads)
    if (p.done[r]) p.lens[r] = 0;
  if (tid == 0) *p.n_free = nfree + n;
}

// One CTA per token: the cos/sin of the token's rotary pairs once in float64, then a warp per head.
constexpr int kRopeThreads = 256;

__global__ void __launch_bounds__(kRopeThreads) paged_rope_kernel(PagedRopeParams p) {
  __shared__ double2 cs[128];
  pdl_wait();  // the projection rows and the plan come from preceding kernels (programmatic dependent launch)
  pdl_launch_dependents();
  const int t = blockIdx.x, slot = p.slots[t], pos = p.positions[t];
  if (slot < 0) return;
  const int half = p.rot / 2, heads = p.nq + p.nkv;
  const int page = slot >> p.page_shift, at = slot & ((1 << p.page_shift) - 1);
  const bool store = page < p.num_pages;
  if (!store && threadIdx.x == 0) set_status(p.status, MIMO_ERANGE);
  for (int i = threadIdx.x; i < half; i += kRopeThreads) {
    double s, c;
    sincos((double)pos * exp(-(double)(2 * i) / (double)p.rot * p.log_base), &s, &c);
    cs[i] = make_double2(c, s);
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint16_t* row = p.qkv + (size_t)t * ((size_t)p.nq * p.dqk + (size_t)p.nkv * (p.dqk + p.dv));
  for (int h = warp; h < heads + p.nkv; h += kRopeThreads / 32) {
    if (h >= heads) {  // a value row
      const int hk = h - heads;
      if (!store) continue;
      const uint16_t* src = row + (size_t)heads * p.dqk + (size_t)hk * p.dv;
      uint16_t* dst = p.v + (((size_t)page * p.nkv + hk << p.page_shift) + at) * p.dv;
      for (int i = lane; i < p.dv; i += 32)
        dst[i] = p.has_vscale ? (uint16_t)f32_to_bf16(bf16_to_f32(src[i]) * p.v_scale) : src[i];
      continue;
    }
    if (h >= p.nq && !store) continue;
    const uint16_t* src = row + (size_t)h * p.dqk;
    uint16_t* dst = h < p.nq ? p.q + ((size_t)t * p.nq + h) * p.dqk
                             : p.k + (((size_t)page * p.nkv + (h - p.nq) << p.page_shift) + at) * p.dqk;
    for (int i = lane; i < half; i += 32) {
      const double x1 = bf16_to_f32(src[i]), x2 = bf16_to_f32(src[i + half]);
      const double2 c = cs[i];
      dst[i] = (uint16_t)f32_to_bf16(__double2float_rn(x1 * c.x - x2 * c.y));
      dst[i + half] = (uint16_t)f32_to_bf16(__double2float_rn(x1 * c.y + x2 * c.x));
    }
    for (int i = p.rot + lane; i < p.dqk; i += 32) dst[i] = src[i];
  }
}

}  // namespace

cudaError_t launch_page_plan(const PagePlanParams& p, cudaStream_t st) {
  const int blocks = std::max(1, std::min(148, (p.tokens + 4 * kPlanThreads - 1) / (4 * kPlanThreads)));
  return launch_k(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), (size_t)(2 * p.R + 2) * 4, st, p);
}

cudaError_t launch_page_release(const PageReleaseParams& p, cudaStream_t st) {
  return launch_k(page_release_kernel, dim3(1), dim3(kPlanThreads), (size_t)(p.R + 1) * 4, st, p);
}

cudaError_t launch_paged_rope(const PagedRopeParams& p, cudaStream_t st) {
  return launch_k(paged_rope_kernel, dim3(p.T), dim3(kRopeThreads), 0, st, p);
}

}  // namespace mimo
