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
// number comes from the free list itself, so no CTA waits for another's table entries.  Its bytes are nothing; a launch
// and a chain of dependent loads are what it takes: 3.1 us for 8 requests, 4.1 for 203, 5.1 for 1024 with 98000 rows.
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

// RoPE + append.  Every value is read once and written once, so memory is what bounds it: a row goes through shared
// memory in bulk copies where it fits there (paged_rope_rows_kernel), else through registers (paged_rope_kernel).
//
// The angle pos * theta^(-2i/rot), its reduction to [-pi, pi], sine and cosine are float64.  The rotation is float32, with
// the cosine (and sine) as a sum of its first 16 bits, whose product with a bf16 value is exact, and the rest: then even
// x1 cos - x2 sin that almost cancels is off by no more than 2^-24 of itself and 2^-40 (|x1| + |x2|), and has the bits of
// the one-sequence kernel's float64 rotation on all but one value in 10^5, without converting every value to float64.
constexpr int kRopeThreads = 256;

// Two float32 values rounded to nearest-even bf16 in one conversion: lo in bits 0-15, hi in bits 16-31.
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float cos_part(float x1, float x2, float4 t) {  // x1 cos - x2 sin; t: first parts, rests
  return fmaf(x1, t.x, -(x2 * t.y)) + fmaf(x1, t.z, -(x2 * t.w));
}
__device__ __forceinline__ float sin_part(float x1, float x2, float4 t) {  // x1 sin + x2 cos
  return fmaf(x1, t.y, x2 * t.x) + fmaf(x1, t.w, x2 * t.z);
}
// The cosine and sine of an angle: first parts, rests.
__device__ __forceinline__ float4 rotary(double a) {
  const double turns = rint(a * 0.15915494309189535);                                         // 1 / 2 pi
  const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, a));  // 2 pi in two parts
  double sn, cn;
  sincos(r, &sn, &cn);
  const float c0 = __uint_as_float(__float_as_uint((float)cn) & 0xFFFFFF00u);
  const float s0 = __uint_as_float(__float_as_uint((float)sn) & 0xFFFFFF00u);
  return make_float4(c0, s0, (float)(cn - (double)c0), (float)(sn - (double)s0));
}
// Two rotary pairs: x1 and x2 become the rotated values.
__device__ __forceinline__ void rotate2(uint32_t& x1, uint32_t& x2, float4 ta, float4 tb) {
  const float a1 = bf16_to_f32(x1 & 0xFFFFu), a2 = bf16_to_f32(x2 & 0xFFFFu);
  const float b1 = bf16_to_f32(x1 >> 16), b2 = bf16_to_f32(x2 >> 16);
  x1 = pack_bf16x2(cos_part(a1, a2, ta), cos_part(b1, b2, tb));
  x2 = pack_bf16x2(sin_part(a1, a2, ta), sin_part(b1, b2, tb));
}
__device__ __forceinline__ uint32_t scaled(uint32_t w, float s) {
  return pack_bf16x2(bf16_to_f32(w & 0xFFFFu) * s, bf16_to_f32(w >> 16) * s);
}

// Whole token rows through shared memory, in CTAs that each hold one: a row of projections comes in with one bulk copy,
// its rotary pairs and values are rotated and scaled in place while other CTAs' rows are on their way, and it goes out
// with one bulk copy for q (the row's q heads lie as they do in the input) and one for each kv head's k and v.  What is in
// flight costs no registers: six rows of 27 KB an SM.  2048 rows of 64 + 4 heads of 192 are 111 MB and take 21.8 us (5.1
// TB/s; 32 through registers), 16000 of them 153 us (5.7 TB/s; 198), 8 rows 2.6 us (2.7).
constexpr size_t kRowSmem = 232448;  // a CTA's most
constexpr int kRowHead = 128 * 16 + 128 * 8 + 128;  // cosines and sines, frequencies, the barrier

__device__ __forceinline__ void bulk_s2g(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) paged_rope_rows_kernel(PagedRopeParams p) {
  extern __shared__ __align__(128) uint8_t rows_smem[];
  float4* cs = reinterpret_cast<float4*>(rows_smem);  // [8][rot / 16]: pair 8 k + e of a head at e * (rot / 16) + k
  double* freq = reinterpret_cast<double*>(rows_smem + 128 * 16);
  uint64_t* bar = reinterpret_cast<uint64_t*>(rows_smem + 128 * 24);
  uint8_t* row = rows_smem + kRowHead;
  const int half = p.rot / 2, rp = p.rot / 16, tid = threadIdx.x;
  const int heads = p.nq + p.nkv, page_mask = (1 << p.page_shift) - 1;
  const uint32_t qk_bytes = (uint32_t)heads * p.dqk * 2, bytes = qk_bytes + (uint32_t)p.nkv * p.dv * 2;
  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_fence_init();
  }
  if (tid < half) freq[tid] = exp(-(double)(2 * tid) / (double)p.rot * p.log_base);
  __syncthreads();
  pdl_wait();  // the projection rows and the plan come from preceding kernels (programmatic dependent launch)
  pdl_launch_dependents();
  uint32_t phase = 0;
  int t = blockIdx.x, slot = -1, pos = 0;
  if (t < p.T) slot = p.slots[t], pos = p.positions[t];
  for (; t < p.T; t += gridDim.x) {
    const int my_slot = slot, my_pos = pos;
    if (t + (int)gridDim.x < p.T) slot = p.slots[t + gridDim.x], pos = p.positions[t + gridDim.x];
    if (my_slot < 0) continue;
    if (tid < 32) {
      asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");  // the row before has left
      __syncwarp();
      if (tid == 0) {
        mbar_arrive_expect_tx(bar, bytes);
        bulk_g2s(row, reinterpret_cast<const uint8_t*>(p.qkv) + (size_t)t * bytes, bytes, bar, l2_evict_first_policy());
      }
    }
    if (tid < half) {
      const double a = (double)my_pos * freq[tid];
      cs[(tid & 7) * rp + (tid >> 3)] = rotary(a);
    }
    const bool ok = __syncthreads_and(mbar_wait(bar, phase));
    phase ^= 1;
    if (!ok) {
      if (tid == 0) set_status(p.status, MIMO_ETIMEOUT);
      mbar_wait(bar, phase ^ 1);  // the copy may still be landing
      break;
    }
    for (int i = tid; i < heads * rp; i += THREADS) {
      const int hd = i / rp, k = i - hd * rp;
      uint4* a4 = reinterpret_cast<uint4*>(row + (uint32_t)hd * p.dqk * 2) + k;
      // heads may lie a multiple of all banks apart: every other one is read from its second piece on
      uint4 *f = a4 + (hd & 1 ? rp : 0), *g = a4 + (hd & 1 ? 0 : rp);
      const uint4 u = *f, w = *g;
      uint4 x = hd & 1 ? w : u, z = hd & 1 ? u : w;
      const float4* e = cs + k;
      rotate2(x.x, z.x, e[0], e[rp]), rotate2(x.y, z.y, e[2 * rp], e[3 * rp]);
      rotate2(x.z, z.z, e[4 * rp], e[5 * rp]), rotate2(x.w, z.w, e[6 * rp], e[7 * rp]);
      *f = hd & 1 ? z : x;
      *g = hd & 1 ? x : z;
    }
    if (p.has_vscale)
      for (int i = tid; i < p.nkv * p.dv / 8; i += THREADS) {
        uint4* w = reinterpret_cast<uint4*>(row + qk_bytes) + i;
        *w = make_uint4(scaled(w->x, p.v_scale), scaled(w->y, p.v_scale), scaled(w->z, p.v_scale),
                        scaled(w->w, p.v_scale));
      }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncthreads();
    if (tid < 32) {
      const int page = my_slot >> p.page_shift, at = my_slot & page_mask;
      const bool store = page < p.num_pages;
      if (tid == 0) {
        if (!store) set_status(p.status, MIMO_ERANGE);
        bulk_s2g(p.q + (size_t)t * p.nq * p.dqk, row, (uint32_t)p.nq * p.dqk * 2);
      }
      if (store)
        for (int h = tid; h < p.nkv; h += 32) {
          const size_t to = (((size_t)page * p.nkv + h) << p.page_shift) + at;
          bulk_s2g(p.k + to * p.dqk, row + (uint32_t)(p.nq + h) * p.dqk * 2, (uint32_t)p.dqk * 2);
          bulk_s2g(p.v + to * p.dv, row + qk_bytes + (uint32_t)h * p.dv * 2, (uint32_t)p.dv * 2);
        }
      asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
    }
  }
  // (in a loop of its own: a branch in the one above made 2048 rows 22.4 us instead of 21.7)
  if (p.clear != nullptr)
    for (t = blockIdx.x; t < p.T; t += gridDim.x)
      if (p.slots[t] < 0)
        for (int i = tid; i < p.clear_n; i += THREADS) p.clear[(size_t)t * p.clear_n + i] = make_uint4(0, 0, 0, 0);
  if (tid < 32) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
}

// What the other does not take: rotary dims that are no multiple of 16, and rows wider than shared memory.  A CTA takes a
// share of one row, value by value.
__global__ void __launch_bounds__(kRopeThreads) paged_rope_kernel(PagedRopeParams p) {
  __shared__ float4 cs[128];
  __shared__ double freq[128];
  const int half = p.rot / 2, tid = threadIdx.x, t = blockIdx.x;
  // the frequencies need no input: before the wait for the kernels before this one
  if (tid < half) freq[tid] = exp(-(double)(2 * tid) / (double)p.rot * p.log_base);
  __syncthreads();
  pdl_wait();  // the projection rows and the plan come from preceding kernels (programmatic dependent launch)
  pdl_launch_dependents();
  const int slot = p.slots[t];
  if (slot < 0) {
    if (p.clear != nullptr)
      for (int i = blockIdx.y * kRopeThreads + tid; i < p.clear_n; i += gridDim.y * kRopeThreads)
        p.clear[(size_t)t * p.clear_n + i] = make_uint4(0, 0, 0, 0);
    return;
  }
  if (tid < half) cs[tid] = rotary((double)p.positions[t] * freq[tid]);
  __syncthreads();
  const int page = slot >> p.page_shift, at = slot & ((1 << p.page_shift) - 1);
  const bool store = page < p.num_pages;
  if (!store && tid == 0) set_status(p.status, MIMO_ERANGE);
  const int heads = p.nq + p.nkv, qk = heads * (p.dqk - half), all = qk + p.nkv * p.dv;  // a rotary pair counts once
  const uint16_t* row = p.qkv + (size_t)t * ((size_t)heads * p.dqk + (size_t)p.nkv * p.dv);
  const int share = (all + gridDim.y - 1) / gridDim.y, last = min(all, (int)(blockIdx.y + 1) * share);
  for (int i = blockIdx.y * share + tid; i < last; i += kRopeThreads) {
    if (i < qk) {
      const int hd = i / (p.dqk - half), e = i - hd * (p.dqk - half);  // pairs 0 .. half - 1, then the other dims
      const uint16_t* src = row + (size_t)hd * p.dqk;
      uint16_t* dst = hd < p.nq ? p.q + ((size_t)t * p.nq + hd) * p.dqk
                      : store   ? p.k + ((((size_t)page * p.nkv + (hd - p.nq)) << p.page_shift) + at) * p.dqk
                                : nullptr;
      if (dst == nullptr) continue;
      if (e < half) {
        const float x1 = bf16_to_f32(src[e]), x2 = bf16_to_f32(src[e + half]);
        dst[e] = (uint16_t)f32_to_bf16(cos_part(x1, x2, cs[e]));
        dst[e + half] = (uint16_t)f32_to_bf16(sin_part(x1, x2, cs[e]));
      } else {
        dst[e + half] = src[e + half];
      }
    } else if (store) {
      const int hd = (i - qk) / p.dv, e = i - qk - hd * p.dv;
      const uint16_t x = row[(size_t)heads * p.dqk + (size_t)hd * p.dv + e];
      p.v[((((size_t)page * p.nkv + hd) << p.page_shift) + at) * p.dv + e] =
          p.has_vscale ? (uint16_t)f32_to_bf16(bf16_to_f32(x) * p.v_scale) : x;
    }
  }
}

}  // namespace

cudaError_t launch_page_plan(const PagePlanParams& p, int num_sms, cudaStream_t st) {
  // a row a thread: the searches and the table entry are latency, the scan that every CTA repeats is small beside them
  const int blocks = std::max(1, std::min(num_sms, (p.tokens + kPlanThreads - 1) / kPlanThreads));
  return launch_k(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), (size_t)(2 * p.R + 2) * 4, st, p);
}

cudaError_t launch_page_release(const PageReleaseParams& p, cudaStream_t st) {
  return launch_k(page_release_kernel, dim3(1), dim3(kPlanThreads), (size_t)(p.R + 1) * 4, st, p);
}

namespace {
template <int THREADS>
cudaError_t launch_rope_rows(const PagedRopeParams& p, size_t smem, int most, cudaStream_t st) {
  static bool attr_set[128] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 128 && !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_rope_rows_kernel<THREADS>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRowSmem);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const int rounds = (p.T + most - 1) / most;  // all CTAs have the same number of rows, or one less
  return launch_k(paged_rope_rows_kernel<THREADS>, dim3((p.T + rounds - 1) / rounds), dim3(THREADS), smem, st, p);
}
}  // namespace

cudaError_t launch_paged_rope(const PagedRopeParams& p, int num_sms, cudaStream_t st) {
  const size_t smem = kRowHead + ((size_t)(p.nq + p.nkv) * p.dqk + (size_t)p.nkv * p.dv) * 2;
  if (p.rot % 16 == 0 && smem <= kRowSmem) {
    const int fit = (int)std::min<size_t>(16, (228 * 1024) / (smem + 1024));  // CTAs an SM
    // A CTA of 128 threads keeps up with memory where several rows of an SM are worked on at once; alone, 384 threads are
    // through its row sooner (8 rows of 64 + 4 heads: 2.6 us against 2.9; 16000 of 32 + 8 heads of 128 with 256 threads:
    // 105 us against 79, as fewer CTAs fit).
    return p.T <= num_sms || fit < 3 ? launch_rope_rows<384>(p, smem, num_sms * fit, st)
                                     : launch_rope_rows<128>(p, smem, num_sms * fit, st);
  }
  // shares of a row down to a value a thread while there are fewer rows than four for each SM
  const int all = (p.nq + p.nkv) * (p.dqk - p.rot / 2) + p.nkv * p.dv;
  const int shares = std::max(1, std::min((all + kRopeThreads - 1) / kRopeThreads, 4 * num_sms / p.T));
  return launch_k(paged_rope_kernel, dim3(p.T, shares), dim3(kRopeThreads), 0, st, p);
}

}  // namespace mimo
