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

// RoPE + append.  A CTA takes a few token rows (and, when there are few, a share of each row's work): the cosines and
// sines of their rotary pairs into shared memory, then the rows in pieces of 16 bytes, a rotary piece together with the
// one half the rotary dims away.  Every value is read once and written once: 2048 rows of 64 + 4 heads of 192 are 111 MB
// and take 32 us (3.5 TB/s), 16000 of 64 + 8 heads 198 us (4.4 TB/s); what is left is the loads in flight that four CTAs
// of 64 registers a thread hold on an SM (more threads of fewer registers, or fewer pieces each, were slower).
//
// The angle pos * theta^(-2i/rot), its reduction to [-pi, pi], sine and cosine are float64.  The rotation is float32, with
// the cosine (and sine) as a sum of its first 16 bits, whose product with a bf16 value is exact, and the rest: then even
// x1 cos - x2 sin that almost cancels is off by no more than 2^-24 of itself and 2^-40 (|x1| + |x2|), and has the bits of
// the one-sequence kernel's float64 rotation on all but one value in 10^5, without converting every value to float64.
constexpr int kRopeThreads = 256;
constexpr int kRopeRows = 4;

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
// Two rotary pairs: x1 and x2 become the rotated values.
__device__ __forceinline__ void rotate2(uint32_t& x1, uint32_t& x2, const float4* t) {
  const float a1 = bf16_to_f32(x1 & 0xFFFFu), a2 = bf16_to_f32(x2 & 0xFFFFu);
  const float b1 = bf16_to_f32(x1 >> 16), b2 = bf16_to_f32(x2 >> 16);
  const float4 ta = t[0], tb = t[1];
  x1 = pack_bf16x2(cos_part(a1, a2, ta), cos_part(b1, b2, tb));
  x2 = pack_bf16x2(sin_part(a1, a2, ta), sin_part(b1, b2, tb));
}
__device__ __forceinline__ uint32_t scaled(uint32_t w, float s) {
  return pack_bf16x2(bf16_to_f32(w & 0xFFFFu) * s, bf16_to_f32(w >> 16) * s);
}

// VEC: the rotary dims are a multiple of 16, so that a row is whole 16-byte pieces; otherwise value by value.
template <bool VEC>
__global__ void __launch_bounds__(kRopeThreads, 4) paged_rope_kernel(PagedRopeParams p) {
  __shared__ float4 cs[kRopeRows * 128];
  __shared__ double freq[128];
  const int half = p.rot / 2, tid = threadIdx.x;
  const int t0 = blockIdx.x * p.rows, nt = min(p.rows, p.T - t0);
  // the frequencies need no input: before the wait for the kernels before this one
  if (tid < half) freq[tid] = exp(-(double)(2 * tid) / (double)p.rot * p.log_base);
  __syncthreads();
  pdl_wait();  // the projection rows and the plan come from preceding kernels (programmatic dependent launch)
  pdl_launch_dependents();
  for (int i = tid; i < nt * half; i += kRopeThreads) {
    const double a = (double)p.positions[t0 + i / half] * freq[i % half];
    const double turns = rint(a * 0.15915494309189535);                                             // 1 / 2 pi
    const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, a));  // 2 pi in two parts
    double sn, cn;
    sincos(r, &sn, &cn);
    const float c0 = __uint_as_float(__float_as_uint((float)cn) & 0xFFFFFF00u);
    const float s0 = __uint_as_float(__float_as_uint((float)sn) & 0xFFFFFF00u);
    cs[i] = make_float4(c0, s0, (float)(cn - (double)c0), (float)(sn - (double)s0));
  }
  __syncthreads();
  const int heads = p.nq + p.nkv, page_mask = (1 << p.page_shift) - 1;
  const size_t rowlen = (size_t)heads * p.dqk + (size_t)p.nkv * p.dv;
  // pieces of a row: the heads' rotary pairs of pieces, their other pieces, the value rows': one after the other, so that
  // a warp has one kind to do (with each head's together, every warp ran the rotation for a fifth of its lanes)
  const int rp = VEC ? p.rot / 16 : half, hp = (p.dqk - p.rot) / (VEC ? 8 : 1), vp = p.dv / (VEC ? 8 : 1);
  const int per_row = heads * (rp + hp) + p.nkv * vp;
  const int share = (per_row + gridDim.y - 1) / gridDim.y;
  const int first = blockIdx.y * share, last = min(per_row, first + share);
  for (int tt = 0; tt < nt; ++tt) {
    const int t = t0 + tt, slot = p.slots[t];
    if (slot < 0) continue;
    const int page = slot >> p.page_shift, at = slot & page_mask;
    const bool store = page < p.num_pages;
    if (!store && tid == 0) set_status(p.status, MIMO_ERANGE);
    const uint16_t* row = p.qkv + (size_t)t * rowlen;
    const float4* c = cs + tt * half;
    // where the head or value row of piece i comes from and goes to (null: nowhere), which piece of it it is (a rotary
    // pair's first), and its kind
    enum { kRotary, kCopy, kValue };
    auto piece = [&](int i, const uint16_t*& src, uint16_t*& dst, int& k) -> int {
      int kind = kRotary, n = rp;
      if (i >= heads * rp) i -= heads * rp, kind = kCopy, n = hp;
      if (kind == kCopy && i >= heads * hp) i -= heads * hp, kind = kValue, n = vp;
      const int hd = i / n;
      k = i - hd * n;
      if (kind == kValue) {
        src = row + (size_t)heads * p.dqk + (size_t)hd * p.dv;
        dst = store ? p.v + ((((size_t)page * p.nkv + hd) << p.page_shift) + at) * p.dv : nullptr;
      } else {
        if (kind == kCopy) k += 2 * rp;
        src = row + (size_t)hd * p.dqk;
        dst = hd < p.nq ? p.q + ((size_t)t * p.nq + hd) * p.dqk
              : store   ? p.k + ((((size_t)page * p.nkv + (hd - p.nq)) << p.page_shift) + at) * p.dqk
                        : nullptr;
      }
      return kind;
    };
    if constexpr (VEC) {
      constexpr int U = 4;  // pieces in flight a thread
      for (int i0 = first + tid; i0 < last; i0 += U * kRopeThreads) {
        uint4 a[U], b[U];
        uint16_t* dst[U];
        int k[U], kind[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * kRopeThreads;
          const uint16_t* src;
          dst[u] = nullptr;
          if (i < last) kind[u] = piece(i, src, dst[u], k[u]);
          if (dst[u] == nullptr) continue;
          a[u] = __ldg(reinterpret_cast<const uint4*>(src) + k[u]);
          if (kind[u] == kRotary) b[u] = __ldg(reinterpret_cast<const uint4*>(src) + k[u] + rp);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (dst[u] == nullptr) continue;
          uint4* d4 = reinterpret_cast<uint4*>(dst[u]) + k[u];
          uint4 w = a[u];
          if (kind[u] == kRotary) {
            uint4 z = b[u];
            const float4* e = c + k[u] * 8;
            rotate2(w.x, z.x, e), rotate2(w.y, z.y, e + 2), rotate2(w.z, z.z, e + 4), rotate2(w.w, z.w, e + 6);
            d4[rp] = z;
          } else if (kind[u] == kValue && p.has_vscale) {
            w = make_uint4(scaled(w.x, p.v_scale), scaled(w.y, p.v_scale), scaled(w.z, p.v_scale),
                           scaled(w.w, p.v_scale));
          }
          *d4 = w;
        }
      }
    } else {
      for (int i = first + tid; i < last; i += kRopeThreads) {
        const uint16_t* src;
        uint16_t* dst;
        int k;
        const int kind = piece(i, src, dst, k);
        if (dst == nullptr) continue;
        if (kind == kRotary) {
          const float x1 = bf16_to_f32(src[k]), x2 = bf16_to_f32(src[k + half]);
          dst[k] = (uint16_t)f32_to_bf16(cos_part(x1, x2, c[k]));
          dst[k + half] = (uint16_t)f32_to_bf16(sin_part(x1, x2, c[k]));
        } else {
          dst[k] = kind == kValue && p.has_vscale ? (uint16_t)f32_to_bf16(bf16_to_f32(src[k]) * p.v_scale) : src[k];
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_page_plan(const PagePlanParams& p, cudaStream_t st) {
  // a row a thread: the searches and the table entry are latency, the scan that every CTA repeats is small beside them
  const int blocks = std::max(1, std::min(148, (p.tokens + kPlanThreads - 1) / kPlanThreads));
  return launch_k(page_plan_kernel, dim3(blocks), dim3(kPlanThreads), (size_t)(2 * p.R + 2) * 4, st, p);
}

cudaError_t launch_page_release(const PageReleaseParams& p, cudaStream_t st) {
  return launch_k(page_release_kernel, dim3(1), dim3(kPlanThreads), (size_t)(p.R + 1) * 4, st, p);
}

cudaError_t launch_paged_rope(PagedRopeParams& p, cudaStream_t st) {
  const bool vec = p.rot % 16 == 0;
  const int per_row = (p.nq + p.nkv) * (vec ? (p.dqk - p.rot / 2) / 8 : p.dqk - p.rot / 2) +
                      p.nkv * (vec ? p.dv / 8 : p.dv);
  // four rows a CTA once that gives every SM one (2048 rows: 32.1 us against 33.5 with one row a CTA, 16000: 198 against
  // 217), else one, and a share of it: down to one piece a thread (8 rows: 3.0 us)
  p.rows = p.T >= kRopeRows * 148 ? kRopeRows : 1;
  const int ctas = (p.T + p.rows - 1) / p.rows, most = (per_row + kRopeThreads - 1) / kRopeThreads;
  const int shares = std::max(1, std::min(most, 4 * 148 / ctas));
  return launch_k(vec ? paged_rope_kernel<true> : paged_rope_kernel<false>, dim3(ctas, shares), dim3(kRopeThreads), 0,
                  st, p);
}

}  // namespace mimo
