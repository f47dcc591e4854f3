// Attention of a step's new tokens over a paged KV cache (include/mimo_moe_paged.h) on the 5th-generation tensor
// cores: a plan of the step's work (one small launch, shared by all layers of a kind), the attention kernel (one
// persistent CTA per SM) and the merge of what was split.
//
// A work unit is one kv head of up to 2 * (128 / G) consecutive new tokens of one request, over the blocks of 128 key
// positions that its queries see: blocks 0 .. nkb - 1 hold the first tokens that stay visible, blocks lb .. the window
// (all, without one).  A tile is 128 query rows, the G = n_heads / n_kv_heads heads of 128 / G tokens, token-major, so
// that one K/V block serves the whole group.  A unit of more than one tile (a pair) works on two, A and B, over the same
// blocks.  A unit of one tile (a decoding request's) works on its even blocks as A and on its odd ones as B, and joins
// the two at its end.  Either way the two softmax groups and the MMAs take turns, so neither waits out the other.
//
// One CTA, 12 warps:
//   warps 0-3, 4-7   softmax of tile A and of tile B, one thread per query row (TMEM lane = row): the scores of S_j from
//                    TMEM into registers, mask, P_j = bf16(2^(s - reference)) back over S_j's own TMEM columns, where the
//                    P V product reads it as its A operand (it never passes through shared memory), the row sum from the
//                    float32 P.  The reference is a maximum of earlier scores, and the output in TMEM is rescaled only
//                    when the row's maximum has grown by more than 2^8;
//   warps 8, 11      TMA producers of Q and K, and of V: chunks of 64 dims x 128 positions (16 KB) through one ring of
//                    shared-memory slots, K_0 V_0 K_1 V_1 ...; a copy is 64 dims of a page that some query of the unit
//                    sees, so with pages of 16 tokens a block is 40 copies: hence two warps;
//   warp 9           MMA issuer: S = Q K^T and O += P V, alternating the tiles, so that one tile's products run while the
//                    other's softmax does: S_A S_B | PV_A S_A' | PV_B S_B' | ...  A tile's PV and its next S are issued
//                    in this order, so when that S is there, O holds PV and P is consumed;
//   warp 10          zeroes the V rows that no query of the unit sees: such slots may hold anything, and 0 * NaN is not 0.
// Every wait is bounded and sets MIMO_ETIMEOUT; the producers drain their copies and the issuer its MMAs before exit.
//
// What bounds it (B200, 64 heads of 192 / 128 over 4 kv heads): a prompt's chunk of 4096 tokens on 12288 takes 3.5 M
// cycles an SM, 58% of them with the tensor core at work, and 2.1 ms under the power cap (1.14 PFLOP/s; a form of 3.15 M
// cycles and more instructions took as long).  A tile's round of softmax (2000 cycles), P V and S (1420) and four
// hand-overs is 4100 cycles and more, in which the tensor core works 2 x 1280.  Without any exponential it is still 3770;
// two threads a row, two issuing warps, P in halves and a helper for the issuer's waits were all slower.  64 decoding
// requests (580 MB of K and V) take 107 us, 5.4 TB/s; 8 of them at 4096 tokens (84 MB) 23 us, of which 9 pass before the
// first product: the plan, the table, K and V come from HBM one after the other.
#include <cstring>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace mimo {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 384;
// setmaxnreg: 2 x 128 softmax threads x 200 + 128 x 104 = 64512 = 384 x 168, what the block is launched with
constexpr int kRegsSoftmax = 200, kRegsOther = 104;

// ------------------------------------------------------------------------------------------------------------ the plan
// There are two lists of work units: small ones (at most kSmallRows query rows) and others, each for a kernel of its own
// (see Shape).  A request of at most tok[kSmall] new tokens is a small unit; when there are no more rows than requests,
// all units are small (a request of more tokens is then several, each of which reads the cache: a chunk of 64 tokens on
// 16320 takes 175 us with a table of 64 requests or more, 70 with one of fewer).
constexpr int kSmall = 0, kLarge = 1, kSmallRows = 32;

struct Lists {
  int tok[2];      // new tokens of a unit at most; 0: the list has none
  bool all_small;
};
__host__ __device__ inline Lists lists_of(int T, int R, int G) {
  Lists l;
  l.tok[kSmall] = kSmallRows / G;
  l.all_small = l.tok[kSmall] > 0 && T <= R;
  l.tok[kLarge] = l.all_small ? 0 : 2 * (128 / G);
  return l;
}

// Tiles of a list at most: the sum of ceil(n_r / tok) over its requests.
__host__ __device__ inline int cap_tiles_of(const Lists& ls, int list, int T, int R) {
  return ls.tok[list] == 0 ? 0 : list == kSmall && !ls.all_small ? R : R + T / ls.tok[list];
}

// Layout of one list in the plan buffer (32-bit words from its start, every part 16-byte aligned).
struct PlanLayout {
  int cap_tiles, cap_segs;
  size_t head, merge, segs, tiles, nb, order, pre, words;
};

__host__ __device__ inline size_t up4(size_t x) { return (x + 3) & ~(size_t)3; }

__host__ __device__ inline PlanLayout plan_layout(int list, int T, int R, int G, int nkv, int n) {
  PlanLayout L;
  L.cap_tiles = cap_tiles_of(lists_of(T, R, G), list, T, R);
  L.cap_segs = L.cap_tiles * nkv + n;
  size_t at = 16;  // header: key, units, mode
  L.head = at, at += (size_t)12 * n;  // of each CTA: (its first segment's place, segments), the first segment itself
  L.merge = at, at += (size_t)8 * n;
  L.segs = at, at += (size_t)8 * L.cap_segs;
  L.tiles = at, at += (size_t)4 * L.cap_tiles;
  L.nb = at, at += up4(L.cap_tiles);
  L.order = at, at += up4(L.cap_tiles);
  L.pre = at, at += up4((size_t)2 * L.cap_tiles + 2);
  L.words = at;
  return L;
}
__host__ __device__ inline size_t list_start(int list, int T, int R, int G, int nkv, int n) {
  return list == kSmall ? 0 : plan_layout(kSmall, T, R, G, nkv, n).words;
}
// Rows of a list's largest unit: one part's rows in the workspace, and the workspace rows before the list's own.
__host__ __device__ inline int part_rows_of(int list, int T, int R, int G) {
  const int tok = lists_of(T, R, G).tok[list];
  return (tok < T ? tok : T) * G;
}
__host__ __device__ inline size_t part_start(int list, int T, int R, int G, int n) {
  return list == kSmall ? 0 : (size_t)2 * n * part_rows_of(kSmall, T, R, G);
}

// Key blocks of a unit whose queries are at qfirst .. qlast.
struct Blocks {
  int lo, keep, nkb, lb, n;
};
__device__ __forceinline__ Blocks blocks_of(int qfirst, int qlast, int window, int keep) {
  Blocks b;
  b.lo = window > 0 ? max(0, qfirst - window + 1) : 0;
  b.keep = min(keep, b.lo);
  b.lb = b.lo >> 7;
  b.nkb = min((b.keep + 127) >> 7, b.lb);
  b.n = b.nkb + (qlast >> 7) - b.lb + 1;
  return b;
}

// A unit of at most five blocks, as those of a short window, is never cut: the two or three blocks that this would save
// its CTA are what the merge and its launch cost, and without cuts no merge is launched (48 decoding requests in a window
// of 128: 19.2 us instead of 20.9).
__host__ __device__ inline bool whole_units(int tok, int window, int keep) {
  return window > 0 && ((long long)keep + 127) / 128 + ((long long)window + tok + 125) / 128 + 1 <= 5;
}

constexpr int kPlanThreads = 1024;
constexpr int kBuckets = 2048;
// A unit's block count as the sort by length and the CTAs' loads take it: itself below 1024 blocks, above that its first
// seven significant bits, so that units of one bucket count the same and their order in it, which atomics give, has no say
// in how the units are dealt.  (A table row of 2^31 positions is 2^24 blocks: bucket 1024 + 14 * 64.)
__device__ __forceinline__ int bucket_of(int nb) {
  return nb < 1024 ? nb : 1024 + (int)((__float_as_uint((float)nb) - __float_as_uint(1024.f)) >> 17);
}
__device__ __forceinline__ int sorted_as(int nb) {
  return nb < 1024 ? nb : (int)__uint_as_float(__float_as_uint((float)nb) & ~0x1FFFFu);
}
// What a unit costs besides its blocks (Q, the first scores, the epilogue), in blocks.
constexpr int kUnitCost = 2;

__device__ __forceinline__ long long block_scan(long long v, long long* excl, long long* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += a;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  long long base = 0, tot = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const long long s = sh[w];
    if (w < warp) base += s;
    tot += s;
  }
  *excl = base + x - v;
  __syncthreads();
  return tot;
}

// One CTA for each list.  Two ways to deal the units to the n CTAs: whole units, longest first, in a snake (no partial
// results), or the units' blocks one after another in n equal ranges (perfect balance; a unit cut by a range's end leaves
// partial results that the merge kernel joins).  The one whose longest CTA takes less is taken, in units of a key block,
// each unit counted as its blocks and kUnitCost more.  Its bytes are nothing; the scans, the sort and the passes over the
// units, one after the other, are what it takes: 10.4 to 11.7 us for up to 64 requests, 15.2 for 200 decoding ones and 3
// chunks (warm, in a graph).
__global__ void __launch_bounds__(kPlanThreads) attn_plan_kernel(AttnPlanParams p) {
  extern __shared__ int sm[];
  int* toff = sm;                       // [R + 1] tiles before request r
  __shared__ int hist[kBuckets];
  __shared__ int load[1024];
  __shared__ long long sh[kPlanThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, n = p.n, list = blockIdx.x;
  const Lists ls = lists_of(p.T, p.R, p.G);
  const int tok = ls.tok[list];
  if (tok == 0) return;
  const PlanLayout L = plan_layout(list, p.T, p.R, p.G, p.nkv, n);
  int32_t* plan = p.plan + list_start(list, p.T, p.R, p.G, p.nkv, n);
  int4* tiles = reinterpret_cast<int4*>(plan + L.tiles);
  int* nbs = plan + L.nb;
  int* order = plan + L.order;
  long long* pre = reinterpret_cast<long long*>(plan + L.pre);
  int4* segs = reinterpret_cast<int4*>(plan + L.segs);
  int4* merge = reinterpret_cast<int4*>(plan + L.merge);
  int4* head = reinterpret_cast<int4*>(plan + L.head);
  for (int i = tid; i < kBuckets; i += kPlanThreads) hist[i] = 0;
  load[tid] = 0;
  // ---- tiles of each request; one whose lengths do not fit has none
  {
    const int per = (p.R + kPlanThreads - 1) / kPlanThreads, r0 = min(tid * per, p.R), r1 = min(r0 + per, p.R);
    bool bad = tid == 0 && (p.cu_q[0] != 0 || p.cu_q[p.R] > p.T);
    auto count = [&](int r) -> int {
      const int a = p.cu_q[r], e = p.cu_q[r + 1], len = p.seq_lens[r];
      if (a < 0 || e < a || e > p.T || len < e - a || (long long)len > ((long long)p.width << p.page_shift)) {
        bad = true;
        return 0;
      }
      const bool small = ls.all_small || (e - a) <= ls.tok[kSmall];
      return small == (list == kSmall) ? (e - a + tok - 1) / tok : 0;
    };
    // the rows of all requests together are at most T, so the tiles fit cap_tiles; overlapping rows could claim more,
    // and are cut off there
    long long mine = 0, ex;
    for (int r = r0; r < r1; ++r) mine += count(r);
    const long long tot = block_scan(mine, &ex, sh);
    bad |= tot > L.cap_tiles;
    for (int r = r0; r < r1; ++r) {
      toff[r] = (int)min(ex, (long long)L.cap_tiles);
      ex += count(r);
    }
    if (tid == 0) toff[p.R] = (int)min(tot, (long long)L.cap_tiles);
    if (bad) set_status(p.status, MIMO_ERANGE);
  }
  __syncthreads();
  const int nt = toff[p.R];
  // ---- the tiles, their block counts and the prefix sums of these
  long long W;
  {
    const int per = (nt + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * per, nt), i1 = min(i0 + per, nt);
    long long mine = 0, ex;
    int r = 0;
    if (i0 < i1) {
      int lo = 0, hi = p.R - 1;  // the last request with toff <= i0 (requests without tiles share an offset)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (toff[mid] <= i0) lo = mid; else hi = mid - 1;
      }
      r = lo;
    }
    for (int i = i0; i < i1; ++i) {
      while (toff[r + 1] <= i) ++r;
      const int a = p.cu_q[r], rows = p.cu_q[r + 1] - a, t0 = (i - toff[r]) * tok;
      const int ntok = min(tok, rows - t0), qfirst = p.seq_lens[r] - rows + t0;
      const int nb = blocks_of(qfirst, qfirst + ntok - 1, p.window, p.keep).n;
      tiles[i] = make_int4(a + t0, ntok, qfirst, r);
      nbs[i] = nb;
      atomicAdd(&hist[kBuckets - 1 - bucket_of(nb)], 1);
      mine += nb + kUnitCost;
    }
    W = block_scan(mine, &ex, sh);
    for (int i = i0; i < i1; ++i) {
      pre[i] = ex;
      ex += nbs[i] + kUnitCost;
    }
    if (tid == 0) pre[nt] = W;
  }
  // ---- longest first
  {
    constexpr int per = kBuckets / kPlanThreads;
    long long mine = 0, ex;
    int c[per];
#pragma unroll
    for (int k = 0; k < per; ++k) c[k] = hist[tid * per + k], mine += c[k];
    block_scan(mine, &ex, sh);
#pragma unroll
    for (int k = 0; k < per; ++k) {
      hist[tid * per + k] = (int)ex;
      ex += c[k];
    }
    __syncthreads();
    for (int i = tid; i < nt; i += kPlanThreads)
      order[atomicAdd(&hist[kBuckets - 1 - bucket_of(nbs[i])], 1)] = i;
    __syncthreads();
  }
  const int units = nt * p.nkv;
  W *= p.nkv;
  const int K = (units + n - 1) / n;  // rounds of the snake
  auto cta_of = [&](int u) -> int {
    const int k = u / n, c = u % n;
    return (k & 1) ? n - 1 - c : c;
  };
  for (int u = tid; u < units; u += kPlanThreads)
    atomicAdd(&load[cta_of(u)], sorted_as(nbs[order[u / p.nkv]]) + kUnitCost);
  __syncthreads();
  int most = tid < n ? load[tid] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  __syncthreads();
  if ((tid & 31) == 0) load[tid >> 5] = most;
  __syncthreads();
  for (int w = 0; w < kPlanThreads / 32; ++w) most = max(most, load[w]);
  // a CTA's range holds at least two blocks: a shorter one costs more in its partial result than it saves
  const long long quota = max(2ll + kUnitCost, (W + n - 1) / n);
  const bool split = !whole_units(tok, p.window, p.keep) && quota + p.merge_cost[list] < most;
  if (tid == 0) {
    plan[1] = units;
    plan[2] = split ? 1 : 0;
    plan[0] = p.key;
  }
  for (int c = tid; c < n; c += kPlanThreads) {
    merge[2 * c] = make_int4(0, 0, 0, 0);
    if (!split) {
      const int full = units / n, rest = units % n;
      head[3 * c] = make_int4(c * K, full + (((full & 1) ? n - 1 - c : c) < rest ? 1 : 0), 0, 0);
    } else if (c * quota >= W) {
      head[3 * c] = make_int4(0, 0, 0, 0);
    } else {
      // the unit that holds x on the line of all units' costs, and where its first block lies (its own cost comes before)
      long long first_block;
      auto unit_at = [&](long long x) -> int {
        int lo = 0, hi = nt - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (pre[mid] * p.nkv <= x) lo = mid; else hi = mid - 1;
        }
        const int len = nbs[lo] + kUnitCost, hk = (int)((x - pre[lo] * p.nkv) / len);
        first_block = pre[lo] * p.nkv + (long long)hk * len + kUnitCost;
        return lo * p.nkv + hk;
      };
      const long long end = min(W, (c + 1) * quota);
      const int first = unit_at(c * quota) + (first_block >= end ? 1 : 0);
      const int last = unit_at(end - 1) - (first_block >= end ? 1 : 0);
      head[3 * c] = make_int4(first + c, max(0, last - first + 1), 0, 0);
    }
  }
  __syncthreads();
  for (int u = tid; u < units; u += kPlanThreads) {
    if (!split) {
      const int i = order[u / p.nkv], c = cta_of(u);
      const int4 a = tiles[i], b = make_int4(u % p.nkv, 0, nbs[i], -1);
      int4* s = segs + 2 * ((size_t)c * K + u / n);
      s[0] = a, s[1] = b;
      if (u < n) head[3 * c + 1] = a, head[3 * c + 2] = b;
    } else {
      const int i = u / p.nkv, hk = u % p.nkv, nb = nbs[i];
      const int4 t = tiles[i];
      const long long s0 = pre[i] * p.nkv + (long long)hk * (nb + kUnitCost) + kUnitCost, s1 = s0 + nb;  // its blocks
      const int c0 = (int)(s0 / quota), c1 = (int)((s1 - 1) / quota);
      int slot0 = -1;
      for (int c = c0; c <= c1; ++c) {
        const int b0 = (int)(max(s0, c * quota) - s0), b1 = (int)(min(s1, (c + 1) * quota) - s0);
        const bool first = head[3 * c].x == u + c;
        const int slot = c0 == c1 ? -1 : 2 * c + (first ? 0 : 1);  // a CTA's first segment, or its last
        if (c == c0) slot0 = slot;
        const int4 b = make_int4(hk, b0, b1 - b0, slot);
        int4* s = segs + 2 * ((size_t)u + c);
        s[0] = t, s[1] = b;
        if (first) head[3 * c + 1] = t, head[3 * c + 2] = b;
      }
      if (c1 > c0) {  // at most one unit runs over the end of CTA c0's range
        merge[2 * c0] = make_int4(t.x, t.y, hk, c0);
        merge[2 * c0 + 1] = make_int4(slot0, c1 - c0 + 1, 0, 0);
      }
    }
  }
}

// -------------------------------------------------------------------------------------------------------- attention
__device__ __forceinline__ float ex2_approx(float x) {  // 2^x on the special-function unit: 2^-inf = +0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {  // within an ulp
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16x2_rn(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two float32 operations in one instruction, each rounded as its scalar form.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 32 TMEM columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// Shared-memory matrix descriptors, 128B swizzle, 8-row groups 1024 bytes apart, sm_100 format: the upper word is the
// same for both layouts, the lower one holds address / 16 (advanced by plain additions) and the leading byte offset:
// unused for a K-major operand (Q, K), the stride between groups of 64 values along N for an MN-major one (V).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t saddr) { return (saddr >> 4) | (1024u << 16); }
// kind::f16 MMAs.  One thread issues them, and a product of K = 16 takes the tensor core 64 cycles, so the issue must
// take fewer: the descriptors are put together from one changing word each.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 da, db;\n"
      "setp.ne.u32 p, %4, 0;\n"
      "mov.b64 da, {%1, %5};\nmov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHi)
      : "memory");
}
// A in TMEM: lane = row of A, a 32-bit column holds two consecutive values along K.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 db;\n"
      "setp.ne.u32 p, %4, 0;\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHi)
      : "memory");
}

__device__ __forceinline__ void tmem_st1(uint32_t taddr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};\n" ::"r"(taddr), "r"(r) : "memory");
}
// 32 bytes, 32-byte aligned: a whole sector.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// True in one lane of the warp, which must be whole here.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(r));
  return r != 0;
}
// A box of a 3-D tensor map into shared memory, completing on `bar` (no multicast).
__device__ __forceinline__ void tma_box(void* dst, const void* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
      : "memory");
}

constexpr uint32_t kHead = 1024 + 2048;  // barriers, the exchange between the softmax groups; tiles start at a multiple
                                         // of 1024 bytes, as the block's shared memory does
constexpr uint32_t kChunk = 16384;  // 128 positions x 64 dims, bf16

// Shared memory of the kernel of each list.  A tile of the MMA is 128 rows either way; a small unit's Q is only
// kSmallRows of them in memory, which leaves the ring of K and V room for what HBM's latency needs in flight: with the
// ring that two whole Q tiles leave, a decoding request's block took 2.5 us, most of it the wait for K.  For the other
// rows the MMA reads what lies behind: zeros, after the second buffer's the first one's rows and then zeros (nobody reads
// these results, but products of zeros take less power: with a ring of 12 slots and other data behind Q, 64 decoding
// requests took 125 us under the power cap instead of 117, and 8 of them 24.8 instead of 23.2).
template <int DQK, int DV, int LIST>
struct Shape {
  static constexpr int QCH = DQK / 64, VCH = DV / 64;
  static constexpr uint32_t QROWS = (LIST == kSmall ? kSmallRows : 128) * 128u;  // the rows of 64 dims of a Q tile
  static constexpr uint32_t QZERO = LIST == kSmall ? 128 * 128u - QROWS : 0;    // and the zeros behind both buffers'
  static constexpr uint32_t QB = QCH * (2 * QROWS + QZERO);
  static constexpr __host__ __device__ uint32_t q_at(int buffer, int chunk) {
    return chunk * (2 * QROWS + QZERO) + (1 - buffer) * QROWS;
  }
  static constexpr int NG = 16;  // barriers of K and V blocks: more than the ring holds
  static constexpr int NS = (int)((232448u - kHead - QB) / kChunk);  // ring slots in what Q leaves
  static constexpr uint32_t SMEM = kHead + QB + NS * kChunk;
  // a single tile's second K block is read before its first V block leaves the ring
  static_assert(2 * QCH + VCH <= NS, "the ring must hold K, V and the next K");
  static_assert(2 * ((NS + QCH + VCH - 1) / (QCH + VCH)) < NG, "a barrier for every block in the ring");
};

struct Seg {
  int row0, ntok, qfirst, r, hk, b0, nblk, slot;
};

template <int DQK, int DV, int LIST>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_kernel(const __grid_constant__ PagedAttnParams p) {
  using S = Shape<DQK, DV, LIST>;
  constexpr int NS = S::NS, NG = S::NG, CPB = S::QCH + S::VCH;  // ring slots, block barriers, chunks per block
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint64_t* full = bars;  // K_j is block 2 j of the ring, V_j block 2 j + 1
  uint64_t* empty = full + NG;
  uint64_t* q_full = empty + NG;
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* fix_req = o_full + 2;
  uint64_t* v_fixed = fix_req + 1;
  uint64_t* drain = v_fixed + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile uint32_t* issuer_gone = tslot + 1;  // a wait of the MMA issuer ran out
  float2* xchg = reinterpret_cast<float2*>(smem + 1024);  // [2][128] (maximum, sum) of the tiles' rows
  uint8_t* sQ = smem + kHead;
  uint8_t* sRing = sQ + S::QB;
  if (smem_u32(smem) & 1023) {  // never seen: the swizzled tiles would be read wrongly
    if (threadIdx.x == 0) set_status(p.status, MIMO_EINVAL);
    return;
  }

  // a small unit's rows are all in the first warp of a tile
  constexpr int kRowThreads = LIST == kSmall ? 32 : 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NG; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kRowThreads);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(fix_req, 1);
    mbar_init(v_fixed, 1);
    mbar_init(drain, 1);
    *issuer_gone = 0;
    mbar_fence_init();
  }
  if constexpr (LIST == kSmall) {
    for (int c = 0; c < S::QCH; ++c)
      for (uint32_t i = threadIdx.x * 16; i < S::QZERO; i += kThreads * 16)
        *reinterpret_cast<uint4*>(sQ + S::q_at(0, c) + S::QROWS + i) = make_uint4(0, 0, 0, 0);
    tc::fence_proxy_async_smem();
  }
  if (warp == 9) {
    tc::tmem_alloc(tslot, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tbase = *tslot;
  // q, the cache and the plan come from preceding kernels (programmatic dependent launch).  Where both lists have a
  // kernel, the small one comes second and runs beside the large one, which it does not depend on: it may start when
  // all CTAs of the large one are past this wait, and so are those kernels; it waits for the large one at its end.
  if (!p.second) pdl_wait();
  pdl_launch_dependents();

  const int32_t* plan = p.plan + p.list[LIST].start;
  const int key = plan[0];
  const int4* head = reinterpret_cast<const int4*>(plan + p.list[LIST].head) + 3 * blockIdx.x;
  const int4 where = head[0], first_a = head[1], first_b = head[2];
  const bool planned = key == p.key;  // a plan of these lengths' shape, this layer kind and this GPU
  if (!planned && threadIdx.x == 0) set_status(p.status, MIMO_ERANGE);
  const int nseg = planned ? where.y : 0;
  const int4* segs = reinterpret_cast<const int4*>(plan + p.list[LIST].segs) + 2 * (size_t)where.x;
  const int tpt = (LIST == kSmall ? kSmallRows : 128) / p.G;  // tokens per tile
  const int part_rows = p.list[LIST].part_rows;
  const size_t part0 = p.list[LIST].part0;
  // the CTA's segments in turn, the next one's load in flight while one is worked on
  struct Segs {
    const int4* at;
    int4 a, b;
    int left;
    __device__ __forceinline__ Seg next() {
      const Seg g{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      at += 2;
      if (--left > 0) a = at[0], b = at[1];
      return g;
    }
  } list{segs, first_a, first_b, nseg};
  bool ok = true;

  // TMA producer of Q and K, or of V.  The whole warp runs it and an elected lane issues: a copy then takes 25 cycles to
  // issue, where a branch of lane 0 took 74 alone and 125 here (a block of pages of 16 tokens is 40 copies).  Pages that no
  // query sees are left out.
  auto produce = [&](auto of_v) {
    constexpr bool isv = decltype(of_v)::value;
    constexpr int c0 = isv ? S::QCH : 0, c1 = isv ? CPB : S::QCH;
    const CUtensorMap* map = isv ? &p.vmap : &p.kmap;
    if (lane == 0) {
      tma_prefetch_map(map);
      if (!isv) tma_prefetch_map(&p.qmap);
    }
    const int P = 1 << p.page_shift, ppb = 128 >> p.page_shift;  // pages per block
    const int nowhere = p.num_pages * p.nkv;                    // a row of pages behind the pool: reads zeros
    uint32_t ci = c0, nb = 0;                                    // ring chunk, key blocks issued
    uint32_t freed = 0;                                          // ring blocks known to be free again
    uint32_t nq = 0, turn = 0;                                   // phases of the Q buffers, the next single tile's
    for (int s = 0; s < nseg && ok; ++s) {
      const Seg g = list.next();
      const int qlast = g.qfirst + g.ntok - 1;
      const Blocks bl = blocks_of(g.qfirst, qlast, p.window, p.keep);
      const int* trow = p.table + (size_t)g.r * p.width;
      // the number of the block's page `lane`, and whether a query sees that page (a flag of its own: the table may hold
      // any number); loaded a block ahead
      int page = 0;
      bool vis = false;
      auto load_page = [&](int j) {
        const int kb = j < bl.nkb ? j : bl.lb + (j - bl.nkb);
        const int pg = kb * ppb + lane, pos = pg << p.page_shift;
        vis = lane < ppb && pg < p.width && pos <= qlast && (pos + P - 1 >= bl.lo || pos < bl.keep);
        if (vis) page = trow[pg];
      };
      load_page(g.b0);
      for (int j = 0; j < g.nblk && ok; ++j) {
        const bool in_pool = (unsigned)page < (unsigned)p.num_pages;
        const int row = in_pool ? page * p.nkv + g.hk : nowhere;
        if (vis && !in_pool) set_status(p.status, MIMO_ERANGE);
        const uint32_t seen = __ballot_sync(0xFFFFFFFFu, vis);
        if (j + 1 < g.nblk) load_page(g.b0 + j + 1);
        int rows[8];  // the same in all lanes: uniform registers, from which a copy is issued in 25 cycles
#pragma unroll
        for (int i = 0; i < 8; ++i) rows[i] = __shfl_sync(0xFFFFFFFFu, row, i);
        uint64_t* bar = &full[(2 * nb + (isv ? 1 : 0)) % NG];
        for (int c = c0; c < c1; ++c) {
          const uint32_t at = ci + (c - c0);
          if (at >= (uint32_t)NS) {  // the ring block whose chunk was in this slot must have been read
            const uint32_t old = at - NS, of = 2 * (old / CPB) + (old % CPB >= (uint32_t)S::QCH ? 1 : 0);
            if (ok && of >= freed) ok = mbar_wait(&empty[of % NG], (of / NG) & 1);
            freed = of + 1;
          }
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          if (elect_one()) {
            if (c == c0) mbar_arrive_expect_tx(bar, (uint32_t)((c1 - c0) * __popc(seen) * P * 128));
            uint8_t* dst = sRing + (at % NS) * kChunk;
            const int dim = (isv ? c - S::QCH : c) * 64;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if ((seen >> i) & 1) tma_box(dst + i * P * 128, map, dim, 0, rows[i], bar);
          }
          __syncwarp();
        }
        if (!isv && j == 0) {  // Q behind the first K block: both buffers, or the one whose turn it is
          const bool pair = LIST == kLarge && g.ntok > tpt;
          for (int x = 0; x < (pair ? 2 : 1); ++x) {
            const int qb = pair ? x : turn;
            if (ok) ok = mbar_wait(&q_empty[qb], ((nq >> qb) & 1) ^ 1);
            nq ^= 1u << qb;
            if (ok && elect_one()) {
              mbar_arrive_expect_tx(&q_full[qb], (uint32_t)(S::QCH * 128 * p.G * tpt));
#pragma unroll
              for (int d = 0; d < S::QCH; ++d)
                tma_box(sQ + S::q_at(qb, d), &p.qmap, d * 64, g.hk * p.G, g.row0 + x * tpt, &q_full[qb]);
            }
          }
          if (!pair) turn ^= 1;
        }
        ci += CPB;
        ++nb;
      }
    }
    // no copy may still be landing when the CTA exits: the last blocks (after a wait that ran out, what there is of the
    // block it was in: this wait runs out too), and Q
    const uint32_t begun = ok ? nb : nb + 1;
    for (uint32_t k = 0; k < (uint32_t)NG / 2 && k < begun; ++k) {
      const uint32_t i = 2 * (begun - 1 - k) + (isv ? 1 : 0);
      mbar_wait(&full[i % NG], (i / NG) & 1);
    }
    if (!isv)
      for (int x = 0; x < 2; ++x) mbar_wait(&q_full[x], ((nq >> x) & 1) ^ 1);
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegsOther));
    if (warp == 8) {
      produce(std::false_type{});
    } else if (warp == 11) {
      produce(std::true_type{});
    } else if (warp == 9) {
      // --------------------------------------------------------------------------------------------- MMA issuer
      // The whole warp runs this and one elected lane issues: what all lanes agree on stays in uniform registers, which
      // the MMA reads its operands from.  (From a branch of one lane an MMA took 70 cycles to issue, 90 to 100 beside
      // the softmax warps; this way 64, the tensor core's own time for 128 x 128 x 16.)
      const uint32_t idesc_s = tc::idesc_bf16(128, 128);
      const uint32_t idesc_o64 = tc::idesc_bf16(128, 64) | (1u << 16);  // B = V, MN-major
      const uint32_t idesc_o = tc::idesc_bf16(128, DV) | (1u << 16);
      const uint32_t aq = desc_k(smem_u32(sQ)), bk = desc_k(smem_u32(sRing)), bv = desc_mn(smem_u32(sRing));
      const uint32_t tb = __shfl_sync(0xFFFFFFFFu, tbase, 0);
      uint32_t nb = 0, slot = 0;  // key blocks before this one, ring slot of its first chunk
      uint32_t nq = 0, turn = 0, np = 0, nfix = 0;  // phases
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
        tc::tc_fence_after();
      };
      auto there = [&](uint32_t g) { wait(&full[g % NG], (g / NG) & 1); };
      auto q_there = [&](int qb) {
        wait(&q_full[qb], (nq >> qb) & 1);
        nq ^= 1u << qb;
      };
      auto p_there = [&](int x) {
        wait(&p_full[x], (np >> x) & 1);
        np ^= 1u << x;
      };
      auto fixed = [&]() { wait(v_fixed, nfix++ & 1); };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc::tc_commit(bar);
      };
      auto wrap = [](uint32_t sl) -> uint32_t { return sl >= (uint32_t)NS ? sl - NS : sl; };
      // S = Q K^T of tile x from Q buffer qb and the K chunks at ring slot `at`
      auto issue_s = [&](int x, int qb, uint32_t at) {
        const uint32_t d = tb + x * 128;
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < S::QCH; ++c) {
            const uint32_t a = aq + S::q_at(qb, c) / 16, b = bk + wrap(at + c) * (kChunk / 16);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma_ss(d, a + kk * 2, b + kk * 2, idesc_s, (c | kk) != 0);
          }
          tc::tc_commit(&s_full[x]);
        }
        __syncwarp();
      };
      // O += P V of tile x from the V chunks at ring slot `at`
      auto issue_pv = [&](int x, uint32_t at, bool first) {
        const uint32_t d = tb + 256 + x * DV, a = tb + x * 128;
        if (elect_one()) {
          if (S::VCH == 1 || at + 1 < (uint32_t)NS) {  // the V chunks lie one behind the other
            const uint32_t b = bv + at * (kChunk / 16);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) mma_ts(d, a + kk * 8, b + kk * 128, idesc_o, kk != 0 || !first);
          } else {
#pragma unroll
            for (int c = 0; c < S::VCH; ++c) {
              const uint32_t b = bv + wrap(at + c) * (kChunk / 16);
#pragma unroll
              for (int kk = 0; kk < 8; ++kk) mma_ts(d + c * 64, a + kk * 8, b + kk * 128, idesc_o64, kk != 0 || !first);
            }
          }
        }
        __syncwarp();
      };
      for (int s = 0; s < nseg && ok; ++s) {
        Seg g = list.next();
        g.ntok = __shfl_sync(0xFFFFFFFFu, g.ntok, 0), g.qfirst = __shfl_sync(0xFFFFFFFFu, g.qfirst, 0);
        g.b0 = __shfl_sync(0xFFFFFFFFu, g.b0, 0), g.nblk = __shfl_sync(0xFFFFFFFFu, g.nblk, 0);
        const int qlast = g.qfirst + g.ntok - 1;
        const Blocks bl = blocks_of(g.qfirst, qlast, p.window, p.keep);
        // block j of the unit has V rows that are nobody's
        auto ragged = [&](int j) -> bool {
          const int kb = j < bl.nkb ? j : bl.lb + (j - bl.nkb), kp = kb * 128;
          return !(kp + 127 <= qlast && (kp >= bl.lo || kp + 127 < bl.keep));
        };
        auto request_fix = [&]() {
          if (ok && elect_one()) mbar_arrive(fix_req);
        };
        if (LIST == kLarge && g.ntok > tpt) {  // a pair: both tiles on every block
          there(2 * nb);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            q_there(x);
            if (!ok) break;
            issue_s(x, x, slot);
            if (g.nblk == 1) commit(&q_empty[x]);
          }
          commit(&empty[(2 * nb) % NG]);
          for (int j = 0; j < g.nblk && ok; ++j, ++nb) {
            const uint32_t vs = wrap(slot + S::QCH), next = wrap(vs + S::VCH);
            const bool more = j + 1 < g.nblk, fix = ragged(g.b0 + j);
            there(2 * nb + 1);
            if (fix) request_fix();  // zeroed while the softmax runs
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              p_there(x);
              if (x == 0 && fix) fixed();
              if (!ok) break;
              issue_pv(x, vs, j == 0);
              if (x == 1) commit(&empty[(2 * nb + 1) % NG]);
              if (more) {
                if (x == 0) there(2 * nb + 2);
                if (!ok) break;
                issue_s(x, x, next);
                if (x == 1) commit(&empty[(2 * nb + 2) % NG]);
                if (j + 2 == g.nblk) commit(&q_empty[x]);
              } else {
                commit(&o_full[x]);
              }
            }
            slot = next;
          }
        } else {  // one tile: blocks in turn as A and B
          const uint32_t qb = turn, nb0 = nb;
          turn ^= 1;
          uint32_t ks = slot, kb = nb;  // the next block whose S is issued
          auto issue_next = [&](int x) {
            there(2 * kb);
            if (!ok) return;
            issue_s(x, qb, ks);
            commit(&empty[(2 * kb) % NG]);
            ks = wrap(ks + CPB);
            if (++kb == nb0 + g.nblk) commit(&q_empty[qb]);
          };
          q_there(qb);
          issue_next(0);
          if (g.nblk > 1) issue_next(1);
          for (int j = 0; j < g.nblk && ok; ++j, ++nb) {
            const int x = j & 1;
            const uint32_t vs = wrap(slot + S::QCH);
            const bool fix = ragged(g.b0 + j);
            there(2 * nb + 1);
            if (fix) request_fix();
            p_there(x);
            if (fix) fixed();
            if (!ok) break;
            issue_pv(x, vs, j < 2);
            commit(&empty[(2 * nb + 1) % NG]);
            // this block's V may have to leave the ring before that K can come
            if (j + 2 < g.nblk) issue_next(x);
            slot = wrap(vs + S::VCH);
          }
          commit(&o_full[0]);
          commit(&o_full[1]);
        }
      }
      if (!ok) *issuer_gone = 1;
      commit(drain);  // every MMA issued above has completed once this arrives
      if (!mbar_wait(drain, 0)) ok = false;
    } else if (warp == 10) {  // --------------------------------------------------- zeroes what nobody sees of V
      uint32_t ci = 0, fixes = 0;
      for (int s = 0; s < nseg && ok; ++s) {
        const Seg g = list.next();
        const int qlast = g.qfirst + g.ntok - 1;
        const Blocks bl = blocks_of(g.qfirst, qlast, p.window, p.keep);
        for (int j = 0; j < g.nblk && ok; ++j, ci += CPB) {
          const int kb = g.b0 + j < bl.nkb ? g.b0 + j : bl.lb + (g.b0 + j - bl.nkb);
          const int kp = kb * 128;
          if (kp + 127 <= qlast && (kp >= bl.lo || kp + 127 < bl.keep)) continue;
          // the block's V is there.  The blocks before it may be any number, whole units among them, so this wait only
          // ends when the issuer's own, which are for single blocks, do
          do ok = mbar_wait(fix_req, fixes & 1);
          while (!ok && !*issuer_gone);
          ++fixes;
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          auto zero = [&](int from, int to) {
            from = max(from, kp), to = min(to, kp + 128);
            for (int i = from * 8 + lane; i < to * 8; i += 32) {  // a row is 128 bytes whatever the swizzle
#pragma unroll
              for (int c = 0; c < S::VCH; ++c)
                *reinterpret_cast<uint4*>(sRing + ((ci + S::QCH + c) % NS) * kChunk + (i - kp * 8) * 16) =
                    make_uint4(0, 0, 0, 0);
            }
          };
          zero(qlast + 1, kp + 128);
          zero(bl.keep, bl.lo);
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(v_fixed);
        }
      }
    }
  } else {  // ------------------------------------------------------------------------------- softmax of tile x
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegsSoftmax));
    const int x = warp >> 2, r = threadIdx.x & 127;
    if (LIST != kSmall || (warp & 3) == 0) {  // a small unit's rows are a tile's first warp's
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tbase + x * 128 + lane_off, tO = tbase + 256 + x * DV + lane_off;
    const int head = r % p.G;  // this row's head of the group
    const float sl2 = p.scale_log2;
    uint32_t ns = 0, no = 0;
    for (int s = 0; s < nseg; ++s) {
      const Seg g = list.next();
      const bool pair = LIST == kLarge && g.ntok > tpt;
      const int tt = r / p.G + (pair ? x * tpt : 0);  // its token of the unit
      const Blocks bl = blocks_of(g.qfirst, g.qfirst + g.ntok - 1, p.window, p.keep);
      const bool row_ok = r < tpt * p.G && tt < g.ntok;
      const bool work = __any_sync(0xFFFFFFFFu, row_ok);  // a warp without a row only keeps the barriers going
      // rows without a query compute on what lies there, unmasked: nobody reads their results
      const int qpos = row_ok ? g.qfirst + tt : 0x7FFFFFFF;
      const int lo = p.window > 0 && row_ok ? max(0, qpos - p.window + 1) : 0;
      const int keep = min(p.keep, lo);
      float m_ref = -INFINITY, m_new = -INFINITY, l = 0.f;
      bool fresh = true;
      const float sink = p.sinks && row_ok ? p.sinks[g.hk * p.G + head] * kLog2e : 0.f;
      // where the row's output goes, worked out while the scores are on their way: itself, or a part in the workspace;
      // and the rows of the pair of lanes that exchange theirs
      const int row = g.row0 + tt;
      const bool store = row_ok && row < p.T;
      const size_t at = part0 + (size_t)max(g.slot, 0) * part_rows + (tt * p.G + head);
      uint8_t* to = g.slot < 0 ? reinterpret_cast<uint8_t*>(p.out + ((size_t)row * p.nq + g.hk * p.G + head) * DV)
                               : reinterpret_cast<uint8_t*>(p.part_o + at * DV);
      uint8_t* pair_to[2] = {to, to};
      uint32_t pair_ok = 0;
      if constexpr (LIST == kLarge) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          pair_to[k] = reinterpret_cast<uint8_t*>(
              __shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(to), (lane & ~1) | k));
        pair_ok = __ballot_sync(0xFFFFFFFFu, store) >> (lane & ~1);
      }
      // after a wait that ran out the loops go on without work, for the barriers that both groups must pass
      for (int j = pair ? 0 : x; j < g.nblk; j += pair ? 1 : 2) {
        if (ok) ok = mbar_wait(&s_full[x], ns & 1);
        ++ns;
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) continue;
        tc::tc_fence_after();
        if (work) {
          const int jb = g.b0 + j, kp = (jb < bl.nkb ? jb : bl.lb + (jb - bl.nkb)) * 128;
          const bool masked = !(kp + 127 <= qpos && (kp >= lo || kp + 127 < keep));
          // 32 columns at a time as a word of visible bits: [c_lo, c_hi] and [0, c_keep)
          auto mask = [&](float* v, int w0) {
            const int c_hi = qpos - kp - w0, c_lo = lo - kp - w0, c_keep = keep - kp - w0;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              auto below = [&](int c) -> uint32_t {  // bits of the columns < c
                const int k = min(max(c - w * 32, 0), 32);
                return k == 32 ? 0xFFFFFFFFu : (1u << k) - 1u;
              };
              const uint32_t seen = below(min(c_hi, 0x7FFFFFFE) + 1) & (~below(c_lo) | below(c_keep));
              if (seen != 0xFFFFFFFFu) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (!(seen & (1u << e))) v[w * 32 + e] = -INFINITY;
              }
            }
          };
          // The reference of the exponentials is a maximum of what came before: a bf16 or float32 value is as exact beside
          // 2^60 as beside 1, so the exponentials need not wait for their own maximum.  A maximum 2^8 above the reference
          // is taken up at the next block, one 2^60 above it (and a row's first) at once.
          // (rows without a query have no say: what they compute on may be anything)
          float to = m_new;
          bool now = row_ok && m_new > m_ref + 8.f;
          m_new = -INFINITY;
          // The halves one after the other through the same instructions, and one copy of what is rare: written out, the
          // loop was larger than the instruction caches hold, and the warps waited for it.
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            // A half that none of the warp's rows sees has no P (a window of 128 is two halves of four, 48 requests: 21.0
            // us instead of 21.8; in the large units' loop it cost more than it saved).
            const int first = kp + hf * 64;
            if (LIST == kSmall && p.window > 0 &&
                !__any_sync(0xFFFFFFFFu, row_ok && ((first <= qpos && first + 63 >= lo) || first < keep))) {
              uint32_t none[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) none[e] = 0;
              tmem_st32(tS + hf * 32, none);
              continue;
            }
            float v[64];
            tmem_ld32(tS + hf * 64, v);
            tmem_ld32(tS + hf * 64 + 32, v + 32);
            tc::tmem_wait_ld();
            if (masked) mask(v, hf * 64);
            if (fresh) {  // rows without a reference yet: the unit's first block, and rows that have seen no key so far
              float a = v[0];
#pragma unroll
              for (int e = 1; e < 63; e += 2) a = fmaxf(fmaxf(a, v[e]), v[e + 1]);
              a = fmaxf(a, v[63]) * sl2;
              if (row_ok && m_ref == -INFINITY && a > -INFINITY) to = a, now = true;
            }
            uint32_t pk[32];
            uint64_t sum[2];
            bool again = false;  // the half's exponentials once more
            for (;;) {
              // A new reference: O, which holds the products of the blocks before (see above), the sum, and in a second
              // half the first half's P are scaled to it.
              if (__any_sync(0xFFFFFFFFu, now)) {
                const float alpha = now && m_ref != -INFINITY ? ex2_approx(m_ref - to) : 1.f;
                if (now) m_ref = to;
                l *= alpha;
                if (__any_sync(0xFFFFFFFFu, alpha != 1.f)) {
#pragma unroll 1
                  for (int c = 0; c < DV; c += 16) {
                    float o[16];
                    tc::tmem_ld<16>(tO + c, o);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= alpha;
                    tmem_st16(tO + c, reinterpret_cast<const uint32_t*>(o));
                  }
                  tmem_wait_st();
                  if (again && hf == 1) {
#pragma unroll 1
                    for (int c = 0; c < 32; ++c) {
                      float w[1];
                      tc::tmem_ld<1>(tS + c, w);
                      tc::tmem_wait_ld();
                      const uint32_t u = __float_as_uint(w[0]);
                      tmem_st1(tS + c, pack_bf16x2_rn(__uint_as_float(u << 16) * alpha,
                                                      __uint_as_float(u & 0xFFFF0000u) * alpha));
                    }
                    tmem_wait_st();
                  }
                }
                fresh = __any_sync(0xFFFFFFFFu, row_ok && m_ref == -INFINITY);
              }
              // P = bf16(2^(s * scale * log2 e - reference)) and their sum, and their maximum on the way (the scale is
              // positive, so it orders the scaled scores alike).  The special-function unit bounds this loop, and what
              // else it does has to lie between its instructions.
              const uint64_t sc = pack2(sl2, sl2), nm = m_ref == -INFINITY ? 0 : pack2(-m_ref, -m_ref);
              float a = -INFINITY, b = -INFINITY;
              sum[0] = sum[1] = 0;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float2 t = unpack2(fma2(pack2(v[2 * i], v[2 * i + 1]), sc, nm));
                const float p0 = ex2_approx(t.x), p1 = ex2_approx(t.y);
                if (i & 1) b = fmaxf(fmaxf(b, v[2 * i]), v[2 * i + 1]);
                else a = fmaxf(fmaxf(a, v[2 * i]), v[2 * i + 1]);
                sum[i & 1] = add2(sum[i & 1], pack2(p0, p1));
                pk[i] = pack_bf16x2_rn(p0, p1);  // rounded to bf16 for the product with V, the sum is not
              }
              to = fmaxf(a, b) * sl2;
              m_new = fmaxf(m_new, to);
              now = row_ok && to > m_ref + 60.f;
              again = __any_sync(0xFFFFFFFFu, now);
              if (!again) break;
            }
            const float2 s0 = unpack2(add2(sum[0], sum[1]));
            l += s0.x + s0.y;
            tmem_st32(tS + hf * 32, pk);
          }
          tmem_wait_st();
        }
        tc::tc_fence_before();
        mbar_arrive(&p_full[x]);
      }
      if (ok) ok = mbar_wait(&o_full[x], no & 1);
      ++no;
      ok = __all_sync(0xFFFFFFFFu, ok);
      // this thread's columns of the row, and the weights of the two outputs they are joined from (a pair's have one)
      int c0 = 0, c1 = DV;
      float w_own = 1.f, w_other = 0.f;
      bool own = true, other = false;  // whether there is such an output (one never written may hold anything)
      if (!pair) {
        xchg[x * 128 + r] = make_float2(m_ref, l);
        named_bar_sync(1, 2 * kRowThreads);
        const float2 o = xchg[(x ^ 1) * 128 + r];
        const float M = fmaxf(m_ref, o.x);
        own = m_ref != -INFINITY || l != 0.f, other = o.x != -INFINITY || o.y != 0.f;
        w_own = m_ref == -INFINITY ? 0.f : ex2_approx(m_ref - M);
        w_other = o.x == -INFINITY ? 0.f : ex2_approx(o.x - M);
        l = l * w_own + o.y * w_other;
        m_ref = M;
        c0 = x * (DV / 2), c1 = c0 + DV / 2;
      }
      tc::tc_fence_after();
      if (work && ok) {
        const uint32_t tOther = tbase + 256 + (x ^ 1) * DV + lane_off;
        float f = 1.f;  // an unnormalised part: maximum (log2), sum and output of these blocks
        if (g.slot < 0) {
          if (p.sinks) {
            const float M = fmaxf(m_ref, sink);
            const float a = m_ref == -INFINITY ? 0.f : ex2_approx(m_ref - M);
            f = a * rcp_approx(l * a + ex2_approx(sink - M));
          } else {
            f = l == 0.f ? 0.f : rcp_approx(l);
          }
        }
        w_own *= f, w_other *= f;
        // 32 columns of the warp's rows: 64 bytes of a row, stored as whole sectors.  A store to 32 different rows takes
        // the load/store unit 32 turns; with eight warps at it, lanes of a pair first exchange theirs, so that a store
        // writes 64 bytes of 16 rows (23 decoding requests + 2 chunks: 113.5 us instead of 117.0).  A small unit's one
        // warp a tile is better off without the shuffles (48 requests in a window of 128: 18.1 us instead of 19.1).
        auto emit = [&](int c, float* o) {
          if (g.slot >= 0) {
            if (store)
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                st_global_v8(reinterpret_cast<float*>(to) + c + e, reinterpret_cast<uint32_t*>(o + e));
            return;
          }
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack_bf16x2_rn(o[2 * e], o[2 * e + 1]);
          if constexpr (LIST == kSmall) {
            if (store) {
              st_global_v8(to + c * 2, w);
              st_global_v8(to + c * 2 + 32, w + 8);
            }
          } else {
            const bool odd = lane & 1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t take = __shfl_xor_sync(0xFFFFFFFFu, odd ? w[e] : w[8 + e], 1);
              w[e] = odd ? take : w[e];
              w[8 + e] = odd ? w[8 + e] : take;
            }
            if (pair_ok & 1) st_global_v8(pair_to[0] + c * 2 + odd * 32, w);
            if (pair_ok & 2) st_global_v8(pair_to[1] + c * 2 + odd * 32, w + 8);
          }
        };
#pragma unroll 1
        for (int c = c0; c < c1; c += pair ? 64 : 32) {  // 64 columns at a time, or 32 of both outputs
          float o[32], q[32];
          tmem_ld32(tO + c, o);
          tmem_ld32(pair ? tO + c + 32 : tOther + c, q);
          tc::tmem_wait_ld();
          if (pair) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= w_own, q[e] *= w_own;
            emit(c, o);
            emit(c + 32, q);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              o[e] = own ? o[e] * w_own : 0.f;
              o[e] = other ? fmaf(q[e], w_other, o[e]) : o[e];
            }
            emit(c, o);
          }
        }
        if (store && g.slot >= 0 && c0 == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_ref, l);
      }
      tc::tc_fence_before();
      if (!pair) named_bar_sync(2, 2 * kRowThreads);  // both outputs are read, and the exchange may be written again
    }
    }
  }
  if (!ok && p.status) set_status(p.status, MIMO_ETIMEOUT);
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tbase, 512);
  }
  if (p.second) pdl_wait();
}

// ------------------------------------------------------------------------------------------------------------ merge
// Joins the parts of the unit that runs over the end of CTA blockIdx.x's range: a warp per query row, in the order of
// the parts, so that the result does not depend on when they were done.
constexpr int kMergeWarps = 8;

template <int DV>
__global__ void __launch_bounds__(kMergeWarps * 32) paged_attn_merge_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int VL = DV / 32, AHEAD = 8;  // parts loaded at a time
  // the plan is older than the attention kernels, which are all past their wait for it when this grid starts
  const int list = p.list[kSmall].part_rows > 0 ? (int)blockIdx.z : kLarge;
  const int32_t* plan = p.plan + p.list[list].start;
  const int key = plan[0];
  const int4* mg = reinterpret_cast<const int4*>(plan + p.list[list].merge) + 2 * (size_t)blockIdx.x;
  const int4 a = mg[0], b = mg[1];  // row0, tokens, kv head, first CTA; slot of the first part, parts
  const int part_rows = p.list[list].part_rows, lane = threadIdx.x & 31;
  const size_t part0 = p.list[list].part0;
  pdl_wait();
  pdl_launch_dependents();
  if (key != p.key) return;
  for (int rr = blockIdx.y * kMergeWarps + (threadIdx.x >> 5); rr < a.y * p.G; rr += gridDim.y * kMergeWarps) {
    const int tt = rr / p.G, qh = a.z * p.G + rr % p.G, row = a.x + tt;
    auto part = [&](int s) -> size_t { return part0 + (size_t)(s == 0 ? b.x : 2 * (a.w + s)) * part_rows + rr; };
    const float sink = p.sinks ? p.sinks[qh] * kLog2e : -INFINITY;
    // the parts in turn, the row's sum and output scaled to the largest maximum so far
    float M = sink, sum = p.sinks ? 1.f : 0.f, acc[VL];
#pragma unroll
    for (int k = 0; k < VL; ++k) acc[k] = 0.f;
    for (int s0 = 0; s0 < b.y; s0 += AHEAD) {
      float2 ml[AHEAD], o[AHEAD][VL / 2];
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        ml[s] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int k = 0; k < VL / 2; ++k) o[s][k] = make_float2(0.f, 0.f);
        if (s0 + s < b.y) {
          const size_t at = part(s0 + s);
          ml[s] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
#pragma unroll
          for (int k = 0; k < VL / 2; ++k)
            o[s][k] = reinterpret_cast<const float2*>(p.part_o + at * DV + lane * VL)[k];
        }
      }
      float Mn = M;
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) Mn = fmaxf(Mn, ml[s].x);
      const float f0 = M == -INFINITY ? 0.f : exp2f(M - Mn);
      sum *= f0;
#pragma unroll
      for (int k = 0; k < VL; ++k) acc[k] *= f0;
      M = Mn;
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) {
        const float f = ml[s].x == -INFINITY ? 0.f : exp2f(ml[s].x - M);
        sum = fmaf(f, ml[s].y, sum);
#pragma unroll
        for (int k = 0; k < VL / 2; ++k) {
          acc[2 * k] = fmaf(f, o[s][k].x, acc[2 * k]);
          acc[2 * k + 1] = fmaf(f, o[s][k].y, acc[2 * k + 1]);
        }
      }
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    if (row >= p.T) continue;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + ((size_t)row * p.nq + qh) * DV + lane * VL);
#pragma unroll
    for (int k = 0; k < VL / 2; ++k) dst[k] = pack_bf16x2_rn(acc[2 * k] * f, acc[2 * k + 1] * f);
  }
}

template <int DQK, int DV, int LIST>
cudaError_t launch_list(PagedAttnParams& p, int num_sms, cudaStream_t st) {
  using S = Shape<DQK, DV, LIST>;
  static bool attr_set[128] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 128 && !attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<DQK, DV, LIST>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    if (e != cudaSuccess) return e;
    attr_set[dev] = true;
  }
  const int tile = (LIST == kSmall ? kSmallRows : 128) / p.G;  // tokens
  const cudaError_t e = bf16_map3(&p.qmap, p.q, (uint64_t)DQK, (uint64_t)p.nq, (uint64_t)p.T, p.G, tile);
  if (e != cudaSuccess) return e;
  return launch_k(paged_attn_kernel<DQK, DV, LIST>, dim3(num_sms), dim3(kThreads), S::SMEM, st, p);
}

template <int DQK, int DV>
cudaError_t launch_t(PagedAttnParams& p, int num_sms, cudaStream_t st) {
  const Lists ls = lists_of(p.T, p.R, p.G);
  const bool both = ls.tok[kSmall] > 0 && ls.tok[kLarge] > 0;
  for (int l : {kSmall, kLarge}) {
    const PlanLayout L = plan_layout(l, p.T, p.R, p.G, p.nkv, num_sms);
    p.list[l] = {list_start(l, p.T, p.R, p.G, p.nkv, num_sms), L.head, L.merge, L.segs,
                 part_start(l, p.T, p.R, p.G, num_sms), part_rows_of(l, p.T, p.R, p.G)};
  }
  cudaError_t e = cudaSuccess;
  if (ls.tok[kLarge] > 0) e = launch_list<DQK, DV, kLarge>(p, num_sms, st);
  if (e != cudaSuccess) return e;
  p.second = both ? 1 : 0;
  if (ls.tok[kSmall] > 0) e = launch_list<DQK, DV, kSmall>(p, num_sms, st);
  const bool whole =
      whole_units(ls.tok[kSmall], p.window, p.keep) && whole_units(ls.tok[kLarge], p.window, p.keep);
  if (e != cudaSuccess || whole) return e;
  const int rows = std::max(part_rows_of(kSmall, p.T, p.R, p.G), part_rows_of(kLarge, p.T, p.R, p.G));
  return launch_k(paged_attn_merge_kernel<DV>,
                  dim3(num_sms, std::min(8, (rows + kMergeWarps - 1) / kMergeWarps), both ? 2 : 1),
                  dim3(kMergeWarps * 32), 0, st, p);
}

}  // namespace

bool attn_units_fit(int T, int R, int G, int nkv) {
  const Lists ls = lists_of(T, R, G);
  for (int l : {kSmall, kLarge})
    if ((long long)cap_tiles_of(ls, l, T, R) * nkv > 1 << 30) return false;
  return true;
}

size_t attn_plan_bytes(int T, int R, int G, int nkv, int num_sms) {
  return 4 * (list_start(kLarge, T, R, G, nkv, num_sms) + plan_layout(kLarge, T, R, G, nkv, num_sms).words);
}

size_t paged_attn_part_rows(int T, int R, int G, int num_sms) {
  return part_start(kLarge, T, R, G, num_sms) + (size_t)2 * num_sms * part_rows_of(kLarge, T, R, G);
}

cudaError_t launch_attn_plan(AttnPlanParams& p, cudaStream_t st) {
  // a split's cost in blocks: its parts' rows written and read again, and the merge
  for (int l : {kSmall, kLarge}) p.merge_cost[l] = 1 + part_rows_of(l, p.T, p.R, p.G) / 64;
  return launch_k(attn_plan_kernel, dim3(2), dim3(kPlanThreads), (size_t)(p.R + 1) * 4, st, p);
}

cudaError_t launch_paged_attention(PagedAttnParams& p, int num_sms, cudaStream_t st) {
  const uint64_t rows = (uint64_t)p.num_pages * p.nkv;
  const int P = 1 << p.page_shift;
  cudaError_t e = bf16_map3(&p.kmap, p.k, (uint64_t)p.dqk, (uint64_t)P, rows, P, 1);
  if (e == cudaSuccess) e = bf16_map3(&p.vmap, p.v, (uint64_t)p.dv, (uint64_t)P, rows, P, 1);
  if (e != cudaSuccess) return e;
  if (p.dqk == 192) return launch_t<192, 128>(p, num_sms, st);
  if (p.dqk == 128) return launch_t<128, 128>(p, num_sms, st);
  return launch_t<64, 64>(p, num_sms, st);
}

}  // namespace mimo
