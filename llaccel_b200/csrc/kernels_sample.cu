// Sampling one token per row of integer logits: temperature, top-k, top-p and min-p from a given
// random number, in integers throughout.
//
// A token g = max - l steps below its row's largest logit has the weight
//   step = rint(log2(e) 2^(32 + exponent) / temperature), at most 2^47
//   e    = (g * step) >> 12                    the gap in units of 2^-20 octaves
//   b    = kDevPow2[(e >> 10) & 1023]          2^31 * 2^-(the next 10 bits)
//   w    = (b - ((b * ((e & 1023) * 2839)) >> 32)) >> (e >> 20)
// 2839 2^-32 is ln(2) 2^-20: the last 10 bits of the exponent enter to first order, which leaves
// a relative error below 2^-21 (their square's half, (ln(2) 2^-10)^2 / 2 = 2^-22.1, and the
// roundings).  w falls monotonically in g, so the tokens that any of the filters keeps are a
// prefix of the order (gap, index): all of gap < G and the first c, by index, of gap == G.
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "device_luts.h"
#include "launch.cuh"
#include "paged.h"

namespace llx {

// The weight of gap g, 0 from `limit` on.  SMALL: step < 2^28, so e stays in 32 bits (g is below 2^16).
template <bool SMALL>
__device__ __forceinline__ uint32_t gap_weight(uint32_t g, uint64_t step, const uint32_t* pow2, uint32_t limit = ~0u) {
  uint32_t e, n;
  if (SMALL) {
    e = __umulhi(g << 16, (uint32_t)step << 4);  // (g * step) >> 12
    if (g >= limit) e = 32u << 20;  // and all such lanes look up the same entry
    n = e >> 20;
  } else {
    const uint64_t x = (g * step) >> 12;
    e = (uint32_t)x;
    n = x >> 20 < 32 && g < limit ? (uint32_t)(x >> 20) : 32u;
  }
  const uint32_t b = pow2[(e >> 10) & 1023u];
  uint32_t w;
  asm("shr.u32 %0, %1, %2;" : "=r"(w) : "r"(b - __umulhi(b, (e & 1023u) * 2839u)), "r"(n));  // 0 from 32 bits on
  return w;
}

// floor and ceiling of total * f / 2^31, f <= 2^31
__device__ __forceinline__ uint64_t part_floor(uint64_t total, uint32_t f) {
  return (total >> 31) * f + (((total & 0x7FFFFFFFull) * f) >> 31);
}
__device__ __forceinline__ uint64_t part_ceil(uint64_t total, uint32_t f) {
  const uint64_t low = (total & 0x7FFFFFFFull) * f;
  return (total >> 31) * f + (low >> 31) + ((low & 0x7FFFFFFFull) ? 1 : 0);
}

// what one row's settings come to
struct SampleRow {
  uint64_t step;
  uint32_t part;   // top-p in units of 2^-31
  uint32_t least;  // min-p's smallest weight
  uint32_t u;      // random number in units of 2^-31
};

__device__ __forceinline__ int64_t row_k(const llx_sample_args& a, int64_t r) {
  if (a.temperature && !(a.temperature[r] > 0.0f)) return 1;
  const int k = a.top_k ? a.top_k[r] : 0;
  return k <= 0 || k > a.vocab ? a.vocab : k;
}

__device__ __forceinline__ SampleRow sample_row(const llx_sample_args& a, int64_t r) {
  SampleRow s;
  const float temp = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  // log2(e) 2^(32 + exponent): a power of two times the double nearest to log2(e)
  const double unit = scalbn(1.4426950408889634, (int)(32 + a.exponent));
  const double q = greedy ? 0.0 : rint(unit / (double)temp);
  s.step = q >= 140737488355328.0 ? 1ull << 47 : (uint64_t)q;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  s.part = !(p > 0.0f) ? 0u : p >= 1.0f ? 1u << 31 : (uint32_t)((double)p * 2147483648.0);
  const float m = a.min_p ? a.min_p[r] : 0.0f;
  s.least = !(m > 0.0f) ? 0u : m >= 1.0f ? 1u << 31 : (uint32_t)ceil((double)m * 2147483648.0);
  const double u = a.random[r];
  s.u = !(u > 0.0) ? 0u : u >= 1.0 ? 0x7FFFFFFFu : (uint32_t)(u * 2147483648.0);
  return s;
}

// ---------------------------------------------------------------------------------------
// A cluster of C CTAs holds a row in shared memory, a slice of consecutive tokens each, so the
// logits are read from memory once; every decision is made by all CTAs alike from what they
// exchange (integer counts and sums: the order of the atomics does not matter).
//
// Top-k first looks at the threads' own maxima, binned while the row is loaded (by level: the largest
// logit is not known yet): as many of them as k lie above some gap, so the k-th token does too (k at
// most the cluster's threads).  Where the tokens up to that gap are few, as they are for the usual k, the
// cluster's first CTA gathers them, orders them by counting and finishes the row, and the others leave:
// 22 us for 128 rows of 151,936 tokens and k = 50 (reading them takes 6), against 45 with the histogram.
//
// Otherwise the cut is found with a histogram of gaps in up to 1024 bins of 2^s levels, then one of the
// levels of the bin it falls into.  Counting every token would cost three shared-memory atomics each, most
// of them for the row's bulk far below the cut, so only tokens that can matter are counted: for top-k those
// up to the gap above, for top-p those heavier than (W - need) / V, because the tokens up to that weight
// add up to W - need at most and the prefix that reaches `need` has only heavier ones.
// What bounds it: reading and a row's chain of exchanges (some 1,500 to 2,500 cycles each) for small k;
// instructions where top-p looks at a whole row, 111 a token and 113 us for 128 such rows, 44 without any
// filter.  A single row of 151,936 tokens with top-p over 16 CTAs takes 23 us, 41,600 cycles of a CTA in one
// chain: its slice loaded 2,600, the largest logit exchanged 2,900, weights summed 2,700 and exchanged 2,400,
// the reach found 1,700, the histogram with its barrier 7,100, bins added over the cluster 5,500, the bin's
// levels 7,500, kept weights 3,900 and exchanged 1,500, the draw 3,700.  A window of exact levels around a cut estimated from a sample of the tokens saves
// the atomics, but its pass does more per token: 155 us.
// ---------------------------------------------------------------------------------------
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2 * kThreads;      // two per thread
constexpr int kMaxBins = kThreads;       // of the threads' maxima: 128 levels each, one per thread
constexpr int kList = kThreads;          // candidates that one CTA finishes alone
constexpr int kMaxCluster = 16;
constexpr int kSliceVecs = 6400;         // 51,200 tokens: a bin's 16-bit halves of weights stay in 32 bits
constexpr int kOut = 1 << 20;            // gap of a place that holds no token

struct CountSum {
  uint64_t sum;
  uint32_t count;
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t peer_u32(const void* local, int rank) {
  uint32_t at, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_at(local)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t peer_u64(const void* local, int rank) {
  uint32_t at;
  uint64_t v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_at(local)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}

struct SampleShared {
  union {
    struct {
      uint32_t count[kBins], low[kBins], high[kBins];  // gaps: tokens, their weights' lower and upper 16 bits
    };
    struct {  // of the CTA that finishes a row from its candidates
      uint64_t keys[kList], kept[kList];
    };
  };
  uint64_t added[3][kBins / 4];  // this CTA's share of the bins, of all CTAs (4 or more)
  uint32_t level[2][64];         // tokens per level of a bin: for top-k, for top-p
  uint64_t list[kList];          // this CTA's candidates: gap and token
  uint32_t most[kMaxBins];       // the threads' maxima
  uint32_t pow2[1024];
  uint64_t warp_sum[kWarps];
  uint32_t warp_count[kWarps];
  SampleRow set;
  // read by the peers
  int32_t max;
  uint32_t listed;
  uint64_t whole;
  uint64_t kept_sum;
  uint32_t ties;
  // this CTA's decisions
  int32_t bin[3];
  uint64_t below_sum[3];
  uint32_t below_count[3];
  int32_t gap;
};

template <int C>
__device__ __forceinline__ void cluster_meet() {
  if (C > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}

__device__ __forceinline__ CountSum warp_scan(CountSum s, int width) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < width; o <<= 1) {
    const uint64_t ys = __shfl_up_sync(0xffffffffu, s.sum, o);
    const uint32_t yc = __shfl_up_sync(0xffffffffu, s.count, o);
    if (lane >= o) {
      s.sum += ys;
      s.count += yc;
    }
  }
  return s;
}

// exclusive prefix over the block's threads, and the whole
__device__ __forceinline__ CountSum block_prefix(CountSum v, SampleShared& sh, CountSum* whole) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const CountSum s = warp_scan(v, 32);
  __syncthreads();
  if (lane == 31) {
    sh.warp_sum[w] = s.sum;
    sh.warp_count[w] = s.count;
  }
  __syncthreads();
  // every warp scans the warps' sums itself
  const CountSum all = warp_scan(lane < kWarps ? CountSum{sh.warp_sum[lane], sh.warp_count[lane]} : CountSum{0, 0}, kWarps);
  const uint64_t before_sum = __shfl_sync(0xffffffffu, all.sum, (w + 31) & 31);
  const uint32_t before_count = __shfl_sync(0xffffffffu, all.count, (w + 31) & 31);
  *whole = CountSum{__shfl_sync(0xffffffffu, all.sum, kWarps - 1), __shfl_sync(0xffffffffu, all.count, kWarps - 1)};
  return CountSum{(w ? before_sum : 0) + s.sum - v.sum, (w ? before_count : 0) + s.count - v.count};
}

// A row's draw from its candidates, one per thread (gap and token, n of them; they hold the k first).
template <class Weight>
__device__ __forceinline__ void draw_from_list(const llx_sample_args& a, int64_t r, uint64_t key, int n, int k, bool by_part,
                                               const SampleRow& set, Weight weight, SampleShared& sh) {
  const int tid = threadIdx.x;
  uint64_t* keys = sh.keys;
  uint64_t* kept = sh.kept;  // in order: weight and token
  keys[tid] = key;
  if (tid == 0) sh.bin[0] = k;
  __syncthreads();
  int place = 0;  // in the order of gap and index
  const uint32_t w = tid < n ? weight((int)(key >> 32)) : 0;
  if (tid < n) {
    for (int j = 0; j < n; ++j) place += keys[j] < key;
    kept[place] = (uint64_t)w << 32 | (uint32_t)key;
  }
  __syncthreads();
  const uint64_t s = tid < k ? kept[tid] >> 32 : 0;
  CountSum whole;
  const CountSum at = block_prefix(CountSum{s, 0}, sh, &whole);
  const uint64_t need = max(part_ceil(whole.sum, set.part), (uint64_t)1);
  if (by_part && at.sum < need && at.sum + s >= need) sh.bin[0] = tid + 1;
  const int heavy = __syncthreads_count(tid < n && w >= set.least);
  const int last = min(sh.bin[0], heavy);
  if (place >= last || tid >= n) return;
  uint64_t start = 0, total = 0;
  for (int j = 0; j < last; ++j) {
    const uint64_t x = kept[j];
    total += x >> 32;
    start += (uint32_t)x < (uint32_t)key ? x >> 32 : 0;
  }
  const uint64_t target = part_floor(total, set.u);
  if (start <= target && target < start + w) {
    a.token[r] = (int)(uint32_t)key;
    if (a.prob) a.prob[r] = (float)((double)w / (double)total);
  }
}

template <int C>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const llx_sample_args a, const int slice) {
  extern __shared__ __align__(16) uint4 vecs[];  // this CTA's part of the row
  __shared__ SampleShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / C;
  const int rank = (int)(blockIdx.x % C);
  for (int x = tid; x < kBins; x += kThreads) sh.count[x] = sh.low[x] = sh.high[x] = 0;
  sh.most[tid] = 0;
  if (tid < 64) sh.level[0][tid] = sh.level[1][tid] = 0;
  if (tid == 0) sh.listed = 0;
  for (int x = tid; x < 1024; x += kThreads) sh.pow2[x] = kDevPow2[x];
  pdl_trigger();
  pdl_wait();
  // The row lies in 16-byte vectors from the one that holds its first token on; this CTA has the
  // vectors [v0, v0 + nv), and of their places [lo, hi) hold tokens.
  const int V = (int)a.vocab;
  const int16_t* row = a.logits + r * a.logits_stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) >> 1);
  const int v0 = rank * slice, nv = max(0, min(slice, (skew + V + 7) / 8 - v0));
  const int lo = max(0, skew - v0 * 8), hi = min(nv * 8, skew + V - v0 * 8);
  const int16_t* from = row - skew + (int64_t)v0 * 8;
  const int64_t k = row_k(a, r);
  const bool by_k = k < V, by_part = a.top_p && a.top_p[r] < 1.0f;
  auto bin_at = [](int level) { return (level + 32768) >> 7; };
  if (by_k) __syncthreads();  // the counts are clear
  uint32_t most = 0x80008000u;  // of the thread's tokens
  for (int v = tid; v < nv; v += kThreads) {
    uint4 x;
    if (v * 8 >= lo && v * 8 + 8 <= hi) {
      x = reinterpret_cast<const uint4*>(from)[v];
    } else {
      x = make_uint4(0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u);
      int16_t* e = reinterpret_cast<int16_t*>(&x);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v * 8 + j >= lo && v * 8 + j < hi) e[j] = from[v * 8 + j];
    }
    vecs[v] = x;
    most = __vmaxs2(most, __vmaxs2(__vmaxs2(x.x, x.y), __vmaxs2(x.z, x.w)));
  }
  const int mine = max((int)(int16_t)(most & 0xffffu), (int)most >> 16);
  const bool any = tid < nv;  // every vector has a token
  if (by_k && any) atomicAdd(&sh.most[bin_at(mine)], 1u);
  // one thread works out the row's settings (doubles) while the others load
  if (tid == kThreads - 1) sh.set = sample_row(a, r);
  {
    const int m = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) sh.warp_count[warp] = (uint32_t)m;
    __syncthreads();
    if (warp == 0) {
      const int x = __reduce_max_sync(0xffffffffu, lane < kWarps ? (int)sh.warp_count[lane] : -32768);
      if (lane == 0) sh.max = x;
    }
  }
  cluster_meet<C>();
  const SampleRow set = sh.set;
  int mx = -32768;
#pragma unroll
  for (int c = 0; c < C; ++c) mx = max(mx, C > 1 ? (int)peer_u32(&sh.max, c) : sh.max);

  // the 8 gaps of a vector; places without a token get kOut
  auto gaps = [&](int v, int (&g)[8]) {
    const uint4 x = vecs[v];
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[2 * j] = mx - (int)(int16_t)(w[j] & 0xffffu);
      g[2 * j + 1] = mx - ((int)w[j] >> 16);
    }
    if (v * 8 < lo || v * 8 + 8 > hi) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v * 8 + j < lo || v * 8 + j >= hi) g[j] = kOut;
    }
  };
  // whether a vector has a token within `reach`: the largest of its places first, two at a time
  auto near = [&](int v, int reach) {
    const uint4 x = vecs[v];
    const uint32_t m = __vmaxs2(__vmaxs2(x.x, x.y), __vmaxs2(x.z, x.w));
    return mx - max((int)(int16_t)(m & 0xffffu), (int)m >> 16) <= reach;
  };
  const bool small = set.step < (1ull << 28);
  auto weight = [&](int g) {
    return small ? gap_weight<true>((uint32_t)g, set.step, sh.pow2) : gap_weight<false>((uint32_t)g, set.step, sh.pow2);
  };
  // weights first, choices after: no branches around the arithmetic
  auto weights = [&](const int (&g)[8], uint32_t (&w)[8], int limit) {
    if (small) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = gap_weight<true>((uint32_t)g[j], set.step, sh.pow2, (uint32_t)limit);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = gap_weight<false>((uint32_t)g[j], set.step, sh.pow2, (uint32_t)limit);
    }
  };
  // largest gap whose weight is at least `least` (weight(0) is): every warp tries 32 gaps a round
  auto farthest = [&](uint32_t least) {
    int l = 0;
#pragma unroll 1
    for (int width = 2048;; width >>= 5) {  // 2048, 64, 2, 1
      if (width == 0) width = 1;
      const int g = l + lane * width;
      const uint32_t ok = __ballot_sync(0xffffffffu, g < 65536 && weight(g) >= least);
      l += (__popc(ok) - 1) * width;
      if (width == 1) break;
    }
    return l;
  };

  int G = 65535;       // kept: gaps below G and `take` tokens of gap G
  int64_t take = V;
  if (by_k || by_part) {
    int reach = 65535;  // no token beyond this gap matters
    if (by_k) {
      if (k <= (int64_t)kThreads * C) {
        // bin d from the largest logit's down holds the gaps (off + 128 (d - 1), off + 128 d]
        const int top = bin_at(mx), off = (mx + 32768) & 127;
        uint32_t n = 0;
        if (tid <= top)
#pragma unroll
          for (int c = 0; c < C; ++c) n += C > 1 ? peer_u32(&sh.most[top - tid], c) : sh.most[top - tid];
        CountSum all;
        const CountSum at = block_prefix(CountSum{0, n}, sh, &all);
        if (tid == 0) sh.bin[2] = kMaxBins - 1;
        __syncthreads();
        if (at.count < k && at.count + n >= k) sh.bin[2] = tid;
        __syncthreads();
        reach = min(reach, off + 128 * sh.bin[2]);
        if (k <= kList / 2) {
          for (int v = tid; v < nv; v += kThreads) {
            if (!near(v, reach)) continue;
            int g[8];
            gaps(v, g);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (g[j] <= reach) {
                const uint32_t x = atomicAdd(&sh.listed, 1u);
                if (x < kList) sh.list[x] = (uint64_t)g[j] << 32 | (uint32_t)((v0 + v) * 8 + j - skew);
              }
          }
          cluster_meet<C>();
          uint64_t key = ~0ull;
          uint32_t n = 0;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const uint32_t m = C > 1 ? peer_u32(&sh.listed, c) : sh.listed;
            if (rank == 0 && tid >= n && tid < n + m && tid - n < kList) key = C > 1 ? peer_u64(&sh.list[tid - n], c) : sh.list[tid - n];
            n += m;
          }
          if (n <= kList) {
            if (C > 1) cluster_meet<C>();  // the first CTA has them all
            if (rank == 0) draw_from_list(a, r, key, (int)n, (int)k, by_part, set, weight, sh);
            return;
          }
        }
      }
    } else {
      uint64_t sum = 0;
      for (int v = tid; v < nv; v += kThreads) {
        int g[8];
        gaps(v, g);
        uint32_t w[8];
        weights(g, w, kOut);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += w[j];
      }
      CountSum all;
      block_prefix(CountSum{sum, 0}, sh, &all);
      if (tid == 0) sh.whole = all.sum;
      cluster_meet<C>();
      uint64_t whole = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) whole += C > 1 ? peer_u64(&sh.whole, c) : sh.whole;
      const uint64_t need = max(part_ceil(whole, set.part), (uint64_t)1);
      const uint64_t light = (whole - need) / (uint64_t)V;
      reach = farthest(light >= 0x80000000ull ? 0x80000000u : (uint32_t)light + 1u);
    }
    // ---- bins of 2^s levels ----
    int s = 0;
    while ((reach >> s) >= kBins) ++s;
    for (int v = tid; v < nv; v += kThreads) {
      if (!near(v, reach)) continue;
      int g[8];
      gaps(v, g);
      uint32_t w[8];
      if (by_part) weights(g, w, kOut);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (g[j] <= reach) {
          const int b = g[j] >> s;
          if (by_k) atomicAdd(&sh.count[b], 1u);
          if (by_part) {
            atomicAdd(&sh.low[b], w[j] & 0xffffu);
            atomicAdd(&sh.high[b], w[j] >> 16);
          }
        }
    }
    cluster_meet<C>();
    CountSum bin[2] = {{0, 0}, {0, 0}}, all;
    if constexpr (C <= 2) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int b = 2 * tid + x;
          bin[x].count += C > 1 ? peer_u32(&sh.count[b], c) : sh.count[b];
          bin[x].sum += (C > 1 ? peer_u32(&sh.low[b], c) : sh.low[b]) + ((uint64_t)(C > 1 ? peer_u32(&sh.high[b], c) : sh.high[b]) << 16);
        }
    } else {
      // every CTA adds up its share of the bins, then all read the sums: 2 x 24 KB over the cluster's
      // network where reading all of every peer's bins would be C x 12
      constexpr int kShare = kBins / C;
#pragma unroll
      for (int x = tid; x < 3 * kShare; x += kThreads) {
        const uint32_t* from = (x < kShare ? sh.count : x < 2 * kShare ? sh.low : sh.high) + rank * kShare + x % kShare;
        uint64_t n = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) n += peer_u32(from, c);
        sh.added[x / kShare][x % kShare] = n;
      }
      cluster_meet<C>();
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int b = 2 * tid + x, c = b / kShare;
        bin[x].count = (uint32_t)peer_u64(&sh.added[0][b % kShare], c);
        bin[x].sum = peer_u64(&sh.added[1][b % kShare], c) + (peer_u64(&sh.added[2][b % kShare], c) << 16);
      }
    }
    const CountSum at = block_prefix(CountSum{bin[0].sum + bin[1].sum, bin[0].count + bin[1].count}, sh, &all);
    // The cut of kind q (0: top-k by count, 1: top-p by weight) among the tokens of its bin, level by
    // level: the first level at which `enough` holds of what is below and within.
    auto cut = [&](int q, auto enough) {
      CountSum below = at;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const CountSum end{below.sum + bin[x].sum, below.count + bin[x].count};
        if (!enough(below) && enough(end)) {
          sh.bin[q] = 2 * tid + x;
          sh.below_sum[q] = below.sum;
          sh.below_count[q] = below.count;
        }
        below = end;
      }
      __syncthreads();
      const int b = sh.bin[q];
      for (int v = tid; v < nv; v += kThreads) {
        if (!near(v, ((b + 1) << s) - 1)) continue;
        int g[8];
        gaps(v, g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g[j] >> s == b) atomicAdd(&sh.level[q][g[j] - (b << s)], 1u);
      }
      cluster_meet<C>();
      if (warp == 0) {
        CountSum lv[2] = {{0, 0}, {0, 0}};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int l = 2 * lane + x;
#pragma unroll
          for (int c = 0; c < C; ++c) lv[x].count += C > 1 ? peer_u32(&sh.level[q][l], c) : sh.level[q][l];
          if (lv[x].count) lv[x].sum = (uint64_t)lv[x].count * weight((b << s) + l);
        }
        CountSum e{lv[0].sum + lv[1].sum, lv[0].count + lv[1].count};
        const CountSum own = e;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t ys = __shfl_up_sync(0xffffffffu, e.sum, o);
          const uint32_t yc = __shfl_up_sync(0xffffffffu, e.count, o);
          if (lane >= o) {
            e.sum += ys;
            e.count += yc;
          }
        }
        CountSum w{sh.below_sum[q] + e.sum - own.sum, sh.below_count[q] + e.count - own.count};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const CountSum end{w.sum + lv[x].sum, w.count + lv[x].count};
          if (!enough(w) && enough(end)) {
            sh.gap = (b << s) + 2 * lane + x;
            sh.below_sum[2] = w.sum;
            sh.below_count[2] = w.count;
          }
          w = end;
        }
      }
      __syncthreads();
    };
    uint64_t total = all.sum;
    if (by_k) {
      cut(0, [&](const CountSum& v) { return (int64_t)v.count >= k; });
      G = sh.gap;
      take = k - (int64_t)sh.below_count[2];
      total = sh.below_sum[2] + (uint64_t)take * weight(G);
    }
    if (by_part) {
      if (!by_k) {
        total = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) total += C > 1 ? peer_u64(&sh.whole, c) : sh.whole;
      }
      const uint64_t need = max(part_ceil(total, set.part), (uint64_t)1);
      __syncthreads();  // the decisions of top-k have been read
      // within the tokens of top-k the sums are those of all tokens, but for the last level
      cut(1, [&](const CountSum& v) { return v.sum >= need; });
      G = sh.gap;
      const uint32_t w = weight(G);
      take = (int64_t)((need - sh.below_sum[2] + w - 1) / w);
    }
  }
  if (weight(G) < set.least) {  // min-p cuts further up
    G = farthest(set.least);
    take = V;
  }
  // ---- kept weights in index order: a segment of the slice per warp, then the draw ----
  const uint32_t wG = weight(G);
  // a thread's vectors follow one another, an odd number of them: 16-byte reads of neighbouring threads
  // then hit different banks
  const int chunk = ((nv + kThreads - 1) / kThreads) | 1, c0 = min(nv, tid * chunk), c1 = min(nv, c0 + chunk);
  auto kept = [&](int v, int (&g)[8]) {
    CountSum t{0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = kOut;
    if (!near(v, G)) return t;
    gaps(v, g);
    uint32_t w[8];
    weights(g, w, G);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      t.sum += w[j];
      t.count += g[j] == G;
    }
    return t;
  };
  CountSum own{0, 0};
  for (int v = c0; v < c1; ++v) {
    int g[8];
    const CountSum t = kept(v, g);
    own.sum += t.sum;
    own.count += t.count;
  }
  CountSum here;  // this CTA's
  const CountSum ahead = block_prefix(own, sh, &here);
  if (tid == 0) {
    sh.kept_sum = here.sum;
    sh.ties = here.count;
  }
  cluster_meet<C>();
  CountSum before{0, 0}, all{0, 0};
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (c == rank) before = all;
    all.sum += C > 1 ? peer_u64(&sh.kept_sum, c) : sh.kept_sum;
    all.count += C > 1 ? peer_u32(&sh.ties, c) : sh.ties;
  }
  if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // nothing more is read from a peer
  before.sum += ahead.sum;
  before.count += ahead.count;
  const int64_t ties = min(take, (int64_t)all.count);
  const uint64_t total = all.sum + (uint64_t)ties * wG, target = part_floor(total, set.u);
  // running kept weight once `sum` of lesser gaps and `n` ties have gone by
  auto run_at = [&](uint64_t sum, int64_t n) { return sum + (uint64_t)min(n, ties) * wG; };
  const bool has = run_at(before.sum, before.count) <= target &&
                   target < run_at(before.sum + own.sum, (int64_t)before.count + own.count);
  const uint32_t who = __ballot_sync(0xffffffffu, has);
  if (who) {  // one thread of one CTA has the token: its vectors, one per lane (a slice has at most 13 a thread)
    const int l = __ffs(who) - 1, v = __shfl_sync(0xffffffffu, c0, l) + lane;
    CountSum w{__shfl_sync(0xffffffffu, before.sum, l), __shfl_sync(0xffffffffu, before.count, l)};
    int g[8];
    CountSum t{0, 0};
    const bool in = v < __shfl_sync(0xffffffffu, c1, l);
    if (in) t = kept(v, g);
    CountSum e = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t ys = __shfl_up_sync(0xffffffffu, e.sum, o);
      const uint32_t yc = __shfl_up_sync(0xffffffffu, e.count, o);
      if (lane >= o) {
        e.sum += ys;
        e.count += yc;
      }
    }
    w.sum += e.sum - t.sum;
    w.count += e.count - t.count;
    if (in && run_at(w.sum, w.count) <= target && target < run_at(w.sum + t.sum, (int64_t)w.count + t.count)) {
      int64_t n = w.count;
#pragma unroll 1
      for (int j = 0; j < 8; ++j) {
        const int x = mx - (int)reinterpret_cast<const int16_t*>(vecs)[v * 8 + j];
        if (v * 8 + j < lo || v * 8 + j >= hi) continue;
        const uint64_t start = run_at(w.sum, n);
        if (x < G) w.sum += weight(x);
        n += x == G;
        const uint64_t end = run_at(w.sum, n);
        if (start <= target && target < end) {
          a.token[r] = (v0 + v) * 8 + j - skew;
          if (a.prob) a.prob[r] = (float)((double)(end - start) / (double)total);
        }
      }
    }
  }
  if (C > 1) {  // no CTA leaves while a peer may still read from it
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

int64_t sample_max_vocab() { return 1ll << 18; }

template <int C>
static cudaError_t launch_sample_t(const llx_sample_args& a, int slice, cudaStream_t st) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(k_sample<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceVecs * 16);
    if (e == cudaSuccess && C > 8) e = cudaFuncSetAttribute(k_sample<C>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_release);
  }
  const dim3 grid((unsigned)(a.rows * C));
  if (C == 1) return launch_k(k_sample<C>, grid, dim3(kThreads), (size_t)slice * 16, st, a, slice);
  return launch_kc(k_sample<C>, grid, dim3(kThreads), (size_t)slice * 16, st, dim3(C, 1, 1), a, slice);
}

cudaError_t launch_sample(const llx_sample_args& a, cudaStream_t st) {
  if (a.rows == 0) return cudaSuccess;
  // Split a row until two CTAs per SM have work, as long as a CTA keeps a vector per thread; and where
  // a slice would not fit.  A CTA's fixed work is what further splits cost: 128 rows of 151,936 tokens over
  // 4 CTAs each 67 us, over 8 88; one row over 16 22.9, over 8 23.3.
  const int64_t vecs = (a.vocab + 14) / 8;  // from any alignment
  int C = 1;
  while (C < kMaxCluster && ((a.rows * C < 2 * 148 && vecs > (int64_t)C * kThreads) || vecs > (int64_t)C * kSliceVecs)) C *= 2;
  const int slice = (int)((vecs + C - 1) / C);
  switch (C) {
    case 1: return launch_sample_t<1>(a, slice, st);
    case 2: return launch_sample_t<2>(a, slice, st);
    case 4: return launch_sample_t<4>(a, slice, st);
    case 8: return launch_sample_t<8>(a, slice, st);
    default: return launch_sample_t<16>(a, slice, st);
  }
}

}  // namespace llx
