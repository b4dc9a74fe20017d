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

__device__ __forceinline__ uint32_t gap_weight(uint32_t g, uint64_t step, const uint32_t* pow2) {
  const uint64_t e = (g * step) >> 12;
  const uint64_t n = e >> 20;
  if (n >= 32) return 0;
  const uint32_t b = pow2[(uint32_t)(e >> 10) & 1023u];
  return (b - __umulhi(b, ((uint32_t)e & 1023u) * 2839u)) >> (uint32_t)n;
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
  int64_t k;       // tokens top-k keeps
  uint32_t part;   // top-p in units of 2^-31
  bool by_part;
  uint32_t least;  // min-p's smallest weight
  uint32_t u;      // random number in units of 2^-31
};

__device__ __forceinline__ SampleRow sample_row(const llx_sample_args& a, int64_t r) {
  SampleRow s;
  const float temp = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  // log2(e) 2^(32 + exponent): a power of two times the double nearest to log2(e)
  const double unit = scalbn(1.4426950408889634, (int)(32 + a.exponent));
  const double q = greedy ? 0.0 : rint(unit / (double)temp);
  s.step = q >= 140737488355328.0 ? 1ull << 47 : (uint64_t)q;
  const int k = a.top_k ? a.top_k[r] : 0;
  s.k = greedy ? 1 : (k <= 0 || k > a.vocab ? a.vocab : k);
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  s.by_part = p < 1.0f;
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
// The cut is found with a histogram of gaps in up to 1024 bins of 2^s levels, then one of the levels
// of the bin it falls into.  Counting every token would cost three shared-memory atomics each, most of
// them for the row's bulk far below the cut, so only tokens that can matter are counted:
//   top-k  as many of the threads' own maxima as k lie above some gap, so the k-th token does too
//          (k at most the cluster's threads);
//   top-p  tokens of weight at most (W - need) / V add up to W - need at most, so the prefix that
//          reaches `need` has only heavier ones.
// ---------------------------------------------------------------------------------------
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2 * kThreads;      // two per thread
constexpr int kMaxCluster = 8;
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
  uint32_t count[kBins], low[kBins], high[kBins];  // gaps: tokens, their weights' lower and upper 16 bits
  uint32_t first[kBins];                           // gaps of the threads' maxima
  uint32_t level[2][64];                           // tokens per level of a bin: for top-k, for top-p
  uint32_t pow2[1024];
  uint64_t warp_sum[kWarps];
  uint32_t warp_count[kWarps];
  // read by the peers
  int32_t max;
  uint64_t whole;
  uint64_t kept;
  uint32_t ties;
  // this CTA's decisions
  int32_t bin[3];
  uint64_t below_sum[3];
  uint32_t below_count[3];
  int32_t gap;
  int64_t take;
};

__device__ __forceinline__ void cluster_meet(int C) {
  if (C > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}

// exclusive prefix over the block's threads, and the whole
__device__ __forceinline__ CountSum block_prefix(CountSum v, SampleShared& sh, CountSum* whole) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  CountSum s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t ys = __shfl_up_sync(0xffffffffu, s.sum, o);
    const uint32_t yc = __shfl_up_sync(0xffffffffu, s.count, o);
    if (lane >= o) {
      s.sum += ys;
      s.count += yc;
    }
  }
  __syncthreads();
  if (lane == 31) {
    sh.warp_sum[w] = s.sum;
    sh.warp_count[w] = s.count;
  }
  __syncthreads();
  CountSum before{0, 0}, all{0, 0};
#pragma unroll
  for (int x = 0; x < kWarps; ++x) {
    if (x == w) before = all;
    all.sum += sh.warp_sum[x];
    all.count += sh.warp_count[x];
  }
  *whole = all;
  return CountSum{before.sum + s.sum - v.sum, before.count + s.count - v.count};
}

__global__ void __launch_bounds__(kThreads, 2) k_sample(const llx_sample_args a, const int C, const int slice) {
  extern __shared__ __align__(16) uint4 vecs[];  // this CTA's part of the row
  __shared__ SampleShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / C;
  const int rank = (int)(blockIdx.x % C);
  for (int x = tid; x < kBins; x += kThreads) sh.count[x] = sh.low[x] = sh.high[x] = sh.first[x] = 0;
  for (int x = tid; x < 1024; x += kThreads) sh.pow2[x] = kDevPow2[x];
  if (tid < 64) sh.level[0][tid] = sh.level[1][tid] = 0;
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
  int mine = -32768;
  bool any = false;
  for (int v = tid; v < nv; v += kThreads) {
    uint4 x;
    int16_t* e = reinterpret_cast<int16_t*>(&x);
    if (v * 8 >= lo && v * 8 + 8 <= hi) {
      x = reinterpret_cast<const uint4*>(from)[v];
#pragma unroll
      for (int j = 0; j < 8; ++j) mine = max(mine, (int)e[j]);
      any = true;
    } else {
      x = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v * 8 + j >= lo && v * 8 + j < hi) {
          e[j] = from[v * 8 + j];
          mine = max(mine, (int)e[j]);
          any = true;
        }
    }
    vecs[v] = x;
  }
  const SampleRow set = sample_row(a, r);
  {
    const int m = __reduce_max_sync(0xffffffffu, any ? mine : INT_MIN);
    if (lane == 0) sh.warp_count[warp] = (uint32_t)m;
    __syncthreads();
    if (tid == 0) {
      int x = INT_MIN;
      for (int w = 0; w < kWarps; ++w) x = max(x, (int)sh.warp_count[w]);
      sh.max = x;
    }
  }
  cluster_meet(C);
  int mx = INT_MIN;
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
  auto weight = [&](int g) { return gap_weight((uint32_t)g, set.step, sh.pow2); };
  auto farthest = [&](uint32_t least) {  // largest gap whose weight is at least `least` (weight(0) is)
    int l = 0, h = 65536;
    while (h - l > 1) {
      const int mid = (l + h) >> 1;
      if (weight(mid) >= least)
        l = mid;
      else
        h = mid;
    }
    return l;
  };

  const bool by_k = set.k < V;
  int G = 65535;       // kept: gaps below G and `take` tokens of gap G
  int64_t take = V;
  if (by_k || set.by_part) {
    int reach = 65535;  // no token beyond this gap matters
    if (by_k) {
      if (set.k <= (int64_t)kThreads * C) {
        if (any) atomicAdd(&sh.first[min((mx - mine) >> 6, kBins - 1)], 1u);
        cluster_meet(C);
        uint32_t n0 = 0, n1 = 0;
        for (int c = 0; c < C; ++c) {
          n0 += C > 1 ? peer_u32(&sh.first[2 * tid], c) : sh.first[2 * tid];
          n1 += C > 1 ? peer_u32(&sh.first[2 * tid + 1], c) : sh.first[2 * tid + 1];
        }
        CountSum all;
        const CountSum at = block_prefix(CountSum{0, n0 + n1}, sh, &all);
        if (tid == 0) sh.bin[2] = kBins - 1;
        __syncthreads();
        if (at.count < set.k && at.count + n0 + n1 >= set.k) sh.bin[2] = at.count + n0 >= set.k ? 2 * tid : 2 * tid + 1;
        __syncthreads();
        if (sh.bin[2] < kBins - 1) reach = sh.bin[2] * 64 + 63;
      }
    } else {
      uint64_t sum = 0;
      for (int v = tid; v < nv; v += kThreads) {
        int g[8];
        gaps(v, g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g[j] != kOut) sum += weight(g[j]);
      }
      CountSum all;
      block_prefix(CountSum{sum, 0}, sh, &all);
      if (tid == 0) sh.whole = all.sum;
      cluster_meet(C);
      uint64_t whole = 0;
      for (int c = 0; c < C; ++c) whole += C > 1 ? peer_u64(&sh.whole, c) : sh.whole;
      const uint64_t need = max(part_ceil(whole, set.part), (uint64_t)1);
      const uint64_t light = (whole - need) / (uint64_t)V;
      reach = farthest(light >= 0x80000000ull ? 0x80000000u : (uint32_t)light + 1u);
    }
    // ---- bins of 2^s levels ----
    int s = 0;
    while ((reach >> s) >= kBins) ++s;
    for (int v = tid; v < nv; v += kThreads) {
      int g[8];
      gaps(v, g);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (g[j] <= reach) {
          const int b = g[j] >> s;
          atomicAdd(&sh.count[b], 1u);
          if (set.by_part) {
            const uint32_t w = weight(g[j]);
            atomicAdd(&sh.low[b], w & 0xffffu);
            atomicAdd(&sh.high[b], w >> 16);
          }
        }
    }
    cluster_meet(C);
    CountSum bin[2] = {{0, 0}, {0, 0}}, all;
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int b = 2 * tid + x;
        bin[x].count += C > 1 ? peer_u32(&sh.count[b], c) : sh.count[b];
        if (set.by_part)
          bin[x].sum += (C > 1 ? peer_u32(&sh.low[b], c) : sh.low[b]) + ((uint64_t)(C > 1 ? peer_u32(&sh.high[b], c) : sh.high[b]) << 16);
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
        int g[8];
        gaps(v, g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (g[j] >> s == b) atomicAdd(&sh.level[q][g[j] - (b << s)], 1u);
      }
      cluster_meet(C);
      if (warp == 0) {
        CountSum lv[2] = {{0, 0}, {0, 0}};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int l = 2 * lane + x;
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
      cut(0, [&](const CountSum& v) { return (int64_t)v.count >= set.k; });
      G = sh.gap;
      take = set.k - (int64_t)sh.below_count[2];
      total = sh.below_sum[2] + (uint64_t)take * weight(G);
    }
    if (set.by_part) {
      if (!by_k) {
        total = 0;
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
  const int seg = (nv + kWarps - 1) / kWarps, s0 = min(nv, warp * seg), s1 = min(nv, s0 + seg);
  auto kept = [&](int v, int (&g)[8]) {
    CountSum t{0, 0};
    if (v < s1) gaps(v, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (v >= s1) g[j] = kOut;
      if (g[j] < G) t.sum += weight(g[j]);
      t.count += g[j] == G;
    }
    return t;
  };
  CountSum own{0, 0};
  for (int v = s0 + lane; v - lane < s1; v += 32) {
    int g[8];
    const CountSum t = kept(v, g);
    own.sum += t.sum;
    own.count += t.count;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    own.sum += __shfl_xor_sync(0xffffffffu, own.sum, o);
    own.count += __shfl_xor_sync(0xffffffffu, own.count, o);
  }
  __syncthreads();
  if (lane == 0) {
    sh.warp_sum[warp] = own.sum;
    sh.warp_count[warp] = own.count;
  }
  __syncthreads();
  if (tid == 0) {
    uint64_t x = 0;
    uint32_t n = 0;
    for (int w = 0; w < kWarps; ++w) {
      x += sh.warp_sum[w];
      n += sh.warp_count[w];
    }
    sh.kept = x;
    sh.ties = n;
  }
  cluster_meet(C);
  CountSum before{0, 0}, all{0, 0};
  for (int c = 0; c < C; ++c) {
    if (c == rank) before = all;
    all.sum += C > 1 ? peer_u64(&sh.kept, c) : sh.kept;
    all.count += C > 1 ? peer_u32(&sh.ties, c) : sh.ties;
  }
  for (int w = 0; w < warp; ++w) {
    before.sum += sh.warp_sum[w];
    before.count += sh.warp_count[w];
  }
  const int64_t ties = min(take, (int64_t)all.count);
  const uint64_t total = all.sum + (uint64_t)ties * wG, target = part_floor(total, set.u);
  // running kept weight once `sum` of lesser gaps and `n` ties have gone by
  auto run_at = [&](uint64_t sum, int64_t n) { return sum + (uint64_t)min(n, ties) * wG; };
  const uint64_t first = run_at(before.sum, before.count), last = run_at(before.sum + own.sum, (int64_t)before.count + own.count);
  if (first <= target && target < last) {  // one warp of one CTA: its segment has the token
    for (int v = s0 + lane; v - lane < s1; v += 32) {
      int g[8];
      const CountSum t = kept(v, g);
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
      uint64_t sum = before.sum + e.sum - t.sum;
      int64_t n = (int64_t)before.count + e.count - t.count;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint64_t start = run_at(sum, n);
        if (g[j] < G) sum += weight(g[j]);
        n += g[j] == G;
        const uint64_t end = run_at(sum, n);
        if (start <= target && target < end) {
          a.token[r] = (v0 + v) * 8 + j - skew;
          if (a.prob) a.prob[r] = (float)((double)(end - start) / (double)total);
        }
      }
      before.sum += __shfl_sync(0xffffffffu, e.sum, 31);
      before.count += __shfl_sync(0xffffffffu, e.count, 31);
    }
  }
  if (C > 1) {  // no CTA leaves while a peer may still read from it
    __syncwarp();
    cluster_meet(C);
  }
}

int64_t sample_max_vocab() { return 1ll << 18; }

cudaError_t launch_sample(const llx_sample_args& a, cudaStream_t st) {
  if (a.rows == 0) return cudaSuccess;
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(k_sample, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceVecs * 16);
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_release);
  }
  // Split a row until two CTAs per SM have work, as long as a CTA keeps a vector per thread; and where
  // a slice would not fit.
  const int64_t vecs = (a.vocab + 14) / 8;  // from any alignment
  int C = 1;
  while (C < kMaxCluster && ((a.rows * C < 2 * 148 && vecs > (int64_t)C * kThreads) || vecs > (int64_t)C * kSliceVecs)) C *= 2;
  const int slice = (int)((vecs + C - 1) / C);
  const dim3 grid((unsigned)(a.rows * C));
  if (C == 1) return launch_k(k_sample, grid, dim3(kThreads), (size_t)slice * 16, st, a, C, slice);
  return launch_kc(k_sample, grid, dim3(kThreads), (size_t)slice * 16, st, dim3(C, 1, 1), a, C, slice);
}

}  // namespace llx
