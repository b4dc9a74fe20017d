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

#include <cmath>
#include <cstdint>

#include "device_luts.h"
#include "launch.cuh"
#include "paged.h"

namespace llx {

constexpr int kSampleThreads = 1024;

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

struct CountSum {
  uint64_t sum;
  uint32_t count;
};

__device__ __forceinline__ CountSum reduce_count_sum(CountSum v, CountSum* scratch) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.sum += __shfl_xor_sync(0xffffffffu, v.sum, o);
    v.count += __shfl_xor_sync(0xffffffffu, v.count, o);
  }
  __syncthreads();
  if (lane == 0) scratch[w] = v;
  __syncthreads();
  CountSum t = scratch[0];
  for (int i = 1; i < kSampleThreads / 32; ++i) {
    t.sum += scratch[i].sum;
    t.count += scratch[i].count;
  }
  return t;
}

// One block per row; the cut is found by bisecting the gap.
__global__ void __launch_bounds__(kSampleThreads) k_sample(const llx_sample_args a) {
  pdl_trigger();
  pdl_wait();
  __shared__ uint32_t pow2[1024];
  __shared__ CountSum scratch[kSampleThreads / 32];
  __shared__ int found;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int V = (int)a.vocab;
  const int16_t* x = a.logits + r * a.logits_stride;
  pow2[tid] = kDevPow2[tid];
  const SampleRow row = sample_row(a, r);
  int mx = -32768;
  for (int i = tid; i < V; i += kSampleThreads) mx = max(mx, (int)x[i]);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((tid & 31) == 0) scratch[tid >> 5].count = (uint32_t)(mx + 32768);
  __syncthreads();
  for (int i = 0; i < kSampleThreads / 32; ++i) mx = max(mx, (int)scratch[i].count - 32768);
  __syncthreads();
  auto upto = [&](int G) {  // tokens of gap <= G
    CountSum v{0, 0};
    for (int i = tid; i < V; i += kSampleThreads) {
      const int g = mx - x[i];
      if (g <= G) {
        v.sum += gap_weight(g, row.step, pow2);
        v.count++;
      }
    }
    return reduce_count_sum(v, scratch);
  };
  // top-k: smallest G with at least k tokens of gap <= G
  int lo = -1, hi = 65535;
  CountSum below{0, 0};  // of gap <= lo
  auto bisect = [&](auto enough) {
    lo = -1;
    below = CountSum{0, 0};
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      const CountSum v = upto(mid);
      if (enough(v)) {
        hi = mid;
      } else {
        lo = mid;
        below = v;
      }
    }
  };
  bisect([&](const CountSum& v) { return (int64_t)v.count >= row.k; });
  int G = hi;
  int64_t c = row.k - below.count;
  uint64_t total = below.sum + (uint64_t)c * gap_weight(G, row.step, pow2);
  if (row.by_part) {
    const uint64_t need = max(part_ceil(total, row.part), (uint64_t)1);
    // within the tokens of top-k the sums are those of all tokens, but for the last gap
    bisect([&](const CountSum& v) { return v.sum >= need; });
    const uint32_t w = gap_weight(hi, row.step, pow2);
    const int64_t more = (int64_t)((need - below.sum + w - 1) / w);
    if (hi < G || more < c) c = more;
    G = hi;
  }
  if (gap_weight(G, row.step, pow2) < row.least) {  // min-p cuts further up
    int l = 0, h = G;                               // weight(l) >= least > weight(h)
    while (h - l > 1) {
      const int mid = (l + h) >> 1;
      if (gap_weight(mid, row.step, pow2) >= row.least)
        l = mid;
      else
        h = mid;
    }
    G = l;
    c = V;
  }
  // kept weights in index order: rounds of one token a thread, a scan in each
  __syncthreads();
  const uint32_t wG = gap_weight(G, row.step, pow2);
  const CountSum less = G > 0 ? upto(G - 1) : CountSum{0, 0};
  const CountSum incl = upto(G);
  const int64_t ties = min(c, (int64_t)(incl.count - less.count));
  total = less.sum + (uint64_t)ties * wG;
  const uint64_t target = part_floor(total, row.u);
  if (tid == 0) found = -1;
  uint64_t run = 0;
  int64_t seen = 0;
  const int lane = tid & 31, warp = tid >> 5;
  for (int i0 = 0; i0 < V; i0 += kSampleThreads) {
    const int i = i0 + tid;
    const int g = i < V ? mx - x[i] : 65536;
    CountSum v{g < G ? gap_weight(g, row.step, pow2) : 0u, g == G ? 1u : 0u};
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
    const bool stop = found >= 0;  // set between the second barrier of a round and the first of the next
    if (lane == 31) scratch[warp] = s;
    __syncthreads();
    if (stop) break;
    CountSum before{run, (uint32_t)seen};
    for (int w = 0; w < kSampleThreads / 32; ++w) {
      if (w < warp) {
        before.sum += scratch[w].sum;
        before.count += scratch[w].count;
      }
      run += scratch[w].sum;
      seen += scratch[w].count;
    }
    const int64_t t1 = (int64_t)before.count + s.count, t0 = t1 - v.count;
    const uint64_t end = before.sum + s.sum + (uint64_t)min(t1, ties) * wG;
    const uint64_t start = before.sum + s.sum - v.sum + (uint64_t)min(t0, ties) * wG;
    if (start <= target && target < end) {
      found = i;
      a.token[r] = i;
      if (a.prob) a.prob[r] = (float)((double)(end - start) / (double)total);
    }
  }
}

int64_t sample_max_vocab() { return 1ll << 18; }

cudaError_t launch_sample(const llx_sample_args& a, cudaStream_t st) {
  if (a.rows == 0) return cudaSuccess;
  return launch_k(k_sample, dim3((unsigned)a.rows), dim3(kSampleThreads), 0, st, a);
}

}  // namespace llx
