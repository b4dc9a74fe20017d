// Paged attention of prompt chunks: tiles of 128 stacked (row, head) pairs of one KV head on the
// 5th-generation tensor cores.
//
// The reference's order (maximum over all keys, then the sum of table exponentials, then the
// normalised integer weights times the values) cannot be rescaled as it goes, so a tile takes three
// passes over its keys, 128 at a time; the scores are recomputed by tcgen05.mma (kind::i8) each time:
//   pass 1  S = Q K^T into TMEM, row maxima;
//   pass 2  S again, sums of exponentials;
//   pass 3  S again, weights as two unsigned bytes into shared memory, O_hi / O_lo += P V.
// K and V rows stream page by page through a ring filled by TMA; V is the MMA's B operand as it
// lies (channels contiguous).  One thread owns 32 keys of one row of every tile, so maxima and sums
// stay in registers until a pass ends.
// Roles: warp 0 loads, warp 1 issues the MMAs, warps 4 to 19 do the softmax.
#include <atomic>

#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace llx {
namespace {

constexpr int kRows = 128, kTK = 128;
constexpr int kSoftWarps = 16, kThreads = 128 + kSoftWarps * 32;
constexpr int kStages = 5;

template <int D>
struct Smem {
  static constexpr int q = 0;
  static constexpr int ring = kRows * D;
  static constexpr int p = ring + kStages * kTK * D;          // [2][hi, lo][128][128]
  static constexpr int bytes = p + 4 * kRows * kTK + 1024;
};

// shared-memory operand of rows of D bytes, swizzled by D bytes: rows along the MMA's M or N with the
// contraction contiguous (scores), or rows along the contraction with N contiguous (values); either
// way groups of 8 rows follow one another
template <int D>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  uint64_t d = (addr >> 4) & 0x3FFFull;
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(8 * D >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)(D == 128 ? 2 : 4) << 61;  // 128-byte or 64-byte swizzle
  return d;
}
// weights (unsigned) times values (signed, N contiguous): N = D
__host__ __device__ constexpr uint32_t idesc_values(int D) {
  return (2u << 4) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t* v) {
  if constexpr (N == 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <int D, bool HIGH>
__global__ void __launch_bounds__(kThreads, 1)
    k_paged_chunk(const llx_paged_attention_args a, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const int box, const int least) {
  using L = Smem<D>;
  constexpr uint32_t kO = 2 * kTK;  // TMEM columns: S[2], O_lo, O_hi
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], s_full[2], s_free[2], p_full[2], p_free[2], o_full;
  __shared__ uint32_t tmem_s;
  __shared__ int lost, any_bad;
  __shared__ int32_t red[4][kRows];
  __shared__ unsigned long long red64[4][kRows];
  __shared__ uint16_t expi[18], expf[256];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      pa::bar_init(&full[s], 1);
      pa::bar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      pa::bar_init(&s_full[s], 1);
      pa::bar_init(&s_free[s], kSoftWarps);
      pa::bar_init(&p_full[s], kSoftWarps);
      pa::bar_init(&p_free[s], 1);
    }
    pa::bar_init(&o_full, 1);
    lost = any_bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int x = tid; x < 256; x += kThreads) expf[x] = kDevExpF[x];
  if (tid < 18) expi[tid] = tid < 16 ? kDevExpI[tid] : 0;
  pdl_trigger();
  pdl_wait();
  const int i = blockIdx.z, kvh = blockIdx.y;
  const SeqView sv = view_sequence(a, i);
  const int rep = (int)(a.n_heads / a.n_kv_heads), P = (int)a.page_size;
  const int rows = (int)min((int64_t)sv.rows, a.max_rows);
  const int64_t pairs = (int64_t)rows * rep;
  // the last rows see the most keys: their tiles start first
  const int tile = (int)((pairs + kRows - 1) / kRows) - 1 - (int)blockIdx.x;
  const int cap = key_cap(a);
  if (blockIdx.x == 0 && kvh == 0 && tid == 0 && pairs >= least) {
    int code = sv.code;
    if (sv.rows > a.max_rows || sv.len > cap) code |= LLX_STATUS_BAD_BOUND;
    if (!code && sv.len < sv.rows) code = LLX_STATUS_BAD_POSITION;
    if (code) raise_status(a.status, code);
  }
  if (tile < 0 || pairs < least) return;
  const int g0 = tile * kRows, nr = (int)min((int64_t)kRows, pairs - g0);
  auto keys_of = [&](int n) {
    const int64_t t = (int64_t)sv.len - sv.rows + (g0 + n) / rep + 1;
    return (int)(t < 0 ? 0 : t > cap ? cap : t);
  };
  const int T = keys_of(nr - 1), tiles = (T + kTK - 1) / kTK;
  const int32_t* pages = a.table + (sv.slot < 0 ? 0 : sv.slot) * a.table_stride;
  unsigned char* base = raw + ((1024 - (pa::s32(raw) & 1023)) & 1023);

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pa::s32(&tmem_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  for (int x = tid; x < (T + P - 1) / P; x += kThreads) {
    const int id = pages[x];
    if (id < 0 || id >= a.n_pages) any_bad = 1;
  }
  // queries as the scores' A operand; rows past the last pair are zero
  for (int x = tid; x < kRows * D / 16; x += kThreads) {
    const int n = x / (D / 16), c = x % (D / 16);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n < nr)
      v = *reinterpret_cast<const uint4*>(a.q8 + (int64_t)(sv.first + (g0 + n) / rep) * a.q8_stride +
                                          (int64_t)(kvh * rep + (g0 + n) % rep) * D + c * 16);
    *reinterpret_cast<uint4*>(base + L::q + pa::tile_at<D>(n, c)) = v;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_s;
  if (tid == 0 && any_bad) raise_status(a.status, LLX_STATUS_BAD_PAGE);

  if (warp == 0) {
    // K of passes 1 and 2, then K 0, K 1, V 0, K 2, V 1, ..., V last
    for (int it = 0; it < 4 * tiles; ++it) {
      const int s = it % kStages, x = it - 2 * tiles;
      bool is_v = false;
      int t = it < tiles ? it : it - tiles;
      if (x >= 0) {
        is_v = x == 2 * tiles - 1 || (x > 0 && x % 2 == 0);
        t = x == 0 ? 0 : x == 2 * tiles - 1 ? tiles - 1 : is_v ? x / 2 - 1 : (x + 1) / 2;
      }
      if (it >= kStages && !pa::bar_wait(&empty[s], (uint32_t)(it / kStages - 1) & 1, &lost)) break;
      const int boxes = (min(kTK, T - t * kTK) + box - 1) / box;
      if (lane == 0) pa::bar_expect(&full[s], (uint32_t)(boxes * box * D));
      __syncwarp();
      if (lane < boxes) {
        const int key = t * kTK + lane * box;
        const int id = pages[key / P];  // absent: page 0 is read in its place, its keys are never used
        pa::load_rows(base + L::ring + s * kTK * D + lane * box * D, is_v ? &mv : &mk, &full[s], kvh * P + key % P,
                      id < 0 || id >= a.n_pages ? 0 : id);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int c = 0, n = 0;  // stages and score tiles consumed
      const bool wide = a.prob_bits > 8;
      auto scores = [&]() {
        const int s = c % kStages;
        bool ok = pa::bar_wait(&full[s], (uint32_t)(c / kStages) & 1, &lost);
        if (n >= 2) ok = pa::bar_wait(&s_free[n & 1], (uint32_t)((n >> 1) - 1) & 1, &lost) && ok;
        if (!ok) return false;
        tc::tc_fence_after();
        const uint32_t q = pa::s32(base + L::q), k = pa::s32(base + L::ring + s * kTK * D);
#pragma unroll
        for (int kb = 0; kb < D / 32; ++kb)
          tc::mma_i8(tmem + (n & 1) * kTK, operand<D>(q + kb * 32), operand<D>(k + kb * 32), tc::idesc_i8(kTK), kb > 0);
        tc::mma_commit(&empty[s]);
        tc::mma_commit(&s_full[n & 1]);
        ++c;
        ++n;
        return true;
      };
      auto values = [&](int t) {
        const int s = c % kStages;
        bool ok = pa::bar_wait(&full[s], (uint32_t)(c / kStages) & 1, &lost);
        ok = pa::bar_wait(&p_full[t & 1], (uint32_t)(t >> 1) & 1, &lost) && ok;
        if (!ok) return false;
        tc::tc_fence_after();
        const uint32_t v = pa::s32(base + L::ring + s * kTK * D);
        const uint32_t p = pa::s32(base + L::p + (t & 1) * 2 * kRows * kTK);
        const int steps = (min(kTK, T - t * kTK) + 31) / 32;
        for (int kb = 0; kb < steps; ++kb) {
          const uint64_t b = operand<D>(v + kb * 32 * D);
          tc::mma_i8(tmem + kO, operand<128>(p + kRows * kTK + kb * 32), b, idesc_values(D), t > 0 || kb > 0);
          if (wide) tc::mma_i8(tmem + kO + D, operand<128>(p + kb * 32), b, idesc_values(D), t > 0 || kb > 0);
        }
        tc::mma_commit(&empty[s]);
        tc::mma_commit(&p_free[t & 1]);
        ++c;
        return true;
      };
      bool ok = true;
      for (int t = 0; t < 2 * tiles && ok; ++t) ok = scores();
      if (ok && tiles) ok = scores();
      for (int t = 1; t < tiles && ok; ++t) ok = scores() && values(t - 1);
      if (ok && tiles) ok = values(tiles - 1);
      if (ok && tiles) tc::mma_commit(&o_full);
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, part = (warp - 4) >> 2;
    const int n = quad * 32 + lane;  // row of the tile
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int Tn = n < nr ? keys_of(n) : 0;
    int st = 0;  // score tiles seen
    // the thread's 32 scores of the next tile, and which of its keys the row sees
    auto take = [&](int t, uint32_t (&v)[32]) {
      pa::bar_wait(&s_full[st & 1], (uint32_t)(st >> 1) & 1, &lost);
      tc::tc_fence_after();
      tmem_load<32>(tmem + lanes + (st & 1) * kTK + part * 32, v);
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) pa::bar_arrive(&s_free[st & 1]);
      ++st;
      const int k0 = t * kTK + part * 32, left = Tn - k0;
      uint32_t m = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
      if (any_bad)
        for (int e = 0; e < 32; e += 16)
          if (k0 + e < T) {
            const int id = pages[(k0 + e) / P];
            if (id < 0 || id >= a.n_pages) m &= ~(0xffffu << e);
          }
      return m;
    };
    uint32_t v[32];
    int mx = INT_MIN;
    for (int t = 0; t < tiles; ++t) {
      const uint32_t m = take(t, v);
      if (__all_sync(0xffffffffu, m == 0xffffffffu)) {
#pragma unroll
        for (int e = 0; e < 32; ++e) mx = max(mx, (int)v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) mx = max(mx, (m >> e) & 1u ? (int)v[e] : INT_MIN);
      }
    }
    red[part][n] = mx;
    pa::named_sync(1, kSoftWarps * 32);
    mx = max(max(red[0][n], red[1][n]), max(red[2][n], red[3][n]));
    const GapScale gs = gap_scale(a.Ms, a.Ss);
    unsigned long long sum = 0;
    for (int t = 0; t < tiles; ++t) {
      const uint32_t m = take(t, v);
      uint32_t s = 0;
      if (__all_sync(0xffffffffu, m == 0xffffffffu)) {
#pragma unroll
        for (int e = 0; e < 32; ++e) s += table_exp(gap_index<HIGH>((uint32_t)mx - v[e], gs), expi, expf);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          s += (m >> e) & 1u ? table_exp(gap_index<HIGH>((uint32_t)mx - v[e], gs), expi, expf) : 0u;
      }
      sum += s;
    }
    red64[part][n] = sum;
    pa::named_sync(1, kSoftWarps * 32);
    sum = red64[0][n] + red64[1][n] + red64[2][n] + red64[3][n];
    const uint32_t inv = sum > 0x80000000ull ? 0u : 0x80000000u / (sum ? (uint32_t)sum : 1u);
    const int psh = 31 - (int)a.prob_bits;
    const uint32_t prnd = 1u << (psh - 1), pmax = (1u << a.prob_bits) - 1u;
    const bool wide = a.prob_bits > 8;
    for (int t = 0; t < tiles; ++t) {
      const uint32_t m = take(t, v);
      const bool whole = __all_sync(0xffffffffu, m == 0xffffffffu);
      if (t >= 2) pa::bar_wait(&p_free[t & 1], (uint32_t)((t >> 1) - 1) & 1, &lost);
      unsigned char* p = base + L::p + (t & 1) * 2 * kRows * kTK;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t pn[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int x = h * 16 + w * 4 + e;
            uint32_t pr = table_exp(gap_index<HIGH>((uint32_t)mx - v[x], gs), expi, expf);
            if (!whole && !((m >> x) & 1u)) pr = 0;
            pn[e] = min((pr * inv + prnd) >> psh, pmax);  // pr <= sum: the product is at most 2^31
          }
          const uint32_t p01 = __byte_perm(pn[0], pn[1], 0x5410), p23 = __byte_perm(pn[2], pn[3], 0x5410);
          lo[w] = __byte_perm(p01, p23, 0x6420);
          hi[w] = __byte_perm(p01, p23, 0x7531);
        }
        const uint32_t at = pa::tile_at<128>(n, part * 2 + h);
        *reinterpret_cast<uint4*>(p + kRows * kTK + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (wide) *reinterpret_cast<uint4*>(p + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) pa::bar_arrive(&p_full[t & 1]);
    }
    // ---- outputs: D / 4 channels a thread ----
    constexpr int W = D / 4;
    uint32_t lo[W], hi[W];
#pragma unroll
    for (int e = 0; e < W; ++e) lo[e] = hi[e] = 0;
    if (tiles) {
      pa::bar_wait(&o_full, 0, &lost);
      tc::tc_fence_after();
      tmem_load<W>(tmem + lanes + kO + part * W, lo);
      if (wide) tmem_load<W>(tmem + lanes + kO + D + part * W, hi);
    }
    if (n < nr) {
      int8_t* dst = a.out + (int64_t)(sv.first + (g0 + n) / rep) * a.out_stride + (int64_t)(kvh * rep + (g0 + n) % rep) * D +
                    part * W;
#pragma unroll
      for (int x = 0; x < W; x += 16) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          int64_t o = (int64_t)(int32_t)hi[x + e] * 256 + (int32_t)lo[x + e];
          if (wide) o = rshr(o, 7);
          w[e >> 2] |= ((uint32_t)sat8(mulshift(o, a.Mo, (int)a.So)) & 255u) << (8 * (e & 3));
        }
        *reinterpret_cast<uint4*>(dst + x) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    tc::tc_fence_before();
  }
  __syncthreads();
  if (lost && tid == 0) raise_status(a.status, LLX_STATUS_LOST);
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int D, bool HIGH>
cudaError_t launch_chunk_t(const llx_paged_attention_args& a, int64_t least, cudaStream_t st) {
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(k_paged_chunk<D, HIGH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::bytes);
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_release);
  }
  CUtensorMap mk, mv;
  const int box = a.page_size < kTK ? (int)a.page_size : kTK;
  e = make_page_map(&mk, a.k_pages, a, box);
  if (e == cudaSuccess) e = make_page_map(&mv, a.v_pages, a, box);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (a.max_rows * (a.n_heads / a.n_kv_heads) + kRows - 1) / kRows;
  const dim3 grid((unsigned)tiles, (unsigned)a.n_kv_heads, (unsigned)a.n_seqs);
  return launch_k(k_paged_chunk<D, HIGH>, grid, dim3(kThreads), Smem<D>::bytes, st, a, mk, mv, box, (int)least);
}

}  // namespace

bool paged_chunk_fits(const llx_paged_attention_args& a) {
  return (a.head_dim == 64 || a.head_dim == 128) && a.n_seqs <= 65535;
}

cudaError_t launch_paged_chunk(const llx_paged_attention_args& a, int64_t least, cudaStream_t st) {
  if (a.head_dim == 128) return a.Ss >= 33 ? launch_chunk_t<128, true>(a, least, st) : launch_chunk_t<128, false>(a, least, st);
  return a.Ss >= 33 ? launch_chunk_t<64, true>(a, least, st) : launch_chunk_t<64, false>(a, least, st);
}

}  // namespace llx
