// Paged attention of few query rows per sequence (decode steps, a handful of draft tokens).
//
// A cluster of C CTAs serves one (sequence, KV head, group of up to 8 stacked (row, head) pairs);
// each CTA takes a slice of the keys.  Two warps stream the slice's K rows, then its V rows, page by page
// through a ring of TMA-filled stages (one warp: 84 us and 112 for the launches below); eight warps consume
// them, so every byte of the cache is read once:
//   scores  S^T (16 keys x 8 pairs) = K (16 x 32) Q^T per int8 MMA, kept in shared memory;
//   maxima  of the slices meet in every CTA of the cluster (the reference's global maximum);
//   table exponentials in place, and their sums meet the same way;
//   values  O^T (16 channels x 8 pairs) += V^T (16 x 32 keys) P^T with the weights normalised on
//           the way into the MMA as two unsigned bytes, O = 256 hi + lo;
//   partial outputs are added by the CTA that finishes them, 1/C of the outputs each.
// Integer maxima and sums: any split gives the same bits.
//
// Bytes bound it.  64 sequences of 1500 to 4200 keys, 8 KV heads of 128: 80.6 us for 361 MB, 4.5 TB/s,
// 0.68 of the copy rate; what is missing are the phases of a CTA that its neighbour on the SM does not
// cover (1.7 waves of two CTAs an SM).  Two sequences of 64k keys: 103 us for 255 MB, 2.5 TB/s: a CTA
// then holds its slice's scores (16 KB a thousand keys at four pairs) next to its ring and has its SM to
// itself, the 16 clusters of 7 to 10 CTAs do not all fit at once, and a wave's exchanges have nothing to
// hide behind.
#include <atomic>
#include <mutex>

#include "paged_attn.cuh"

namespace llx {
namespace {

constexpr int kWarps = 8, kConsumers = kWarps * 32, kLoaders = 2, kThreads = kConsumers + 32 * kLoaders;
constexpr int kPairs = 8;                        // stacked (row, head) pairs per CTA
constexpr int kTK = 128;                         // keys per stage
constexpr int kMaxCluster = 16;
constexpr size_t kSmemMost = 220 * 1024;         // of a CTA
constexpr size_t kStatic = 5 * 1024;             // of it, static arrays
// dynamic shared memory with which that many CTAs fit on an SM (1 KB of each is the system's)
constexpr size_t kSmemAt[4] = {0, kSmemMost - kStatic, 107 * 1024, 69 * 1024};
constexpr int kMaxRing = 6;  // stages
constexpr int kOrdered = 512;  // sequences whose order a block works out

// row stride of the scores in words, = 8 mod 32: a warp's 8-byte reads of 4 pairs x 8 keys and its
// stores hit different banks
__host__ __device__ constexpr int score_stride(int cap) { return (cap + 31) / 32 * 32 + 8; }

struct DecodeShape {
  int cluster, cap, box;  // CTAs per cluster, keys per slice (multiple of 64), rows per TMA box
  int nr;                 // score rows held
  int ring;               // stages
};

template <int D>
__host__ __device__ inline size_t decode_smem(int nr, int cap, int P, int ring) {
  return 1024 + (size_t)ring * kTK * D + (size_t)nr * score_stride(cap) * 4 + (size_t)(2 * nr * D + kMaxCluster) * 4 +
         (size_t)(cap / P + 2) * 4;
}

template <int D, bool HIGH>
__global__ void __launch_bounds__(kThreads) k_paged_decode(const llx_paged_attention_args a, const __grid_constant__ CUtensorMap mk,
                                                           const __grid_constant__ CUtensorMap mv, const DecodeShape shape,
                                                           const bool ordered) {
  constexpr int KB = D / 32, MB = D / 16;
  const int S = shape.ring;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t full[kMaxRing], empty[kMaxRing], met[3];
  __shared__ int lost, any_bad, chosen;
  __shared__ int lens[kOrdered];
  __shared__ uint32_t xmax[kMaxCluster * kPairs], xsum[kMaxCluster * kPairs], wred[kWarps * kPairs], gather[kPairs];
  __shared__ uint16_t expi[18], expf[256];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = shape.cluster;
  const uint32_t rank = C > 1 ? pa::cluster_rank() : 0;
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      pa::bar_init(&full[s], 1);
      pa::bar_init(&empty[s], kWarps);
    }
    for (int s = 0; s < 3; ++s) pa::bar_init(&met[s], C);
    lost = any_bad = 0;
    for (int n = 0; n < kPairs; ++n) gather[n] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int x = tid; x < 256; x += kThreads) expf[x] = kDevExpF[x];
  if (tid < 18) expi[tid] = tid < 16 ? kDevExpI[tid] : 0;
  pdl_trigger();
  pdl_wait();
  const int kvh = blockIdx.y;
  int i = blockIdx.x / C;
  // More clusters than a wave holds: the longest sequences start first, so that the last to run are
  // short.  A block ranks the lengths itself.
  if (ordered) {
    const int n = (int)a.n_seqs;
    for (int x = tid; x < n; x += kThreads) {
      const int slot = a.seqs ? a.seqs[x] : x;
      lens[x] = slot >= 0 && slot < a.max_seqs ? a.length[slot] : 0;
    }
    __syncthreads();
    for (int x = tid; x < n; x += kThreads) {
      int before = 0;
      for (int y = 0; y < n; ++y) before += lens[y] > lens[x] || (lens[y] == lens[x] && y < x);
      if (before == i) chosen = x;
    }
    __syncthreads();
    i = chosen;
  }
  const SeqView sv = view_sequence(a, i);
  const int rep = (int)(a.n_heads / a.n_kv_heads), P = (int)a.page_size;
  const int pshift = 31 - __clz(P);  // pages hold a power of two
  const int rows = min(sv.rows, (int)min(a.max_rows, (int64_t)INT_MAX));
  const int64_t pairs = (int64_t)rows * rep;
  const int g0 = blockIdx.z * kPairs;
  if (g0 >= pairs) {  // the whole cluster agrees
    if (sv.code && rank == 0 && kvh == 0 && g0 == 0 && tid == 0) raise_status(a.status, sv.code);
    return;
  }
  const int nr = min(kPairs, (int)pairs - g0);
  // row j of the sequence sees keys 0 .. len - rows + j
  const int cap = key_cap(a);
  auto keys_of = [&](int n) {  // of pair g0 + n
    const int64_t t = (int64_t)sv.len - sv.rows + (g0 + n) / rep + 1;
    return (int)(t < 0 ? 0 : t > cap ? cap : t);
  };
  const int T = keys_of(nr - 1);
  int slice = ((T + C - 1) / C + 63) & ~63;
  const int k0 = (int)min((int64_t)T, (int64_t)rank * slice), k1 = (int)min((int64_t)T, (int64_t)k0 + slice), nkeys = k1 - k0;
  const int tiles = (nkeys + kTK - 1) / kTK;
  const int ss = score_stride(shape.cap);
  unsigned char* base = raw + ((1024 - (pa::s32(raw) & 1023)) & 1023);
  unsigned char* ring = base;
  int32_t* sc = reinterpret_cast<int32_t*>(base + S * kTK * D);  // [nr][ss]
  int32_t* opart = sc + shape.nr * ss;                            // [nr][D] this slice's sums
  int32_t* xo = opart + shape.nr * D;                             // [C][share] peers' sums of this CTA's share
  int32_t* ids = xo + shape.nr * D + kMaxCluster;                               // page ids of the slice
  const int p0 = k0 >> pshift, np = nkeys ? ((k1 - 1) >> pshift) - p0 + 1 : 0;
  const int32_t* pages = a.table + (sv.slot < 0 ? 0 : sv.slot) * a.table_stride + p0;
  __syncthreads();
  for (int x = tid; x < np; x += kThreads) {
    int id = pages[x];
    if (id < 0 || id >= a.n_pages) {
      id = -1;
      any_bad = 1;
    }
    ids[x] = id;
  }
  for (int x = tid; x < nr * D; x += kThreads) opart[x] = 0;
  if (C > 1)
    pa::cluster_sync();  // the peers' barriers are there
  else
    __syncthreads();
  if (rank == 0 && kvh == 0 && tid == 0) {
    int code = sv.code;
    if (sv.rows > a.max_rows || sv.len > cap) code |= LLX_STATUS_BAD_BOUND;
    if (!code && sv.len < sv.rows) code = LLX_STATUS_BAD_POSITION;
    if (code) raise_status(a.status, code);
  }
  if (tid == 0 && any_bad) raise_status(a.status, LLX_STATUS_BAD_PAGE);

  if (warp >= kWarps) {
    // A stage costs its loading warp some 750 cycles of latency (its barrier, the count of bytes, the
    // copies), 22 bytes a cycle: two warps load every other stage.  The
    // ring is even, so each keeps to its own stages: a barrier's parity tells two turns apart, not three,
    // and a warp that shared a stage could find a turn done that has not begun.
    if (lane == 0) {
      const int bshift = 31 - __clz(shape.box);
      int s = warp - kWarps;
      uint32_t turn = 1;
      for (int it = s; it < 2 * tiles; it += kLoaders) {
        const int t0 = (it < tiles ? it : it - tiles) * kTK;
        if (it >= S && !pa::bar_wait(&empty[s], turn, &lost)) break;
        const int boxes = (min(kTK, nkeys - t0) + shape.box - 1) >> bshift;
        pa::bar_expect(&full[s], (uint32_t)(boxes * shape.box * D));
        for (int b = 0; b < boxes; ++b) {
          const int key = k0 + t0 + b * shape.box;
          // absent pages: page 0 is read in their place, its keys are never used
          pa::load_rows(ring + s * kTK * D + b * shape.box * D, it < tiles ? &mk : &mv, &full[s], kvh * P + (key & (P - 1)),
                        max(ids[(key >> pshift) - p0], 0));
        }
        s += kLoaders;
        if (s >= S) {
          s -= S;
          turn ^= 1;
        }
      }
    }
  } else {
    const int g = lane >> 2, tig = lane & 3;
    // ---- scores ----
    uint32_t qf[KB][2];
    {
      const int n = g0 + g;
      const int8_t* q = a.q8 + (int64_t)(sv.first + n / rep) * a.q8_stride + (int64_t)(kvh * rep + n % rep) * D + 4 * tig;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        qf[kb][0] = g < nr ? *reinterpret_cast<const uint32_t*>(q + kb * 32) : 0u;
        qf[kb][1] = g < nr ? *reinterpret_cast<const uint32_t*>(q + kb * 32 + 16) : 0u;
      }
    }
    const int ra = 2 * tig, rb = ra + 1;
    const int Ta = ra < nr ? keys_of(ra) - k0 : 0, Tb = rb < nr ? keys_of(rb) - k0 : 0;  // visible keys of the slice
    int mxa = INT_MIN, mxb = INT_MIN;
    int s = 0;  // stage, and the turn of the ring
    uint32_t turn = 0;
    auto done = [&]() {
      __syncwarp();
      if (lane == 0) pa::bar_arrive(&empty[s]);
      if (++s == S) {
        s = 0;
        turn ^= 1;
      }
    };
    for (int it = 0; it < tiles; ++it) {
      pa::bar_wait(&full[s], turn, &lost);
      const int t0 = it * kTK + warp * 16;  // 16 keys per warp
      if (t0 < nkeys) {
        const uint32_t tile = pa::s32(ring + s * kTK * D);
        int32_t c[4] = {0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t f[4];
          pa::ldmatrix4(f, tile + pa::tile_at<D>(warp * 16 + (lane & 15), kb * 2 + (lane >> 4)));
          pa::mma16832<false>(c, f[0], f[1], f[2], f[3], qf[kb][0], qf[kb][1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = t0 + h * 8 + g;  // key of the slice
          const bool there = !any_bad || t >= nkeys || ids[((k0 + t) >> pshift) - p0] >= 0;
          const int va = t < Ta && there ? c[2 * h] : INT_MIN, vb = t < Tb && there ? c[2 * h + 1] : INT_MIN;
          if (ra < nr) sc[ra * ss + t] = va;
          if (rb < nr) sc[rb * ss + t] = vb;
          mxa = max(mxa, va);
          mxb = max(mxb, vb);
        }
      } else if (t0 < ((nkeys + 31) & ~31)) {  // the values are taken 32 keys at a time
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (ra < nr) sc[ra * ss + t0 + h * 8 + g] = INT_MIN;
          if (rb < nr) sc[rb * ss + t0 + h * 8 + g] = INT_MIN;
        }
      }
      done();
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      mxa = max(mxa, __shfl_xor_sync(0xffffffffu, mxa, o));
      mxb = max(mxb, __shfl_xor_sync(0xffffffffu, mxb, o));
    }
    if (g == 0) {
      wred[warp * kPairs + ra] = (uint32_t)mxa;
      wred[warp * kPairs + rb] = (uint32_t)mxb;
    }
    pa::named_sync(1, kConsumers);
    // every CTA of the cluster gets every slice's maxima: x[slice][pair]
    auto meet = [&](uint32_t v, uint32_t* x, uint64_t* bar) {  // thread c * kPairs + n brings pair n to CTA c
      const int n = tid % kPairs, c = tid / kPairs;
      if (C == 1) {
        if (tid < kPairs) x[n] = v;
        pa::named_sync(1, kConsumers);
        return;
      }
      if (c < C) pa::peer_store(pa::peer(x + rank * kPairs + n, (uint32_t)c), v);
      pa::named_sync(1, kConsumers);
      if (tid < C) pa::peer_arrive(pa::peer(bar, (uint32_t)tid));
      pa::bar_wait<true>(bar, 0, &lost);
    };
    {
      int v = INT_MIN;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = max(v, (int)wred[w * kPairs + tid % kPairs]);
      meet((uint32_t)v, xmax, &met[0]);
    }
    // ---- exponentials of the slice, in place; sums ----
    const int nfill = (nkeys + 31) & ~31;  // the score pass wrote up to here
    const GapScale gs = gap_scale<HIGH>(a.Ms, a.Ss);
    {
      // a pair's keys are dealt to kConsumers / nr threads, 4 neighbouring ones at a time
      const int team = kConsumers / nr, n = tid / team;
      uint32_t sum = 0;
      if (n < nr) {
        int mx = INT_MIN;
        for (int c = 0; c < C; ++c) mx = max(mx, (int)xmax[c * kPairs + n]);
        int4* row = reinterpret_cast<int4*>(sc + n * ss);
#pragma unroll 2
        for (int t = tid - n * team; t < nfill / 4; t += team) {
          const int4 v = row[t];
          auto weight = [&](int x) {
            const uint32_t e = table_exp(gap_index<HIGH>((uint32_t)mx - (uint32_t)x, gs), expi, expf);
            return x == INT_MIN ? 0u : e;
          };
          const uint32_t p0 = weight(v.x), p1 = weight(v.y), p2 = weight(v.z), p3 = weight(v.w);
          row[t] = make_int4((int)p0, (int)p1, (int)p2, (int)p3);
          sum += p0 + p1 + p2 + p3;
        }
        // a slice has less than 2^16 keys of at most 65535: 32 bits hold its sum
        if (sum) atomicAdd(&gather[n], sum);
      }
      pa::named_sync(1, kConsumers);
    }
    meet(gather[tid % kPairs], xsum, &met[1]);
    // ---- values: weights of pair g, normalised as they are read ----
    uint64_t whole = 0;
    for (int c = 0; c < C; ++c) whole += xsum[c * kPairs + g];
    const uint32_t inv = whole > 0x80000000ull ? 0u : 0x80000000u / (whole ? (uint32_t)whole : 1u);
    const int psh = 31 - (int)a.prob_bits;
    const uint32_t prnd = 1u << (psh - 1), pmax = (1u << a.prob_bits) - 1u;
    const bool wide = a.prob_bits > 8;
    // a warp takes 32 keys of a stage and half of the channels
    constexpr int HB = MB / 2;
    const int keys = (warp & 3) * 32, side = warp >> 2;
    int32_t ah[HB][4], al[HB][4];
#pragma unroll
    for (int m = 0; m < HB; ++m)
#pragma unroll
      for (int k = 0; k < 4; ++k) ah[m][k] = al[m][k] = 0;
    for (int it = tiles; it < 2 * tiles; ++it) {
      pa::bar_wait(&full[s], turn, &lost);
      const int t0 = (it - tiles) * kTK + keys;
      if (t0 < nkeys) {
        const unsigned char* tile = ring + s * kTK * D;
        // MMA key index 4 tig + e of a 16-key half stands for key 2 tig + (e & 1) + 8 (e >> 1), in the
        // weights as in the values: a thread's weights are two 8-byte reads
        uint32_t w[2][HB * 2], bl[2], bh[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pn[4] = {0, 0, 0, 0};
          if (g < nr) {
            const int2 x = *reinterpret_cast<const int2*>(sc + g * ss + t0 + h * 16 + 2 * tig);
            const int2 y = *reinterpret_cast<const int2*>(sc + g * ss + t0 + h * 16 + 2 * tig + 8);
            // p <= sum, so p * inv <= 2^31
            pn[0] = min(((uint32_t)x.x * inv + prnd) >> psh, pmax);
            pn[1] = min(((uint32_t)x.y * inv + prnd) >> psh, pmax);
            pn[2] = min(((uint32_t)y.x * inv + prnd) >> psh, pmax);
            pn[3] = min(((uint32_t)y.y * inv + prnd) >> psh, pmax);
          }
          const uint32_t p01 = __byte_perm(pn[0], pn[1], 0x5410), p23 = __byte_perm(pn[2], pn[3], 0x5410);
          bl[h] = __byte_perm(p01, p23, 0x6420);
          bh[h] = __byte_perm(p01, p23, 0x7531);
          const int r0 = keys + h * 16 + 2 * tig;
          if constexpr (D == 128) {
            uint2 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = *reinterpret_cast<const uint2*>(tile + pa::tile_at<D>(r0 + (e & 1) + 8 * (e >> 1), g) + side * 8);
            pa::transpose4(v[0].x, v[1].x, v[2].x, v[3].x, w[h]);
            pa::transpose4(v[0].y, v[1].y, v[2].y, v[3].y, w[h] + 4);
          } else {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = *reinterpret_cast<const uint32_t*>(tile + pa::tile_at<D>(r0 + (e & 1) + 8 * (e >> 1), g >> 1) + (g & 1) * 8 +
                                                        side * 4);
            pa::transpose4(v[0], v[1], v[2], v[3], w[h]);
          }
        }
#pragma unroll
        for (int m = 0; m < HB; ++m) {
          pa::mma16832<true>(al[m], w[0][2 * m], w[0][2 * m + 1], w[1][2 * m], w[1][2 * m + 1], bl[0], bl[1]);
          if (wide) pa::mma16832<true>(ah[m], w[0][2 * m], w[0][2 * m + 1], w[1][2 * m], w[1][2 * m + 1], bh[0], bh[1]);
        }
      }
      done();
    }
    // block row g of m stands for channel g D / 8 + side D / 16 + 2 m, row g + 8 for the next one
#pragma unroll
    for (int m = 0; m < HB; ++m)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = 2 * tig + (k & 1), ch = g * (D / 8) + side * (D / 16) + 2 * m + (k >> 1);
        if (n < nr) atomicAdd(&opart[n * D + ch], ah[m][k] * 256 + al[m][k]);
      }
    pa::named_sync(1, kConsumers);
    // ---- each CTA finishes its share of the outputs ----
    const int share = (nr * D + C - 1) / C, e0 = (int)rank * share;
    if (C > 1) {
      for (int e = tid; e < nr * D; e += kConsumers) {
        const int c = e / share;
        pa::peer_store(pa::peer(xo + rank * share + (e - c * share), (uint32_t)c), (uint32_t)opart[e]);
      }
      pa::named_sync(1, kConsumers);
      if (tid < C) pa::peer_arrive(pa::peer(&met[2], (uint32_t)tid));
      pa::bar_wait<true>(&met[2], 0, &lost);
    }
    for (int x = tid; x < share && e0 + x < nr * D; x += kConsumers) {
      int64_t o = 0;
      if (C > 1)
        for (int c = 0; c < C; ++c) o += xo[c * share + x];
      else
        o = opart[x];
      if (a.prob_bits == 15) o = rshr(o, 7);
      const int e = e0 + x, n = g0 + e / D;
      a.out[(int64_t)(sv.first + n / rep) * a.out_stride + (int64_t)(kvh * rep + n % rep) * D + e % D] =
          (int8_t)sat8(mulshift(o, a.Mo, (int)a.So));
    }
    if (lost && tid == 0) raise_status(a.status, LLX_STATUS_LOST);
  }
  // no CTA leaves while a peer may still write to it
  if (C > 1) {
    __syncwarp();
    pa::cluster_sync();
  }
}

// Clusters of each size that the device holds at once with 1, 2 or 3 CTAs on an SM, asked for once.
struct Capacity {
  int clusters[4][kMaxCluster + 1];
};
template <int D, bool HIGH>
cudaError_t prepare_decode(int dev, const Capacity** out) {
  static std::atomic<bool> ready[64];
  static std::mutex lock;
  static Capacity caps[64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> hold(lock);
    cudaError_t e = cudaFuncSetAttribute(k_paged_decode<D, HIGH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_paged_decode<D, HIGH>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    for (int occ = 1; occ <= 3 && e == cudaSuccess; ++occ)
      for (int c = 1; c <= kMaxCluster && e == cudaSuccess; ++c) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(c);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemAt[occ];
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = c;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        e = cudaOccupancyMaxActiveClusters(&n, k_paged_decode<D, HIGH>, &cfg);
        caps[dev].clusters[occ][c] = n;
      }
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_release);
  }
  *out = &caps[dev];
  return cudaSuccess;
}

int slice_cap(int64_t max_len, int C) { return (int)(((max_len + C - 1) / C + 63) / 64 * 64); }

size_t smem_for(const llx_paged_attention_args& a, int nr, int64_t len, int C, int ring) {
  const int cap = slice_cap(len, C), P = (int)a.page_size;
  return a.head_dim == 128 ? decode_smem<128>(nr, cap, P, ring) : decode_smem<64>(nr, cap, P, ring);
}

int64_t longest(const llx_paged_attention_args& a) {
  const int64_t held = a.max_pages * a.page_size;
  const int64_t n = a.max_len < held ? a.max_len : held;
  return n < 1 ? 1 : n;
}

}  // namespace

// A slice's scores stay on chip, so max_len has a limit: with pages of 64 about 88,000 keys at head size 128 and
// 8 pairs a KV head or more, 101,000 at 7, 181,000 at 4; at head size 64 98,000 at 8.  Beyond it the chunk
// kernel takes the launch, a CTA per KV head and sequence: 2 single tokens of 80,000 keys, 64 heads on 8 of
// 128, 214 us here; of 100,000 keys 1,543 there.  It reads the bound only for this choice: 16 single tokens of
// 2,000 keys under a bound of 131,072 take 43 us there.
bool paged_decode_fits(const llx_paged_attention_args& a, int64_t pairs) {
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  if (longest(a) > (1 << 19)) return false;  // a slice's keys and sums stay in range
  return smem_for(a, (int)(pairs < kPairs ? pairs : kPairs), longest(a), kMaxCluster, 2) + kStatic <= kSmemMost;
}

template <int D, bool HIGH>
static cudaError_t launch_decode_t(const llx_paged_attention_args& a, cudaStream_t st) {
  int dev = 0;
  const Capacity* cap = nullptr;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = prepare_decode<D, HIGH>(dev, &cap);
  if (e != cudaSuccess) return e;
  const int64_t rep = a.n_heads / a.n_kv_heads, len = longest(a);
  const int64_t pairs = a.max_rows * rep;
  const int groups = (int)((pairs + kPairs - 1) / kPairs);
  DecodeShape sh;
  sh.nr = (int)(pairs < kPairs ? pairs : kPairs);
  sh.box = a.page_size < 64 ? (int)a.page_size : 64;
  const int64_t units = a.n_seqs * a.n_kv_heads * groups;
  // How many CTAs share a sequence's keys, and how deep their rings are: the cheapest by this count
  // (bytes and ns).  A wave takes what HBM needs for its bytes (6.5 KB a ns), or what its CTAs do: a
  // ring's bytes per 1.9 us of loaded latency, 49 B a ns of an SM with one CTA on it, 60 with more.  A wave's
  // phases cost 6 us where a CTA is alone on its SM, less where others stream meanwhile.  The constants come
  // from two launches.  64 sequences of 1500 to 4200 keys, 8 KV heads: one CTA each, ring of 4 82 us, of 2
  // 106; two CTAs, ring of 4 95, of 2 112.  Two of 64k keys: 10 CTAs, ring of 6 103 us; 9, 6 113; 16, 2 118;
  // 8, 4 127.
  // Lengths are max_len here, the sequences' own being on the device: a bound far above them costs.  16 single
  // tokens of 2,000 keys, 64 heads on 8 of 128: 21 us with a bound of 2,048, 190 with 80,000.
  double best = 1e30;
  bool waves = false;
  for (int c = 1; c <= kMaxCluster; ++c) {
    if (c > 1 && len <= (int64_t)(c - 1) * 64) break;
    for (int ring = 2; ring <= kMaxRing; ring += kLoaders) {  // each loading warp keeps to its own stages
      const size_t smem = smem_for(a, sh.nr, len, c, ring) + kStatic;
      if (smem > kSmemMost) break;
      const int occ = smem <= kSmemAt[3] + kStatic ? 3 : smem <= kSmemAt[2] + kStatic ? 2 : 1;
      const int64_t wave = cap->clusters[occ][c];
      if (wave < 1) continue;
      const double bytes = 2.0 * D * ((len + c - 1) / c);  // of a CTA
      const double rate = ring * kTK * D / 1900.0, fixed = occ == 1 ? 6000 : occ == 2 ? 3500 : 2500;
      auto run = [&](int64_t clusters) {  // one wave of them
        const int64_t ctas = clusters * c, per_sm = (ctas + 147) / 148;
        const double even = ctas * bytes / 6.5e3, most = per_sm > 1 ? 60.0 / per_sm : 49.0;
        const double own = bytes / (rate < most ? rate : most);
        return (even > own ? even : own) + fixed;
      };
      const int64_t full = units / wave, rest = units % wave;
      const double t = (full ? full * run(wave) : 0) + (rest ? run(rest) : 0) + (c > 1 ? 800 + 100 * c : 0);
      if (t < best) {
        best = t;
        sh.cluster = c;
        sh.ring = ring;
        waves = full > 0 && rest > 0;
      }
    }
  }
  if (best == 1e30) return cudaErrorInvalidConfiguration;
  sh.cap = slice_cap(len, sh.cluster);
  const bool ordered = waves && a.n_seqs > 1 && a.n_seqs <= kOrdered;
  CUtensorMap mk, mv;
  e = make_page_map(&mk, a.k_pages, a, sh.box);
  if (e == cudaSuccess) e = make_page_map(&mv, a.v_pages, a, sh.box);
  if (e != cudaSuccess) return e;
  const size_t smem = decode_smem<D>(sh.nr, sh.cap, (int)a.page_size, sh.ring);
  const dim3 grid((unsigned)(a.n_seqs * sh.cluster), (unsigned)a.n_kv_heads, (unsigned)groups);
  if (sh.cluster == 1) return launch_k(k_paged_decode<D, HIGH>, grid, dim3(kThreads), smem, st, a, mk, mv, sh, ordered);
  return launch_kc(k_paged_decode<D, HIGH>, grid, dim3(kThreads), smem, st, dim3(sh.cluster, 1, 1), a, mk, mv, sh, ordered);
}

cudaError_t launch_paged_decode(const llx_paged_attention_args& a, cudaStream_t st) {
  if (a.head_dim == 128) return a.Ss >= 33 ? launch_decode_t<128, true>(a, st) : launch_decode_t<128, false>(a, st);
  return a.Ss >= 33 ? launch_decode_t<64, true>(a, st) : launch_decode_t<64, false>(a, st);
}

}  // namespace llx
