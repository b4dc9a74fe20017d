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
// Recomputing S costs the tensor cores 2.5 times the least; keeping it would cost 64 KB a tile.
//
// Shared memory bounds it, not the tensor cores (23 % busy): per tile of 128 x 128 pass 1 takes some 520
// cycles (K from L2), pass 2 1800 and pass 3 2600, most of it the lookup of every score's exponential, a
// word of a table of 4096 at 3.7 wavefronts a warp.  The two-table form of the definition (256 fractions,
// kept once per bank, times 16 whole parts) has no conflicts but takes two lookups and a product: 367 us
// against 322 then.  Four chunks of some 500 rows over
// 2,100 to 4,000 earlier keys, 32 heads on 8: 273 us, 0.35 PFLOP/s of the operator's own products.  Steps:
// one block per row and head 57,717 us; this form 494; exponentials from one table 405; whole tiles without
// masks and cheaper waits 372; the table in words 323; page ids read ahead 303; a second loading warp 273.
// A tile's keys stay with one CTA: launches of few tiles over long contexts leave SMs idle (14 CTAs for 110
// rows, 16 heads on 2, about 50k keys: 1.1 ms).  And the grid is the longest chunk's tiles for every sequence
// and KV head: of some 1,344 CTAs of a mixed launch (2 chunks of 300 to 420 rows, 30 single rows, 74 us) 144 have a
// tile, and the others, an SM each, set up their barriers and the table before they see that; the chain of
// the longest tile, 21 tiles of keys, is some 55 us of it.
// Roles: warps 0 and 1 load (every other stage), warps 2 and 3 issue the MMAs (every other score tile of
// passes 1 and 2; the scores and the values of pass 3), warps 4 to 19 do the softmax.
#include <atomic>
#include <type_traits>

#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace llx {
namespace {

constexpr int kRows = 128, kTK = 128;
constexpr int kSoftWarps = 16, kThreads = 128 + kSoftWarps * 32;
// Even: the two loading warps, and in passes 1 and 2 the two issuing ones, then each keep to their own
// stages.  A barrier's parity tells two turns apart, not three: a warp that shared a stage with the
// other could find a turn done that has not begun.
constexpr int kStages = 6;
static_assert(kStages % 2 == 0, "");
constexpr uint32_t kHidden = 0x80000000u;  // score of a key that a row does not see

template <int D>
struct Smem {
  static constexpr int q = 0;
  static constexpr int ring = kRows * D;
  static constexpr int p = ring + kStages * kTK * D;  // [2][hi, lo][128][128]
  static constexpr int curve = p + 4 * kRows * kTK;   // table_exp of every index below 4096
  static constexpr int bytes = curve + 4096 * 4 + 1024;
};

// shared-memory operand of rows of D bytes, swizzled by D bytes: rows along the MMA's M or N with the
// contraction contiguous (scores), or rows along the contraction with N contiguous (values); either
// way groups of 8 rows follow one another.  The address is the lower word's, in units of 16 bytes.
template <int D>
__device__ __forceinline__ uint64_t operand(uint32_t at) {
  constexpr uint32_t hi = (8 * D >> 4) | 1u << 14 | (D == 128 ? 2u : 4u) << 29;  // group stride, version, swizzle
  return (uint64_t)hi << 32 | (at | 1u << 16);
}
// weights (unsigned) times values (signed, N contiguous): N = D
__host__ __device__ constexpr uint32_t idesc_values(int D) {
  return (2u << 4) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// N columns of a thread's TMEM lane.  Load and wait are one statement: the registers hold the
// values for whatever the compiler does with them next.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[N]) {
  if constexpr (N == 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr)
        : "memory");
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr)
        : "memory");
}

template <int D, bool HIGH>
__global__ void __launch_bounds__(kThreads, 1)
    k_paged_chunk(const llx_paged_attention_args a, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const int box, const uint32_t word) {
  using L = Smem<D>;
  constexpr uint32_t kO = 2 * kTK;  // TMEM columns: S[2], O_lo, O_hi
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], s_full[2], s_free[2], p_full[2], p_free[2], o_full;
  __shared__ uint32_t tmem_s;
  __shared__ int lost, any_bad;
  __shared__ int32_t red[4][kRows];
  __shared__ unsigned long long red64[4][kRows];
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
  unsigned char* base = raw + ((1024 - (pa::s32(raw) & 1023)) & 1023);
  for (int x = tid; x < 1024; x += kThreads)
    reinterpret_cast<uint4*>(base + L::curve)[x] = reinterpret_cast<const uint4*>(kDevCurve)[x];
  __syncthreads();  // any_bad is clear before a thread sets it
  pdl_wait();
  const int i = blockIdx.z, kvh = blockIdx.y;
  const SeqView sv = view_sequence(a, i);
  const int rep = (int)(a.n_heads / a.n_kv_heads), P = (int)a.page_size;
  const int pshift = 31 - __clz(P);  // pages hold a power of two
  const int rows = (int)min((int64_t)sv.rows, a.max_rows);
  const int64_t pairs = (int64_t)rows * rep;
  // the last rows see the most keys: their tiles start first
  const int tile = (int)((pairs + kRows - 1) / kRows) - 1 - (int)blockIdx.x;
  const int cap = key_cap(a);
  if (blockIdx.x == 0 && kvh == 0 && tid == 0) {
    int code = sv.code;
    if (sv.rows > a.max_rows || (sv.rows && sv.len > cap)) code |= LLX_STATUS_BAD_BOUND;
    if (!code && sv.rows && sv.len < sv.rows) code = LLX_STATUS_BAD_POSITION;
    if (code) raise_status(a.status, code);
  }
  if (tile < 0) return;
  const int g0 = tile * kRows, nr = (int)min((int64_t)kRows, pairs - g0);
  auto keys_of = [&](int n) {
    const int64_t t = (int64_t)sv.len - sv.rows + (g0 + n) / rep + 1;
    return (int)(t < 0 ? 0 : t > cap ? cap : t);
  };
  const int T = keys_of(nr - 1), tiles = (T + kTK - 1) / kTK;
  const int32_t* pages = a.table + (sv.slot < 0 ? 0 : sv.slot) * a.table_stride;
  if (warp == 2) {
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
  // Dependents launch once every CTA has its TMEM columns or has left: a GEMM that follows takes columns
  // before it waits for this grid, and a CTA here that found too few left would wait for it in turn.
  pdl_trigger();
  if (tid == 0 && any_bad) raise_status(a.status, LLX_STATUS_BAD_PAGE);

  if (warp < 2) {
    // K of passes 1 and 2, then K 0, K 1, V 0, K 2, V 1, ..., V last.  A lane loads one box; the page
    // ids of the next load are read before this one's stage is waited for.  A stage costs its warp some
    // 750 cycles of latency, hence two of them.
    const int row = lane * box;  // of the tile
    auto tile_of = [&](int it, bool* is_v) {
      const int x = it - 2 * tiles;
      *is_v = x == 2 * tiles - 1 || (x > 0 && (x & 1) == 0);
      return it < tiles ? it : x < 0 ? it - tiles : x == 2 * tiles - 1 ? tiles - 1 : *is_v ? (x >> 1) - 1 : (x + 1) >> 1;
    };
    auto page_at = [&](int t) {
      const int key = t * kTK + row;
      int id = row < kTK && key < T ? pages[key >> pshift] : 0;
      return id < 0 || id >= a.n_pages ? 0 : id;  // absent: page 0 is read in its place, its keys are never used
    };
    bool is_v;
    int t = tiles ? tile_of(warp, &is_v) : 0, id = page_at(t), s = warp;
    uint32_t turn = 1;
    for (int it = warp; it < 4 * tiles; it += 2) {
      bool next_v;
      const int next = it + 2 < 4 * tiles ? tile_of(it + 2, &next_v) : t, next_id = page_at(next);
      if (it >= kStages && !pa::bar_wait(&empty[s], turn, &lost)) break;
      const int boxes = (min(kTK, T - t * kTK) + box - 1) >> (31 - __clz(box));
      if (lane == 0) pa::bar_expect(&full[s], (uint32_t)(boxes * box * D));
      __syncwarp();
      if (lane < boxes) {
        const int key = t * kTK + row;
        pa::load_rows(base + L::ring + s * kTK * D + row * D, is_v ? &mv : &mk, &full[s], kvh * P + (key & (P - 1)), id);
      }
      t = next;
      id = next_id;
      is_v = next_v;
      s += 2;
      if (s >= kStages) {
        s -= kStages;
        turn ^= 1;
      }
    }
  } else if (warp <= 3) {
    // A whole warp runs the loop and one elected thread issues: the operands' descriptors then live in
    // uniform registers.  A tile costs an issuing warp 900 cycles (two barriers, MMAs, two commits),
    // most of it latency, against 300 for the MMAs: hence two of them.
    uint32_t leader;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
    const uint32_t at_q = pa::s32(base + L::q) >> 4, at_ring = pa::s32(base + L::ring) >> 4, at_p = pa::s32(base + L::p) >> 4;
    const bool wide = a.prob_bits > 8;
    auto scores = [&](int n, int it) {  // score tile n from load it
      const int s = it % kStages;
      const uint32_t turn = (uint32_t)(it / kStages) & 1;
      if (!(n >= 2 ? pa::bar_wait2(&full[s], turn, &s_free[n & 1], (uint32_t)((n >> 1) - 1) & 1, &lost)
                   : pa::bar_wait(&full[s], turn, &lost)))
        return false;
      tc::tc_fence_after();
      if (leader) {
        const uint32_t k = at_ring + s * (kTK * D >> 4), d = tmem + (n & 1) * kTK;
#pragma unroll
        for (int kb = 0; kb < D / 32; ++kb)
          tc::mma_i8(d, operand<D>(at_q + 2 * kb), operand<D>(k + 2 * kb), tc::idesc_i8(kTK), kb > 0);
        tc::mma_commit(&s_full[n & 1]);
        tc::mma_commit(&empty[s]);
      }
      __syncwarp();
      return true;
    };
    auto values = [&](int t, int it) {
      const int s = it % kStages;
      if (!pa::bar_wait2(&full[s], (uint32_t)(it / kStages) & 1, &p_full[t & 1], (uint32_t)(t >> 1) & 1, &lost)) return false;
      tc::tc_fence_after();
      if (leader) {
        const uint32_t v = at_ring + s * (kTK * D >> 4), p = at_p + (t & 1) * (2 * kRows * kTK >> 4);
        const int steps = (min(kTK, T - t * kTK) + 31) / 32;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          if (kb < steps) {
            const uint64_t b = operand<D>(v + kb * (32 * D >> 4));
            tc::mma_i8(tmem + kO, operand<128>(p + (kRows * kTK >> 4) + 2 * kb), b, idesc_values(D), t > 0 || kb > 0);
            if (wide) tc::mma_i8(tmem + kO + D, operand<128>(p + 2 * kb), b, idesc_values(D), t > 0 || kb > 0);
          }
        }
        tc::mma_commit(&p_free[t & 1]);
        tc::mma_commit(&empty[s]);
        if (t == tiles - 1) tc::mma_commit(&o_full);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    for (int n = warp - 2; n < 2 * tiles && ok; n += 2) ok = scores(n, n);
    // pass 3 loads K 0, K 1, V 0, K 2, V 1, ...
    if (warp == 2)
      for (int t = 0; t < tiles && ok; ++t) ok = scores(2 * tiles + t, 2 * tiles + (t ? 2 * t - 1 : 0));
    else
      for (int t = 0; t < tiles && ok; ++t) ok = values(t, t < tiles - 1 ? 2 * tiles + 2 * t + 2 : 4 * tiles - 1);
  } else if ((warp & 3) * 32 >= nr) {
    // a tile of few rows (a sequence's next token among prompt chunks): the warps past them only keep step
    for (int st = 0; st < 3 * tiles; ++st) {
      pa::bar_wait(&s_full[st & 1], (uint32_t)(st >> 1) & 1, &lost);
      __syncwarp();
      if (lane == 0) pa::bar_arrive(&s_free[st & 1]);
      const int t = st - 2 * tiles;
      if (t >= 0) {
        if (t >= 2) pa::bar_wait(&p_free[t & 1], (uint32_t)((t >> 1) - 1) & 1, &lost);
        __syncwarp();
        if (lane == 0) pa::bar_arrive(&p_full[t & 1]);
      }
      if (st + 1 == tiles || st + 1 == 2 * tiles) pa::named_sync(1, kSoftWarps * 32);
    }
    if (tiles == 0) {
      pa::named_sync(1, kSoftWarps * 32);
      pa::named_sync(1, kSoftWarps * 32);
    }
  } else {
    const int quad = warp & 3, part = (warp - 4) >> 2;
    const int n = quad * 32 + lane;  // row of the tile
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int Tn = n < nr ? keys_of(n) : 0;
    // tiles that every row sees whole come first and need no masks
    const int open = any_bad ? 0 : keys_of(0) / kTK;
    int st = 0;  // score tiles taken
    // One pass: f(tile, scores) for the thread's 32 keys of every tile, hidden keys' scores replaced.
    auto pass = [&](auto f) {
      uint32_t v[32];
      auto take = [&]() {
        pa::bar_wait(&s_full[st & 1], (uint32_t)(st >> 1) & 1, &lost);
        tc::tc_fence_after();
        tmem_load<32>(tmem + lanes + (st & 1) * kTK + part * 32, v);
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) pa::bar_arrive(&s_free[st & 1]);
        ++st;
      };
      int t = 0;
      for (; t < open; ++t) {
        take();
        f(t, v);
      }
      for (; t < tiles; ++t) {
        take();
        const int k0 = t * kTK + part * 32, left = Tn - k0;
        uint32_t m = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
        if (any_bad)
          for (int e = 0; e < 32 && k0 + e < T; e += 16) {
            const int id = pages[(k0 + e) >> pshift];
            if (id < 0 || id >= a.n_pages) m &= ~(0xffffu << e);
          }
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!((m >> e) & 1u)) v[e] = kHidden;
        f(t, v);
      }
    };
    int mx = INT_MIN;
    pass([&](int, uint32_t (&v)[32]) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) mx = max(mx, max((int)v[e], (int)v[e + 1]));
    });
    red[part][n] = mx;
    pa::named_sync(1, kSoftWarps * 32);
    mx = max(max(red[0][n], red[1][n]), max(red[2][n], red[3][n]));
    const GapScale gs = gap_scale<HIGH>(a.Ms, a.Ss);
    // HIGH: the gap's product and its rounding are one multiply-add, (mx - s) Ms + round 2^32 =
    // (mx Ms + round 2^32) + s (-Ms), whose high word is shifted.  A hidden key's s of -2^31 then
    // lands beyond the table's end by itself (launch_paged_chunk checks that Ms and Ss make it);
    // a row without keys is put there whole.
    const int64_t top = mx == INT_MIN ? 1ll << 62 : (int64_t)mx * (int32_t)gs.M + ((int64_t)gs.round << 32);
    const int32_t minus = -(int32_t)gs.M;
    const uint32_t curve_at = pa::s32(base + L::curve);
    auto weight = [&](uint32_t s) {
      uint32_t z = HIGH ? (uint32_t)((uint64_t)(top + (int64_t)(int32_t)s * minus) >> 32) >> gs.shift
                        : gap_index<false>((uint32_t)mx - s, gs);
      z = min(z, 4095u);  // the 15th integer part is 0
      if (!HIGH && s == kHidden) z = 4095u;
      uint32_t p;
      // the address as a multiply-add (word is 4): the multipliers have room, the integer units have not
      asm("ld.shared.u32 %0, [%1];" : "=r"(p) : "r"(z * word + curve_at));
      return p;
    };
    unsigned long long sum = 0;
    pass([&](int, uint32_t (&v)[32]) {
      uint32_t s = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) s += weight(v[e]);
      sum += s;
    });
    red64[part][n] = sum;
    pa::named_sync(1, kSoftWarps * 32);
    sum = red64[0][n] + red64[1][n] + red64[2][n] + red64[3][n];
    const uint32_t inv = sum > 0x80000000ull ? 0u : 0x80000000u / (sum ? (uint32_t)sum : 1u);
    const int psh = 31 - (int)a.prob_bits;
    const uint32_t prnd = 1u << (psh - 1), pmax = (1u << a.prob_bits) - 1u;
    const bool wide = a.prob_bits > 8;
    // A weight p below 2^31 / inv keeps p inv + 2^15 below 2^31: with 15 bits its upper half is the
    // normalised weight and nothing needs the upper bound.  Otherwise (a row of nearly one key, 8
    // bits) the weight is shifted and bounded; both leave it in the upper half.
    const bool plain = __all_sync(0xffffffffu, wide && 65535ull * inv + prnd < 0x80000000ull);
    auto normalise = [&](auto simple) {
      pass([&](int t, uint32_t (&v)[32]) {
        if (t >= 2) pa::bar_wait(&p_free[t & 1], (uint32_t)((t >> 1) - 1) & 1, &lost);
        unsigned char* p = base + L::p + (t & 1) * 2 * kRows * kTK;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t lo[4], hi[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = weight(v[h * 16 + w * 4 + e]) * inv + prnd;  // at most 2^31 + 2^22: a weight is at most the sum
              if (!decltype(simple)::value) x[e] = min(x[e] >> psh, pmax) << 16;
            }
            const uint32_t p01 = __byte_perm(x[0], x[1], 0x7632), p23 = __byte_perm(x[2], x[3], 0x7632);
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
      });
    };
    if (plain)
      normalise(std::true_type{});
    else
      normalise(std::false_type{});
    // ---- outputs: D / 4 channels a thread ----
    constexpr int W = D / 4;
    if (tiles) {
      pa::bar_wait(&o_full, 0, &lost);
      tc::tc_fence_after();
    }
    int8_t* dst = a.out + (int64_t)(sv.first + (g0 + n) / rep) * a.out_stride + (int64_t)(kvh * rep + (g0 + n) % rep) * D + part * W;
#pragma unroll
    for (int x = 0; x < W; x += 16) {
      uint32_t lo[16], hi[16], w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 16; ++e) lo[e] = hi[e] = 0;
      if (tiles) {
        tmem_load<16>(tmem + lanes + kO + part * W + x, lo);
        if (wide) tmem_load<16>(tmem + lanes + kO + D + part * W + x, hi);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        int64_t o = (int64_t)(int32_t)hi[e] * 256 + (int32_t)lo[e];
        if (wide) o = rshr(o, 7);
        w[e >> 2] |= ((uint32_t)sat8(mulshift(o, a.Mo, (int)a.So)) & 255u) << (8 * (e & 3));
      }
      if (n < nr) *reinterpret_cast<uint4*>(dst + x) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    tc::tc_fence_before();
  }
  __syncthreads();
  if (lost && tid == 0) raise_status(a.status, LLX_STATUS_LOST);
  if (warp == 2) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int D, bool HIGH>
cudaError_t launch_chunk_t(const llx_paged_attention_args& a, cudaStream_t st) {
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
  return launch_k(k_paged_chunk<D, HIGH>, grid, dim3(kThreads), Smem<D>::bytes, st, a, mk, mv, box, 4u);
}

}  // namespace

bool paged_chunk_fits(const llx_paged_attention_args& a) {
  return (a.head_dim == 64 || a.head_dim == 128) && a.n_seqs <= 65535;
}

cudaError_t launch_paged_chunk(const llx_paged_attention_args& a, cudaStream_t st) {
  // how the quantizer normalises its multipliers; and a score of -2^31 gives an index past the table
  const bool high = a.Ss >= 33 && a.Ms < (1ll << 31) && (a.Ms >> 2 >> (a.Ss - 32)) >= 4096;
  if (a.head_dim == 128) return high ? launch_chunk_t<128, true>(a, st) : launch_chunk_t<128, false>(a, st);
  return high ? launch_chunk_t<64, true>(a, st) : launch_chunk_t<64, false>(a, st);
}

}  // namespace llx
