// Shared by the paged attention kernels: a launch's sequences, the table exponential, TMA loads of
// page rows, mbarriers (every wait bounded) and cluster-wide exchange.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "device_luts.h"
#include "launch.cuh"
#include "numerics.cuh"
#include "paged.h"

namespace llx {

// One sequence of a launch as the kernels see it.
struct SeqView {
  int slot;   // -1: none
  int rows;   // rows of the launch
  int first;  // launch row of the first one
  int len;    // positions the sequence has, new rows included
  int code;   // LLX_STATUS_*
};

__device__ __forceinline__ SeqView view_sequence(const llx_paged_attention_args& a, int i) {
  SeqView v;
  v.code = 0;
  v.first = a.q_start[i];
  const int end = a.q_start[i + 1];
  v.rows = end - v.first;
  v.slot = a.seqs ? a.seqs[i] : i;
  v.len = 0;
  if (v.first < 0 || v.rows < 0 || end > a.rows) {
    v.rows = 0;
    v.slot = -1;
    v.code = LLX_STATUS_BAD_BOUND;
  } else if (v.slot < 0 || v.slot >= a.max_seqs) {
    v.slot = -1;
    v.code = LLX_STATUS_BAD_SLOT;
  } else {
    v.len = a.length[v.slot];
  }
  return v;
}

// keys that a launch lets a row see at most
__device__ __forceinline__ int key_cap(const llx_paged_attention_args& a) {
  const int64_t held = a.max_pages * a.page_size;
  const int64_t cap = a.max_len < held ? a.max_len : held;
  return cap > INT_MAX - 1024 ? INT_MAX - 1024 : (int)cap;
}

// The score gap's exponential index z = rshr(d * Ms, Ss), d = max - s < 2^23.  With Ss >= 33 it
// comes from the product's high word: the rounding constant 2^(Ss-1) leaves the low word alone,
// and the low word adds less than one to a value that is floored anyway.  That needs the sum of
// high word and constant to stay in 32 bits: 2^23 + 2^30 at most, for Ss <= 63.
struct GapScale {
  uint32_t M, round;
  int shift;  // HIGH: of the high word; else of the whole product
};
template <bool HIGH>
__device__ __forceinline__ GapScale gap_scale(int64_t Ms, int64_t Ss) {
  GapScale g;
  g.M = (uint32_t)Ms;
  g.shift = (int)(HIGH ? Ss - 32 : Ss);
  g.round = HIGH ? 1u << (Ss - 33) : 0u;
  return g;
}
template <bool HIGH>
__device__ __forceinline__ uint32_t gap_index(uint32_t d, const GapScale& g) {
  if (HIGH) return (__umulhi(d, g.M) + g.round) >> g.shift;
  const uint64_t p = (uint64_t)d * g.M;
  const uint64_t z = g.shift == 0 ? p : (p >> g.shift) + ((p >> (g.shift - 1)) & 1u);
  return z > 4096u ? 4096u : (uint32_t)z;
}
// table exponential (numerics.h:104-107); expi has a 17th entry of 0 for every z >= 4096
__device__ __forceinline__ uint32_t table_exp(uint32_t z, const uint16_t* expi, const uint16_t* expf) {
  const uint32_t zc = z < 4096u ? z : 4096u;
  return ((uint32_t)expi[zc >> 8] * (uint32_t)expf[zc & 255u] + 32768u) >> 16;
}

namespace pa {

// A try suspends the thread for up to kSuspend ns instead of taking issue slots; kPolls of them
// (over a second) bound a wait.
constexpr uint32_t kSuspend = 20000, kPolls = 1u << 16;

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(b)), "r"(n));
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s32(b)), "r"(bytes) : "memory");
}
template <bool CLUSTER>
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  if (CLUSTER)  // for a barrier that other CTAs of the cluster arrive on
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(s32(b)), "r"(parity), "r"(kSuspend)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(s32(b)), "r"(parity), "r"(kSuspend)
        : "memory");
  return ok != 0;
}
// Waits for a phase; false once it has not come within the limit.  `lost` then stays set and makes
// the block's later waits short, so that it ends.  The first try reads nothing else: a loop of
// waits that have ended already is as fast as their tries.
template <bool CLUSTER = false>
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, volatile int* lost) {
  if (bar_try<CLUSTER>(b, parity)) return true;
  for (uint32_t i = 1; i < kPolls; ++i) {
    if (bar_try<CLUSTER>(b, parity)) return true;
    if ((i & 255u) == 0 && *lost) return false;
  }
  *lost = 1;
  return false;
}
// both phases; the tries overlap
__device__ __forceinline__ bool bar_wait2(uint64_t* b, uint32_t pb, uint64_t* c, uint32_t pc, volatile int* lost) {
  const bool b1 = bar_try<false>(b, pb), c1 = bar_try<false>(c, pc);
  if (b1 && c1) return true;
  const bool b2 = b1 || bar_wait(b, pb, lost);
  return (c1 || bar_wait(c, pc, lost)) && b2;
}
__device__ __forceinline__ uint32_t peer(const void* local, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(s32(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_store(uint32_t at, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void peer_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// rows of one head of one page: box {head_dim, rows} at (0, row, page)
__device__ __forceinline__ void load_rows(void* dst, const CUtensorMap* map, uint64_t* bar, int row, int page) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
          "r"(s32(dst)),
      "l"((uint64_t)map), "r"(s32(bar)), "r"(0), "r"(row), "r"(page)
      : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d += a (16 x 32, s8) b (32 x 8, s8 or u8)
template <bool B_U8>
__device__ __forceinline__ void mma16832(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (B_U8)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16-byte chunk of a row of D bytes in a tile that TMA wrote with a D-byte swizzle (D 64 or 128):
// the chunk index is xored with the row, so the 8 rows of a fragment fall into different banks
template <int D>
__device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
  return D == 128 ? (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4))
                  : (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}
// 4 x 4 byte transpose: x_e holds channels 0..3 of key e; w[q] gets channel q of keys 0..3
__device__ __forceinline__ void transpose4(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t* w) {
  const uint32_t t0 = __byte_perm(x0, x1, 0x5140), t1 = __byte_perm(x0, x1, 0x7362);
  const uint32_t t2 = __byte_perm(x2, x3, 0x5140), t3 = __byte_perm(x2, x3, 0x7362);
  w[0] = __byte_perm(t0, t2, 0x5410);
  w[1] = __byte_perm(t0, t2, 0x7632);
  w[2] = __byte_perm(t1, t3, 0x5410);
  w[3] = __byte_perm(t1, t3, 0x7632);
}

}  // namespace pa

// Tensor map of a layer's pages for boxes of `box_rows` rows of one head, swizzled by the row's
// width; head_dim 64 or 128.
cudaError_t make_page_map(CUtensorMap* map, const void* base, const llx_paged_attention_args& a, int box_rows);

// Few query rows per sequence: `pairs` stacked (row, head) pairs per KV head at most.  False: this
// geometry has no such kernel.
bool paged_decode_fits(const llx_paged_attention_args& a, int64_t pairs);
cudaError_t launch_paged_decode(const llx_paged_attention_args& a, cudaStream_t st);

// Any number of rows and keys, head_dim 64 or 128.
bool paged_chunk_fits(const llx_paged_attention_args& a);
cudaError_t launch_paged_chunk(const llx_paged_attention_args& a, cudaStream_t st);

}  // namespace llx
