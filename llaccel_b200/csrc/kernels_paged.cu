// Paged cache kernels: the launch's queries, keys and values on their way into the cache
// (k_paged_append), and the management of pages (reserve, fork, free, compact).
#include <cuda_runtime.h>

#include <cstdint>

#include "launch.cuh"
#include "numerics.cuh"
#include "paged.h"

namespace llx {

// ---------------------------------------------------------------------------------------
// Append: per row and head, RMSNorm over the head (numerics.h:60-71), rotation at the row's
// position (numerics.h:75-84) and requantization; queries to q8, keys and values to the page
// of their position.
// ---------------------------------------------------------------------------------------

// Where a launch row goes: its position and page, or a status code.
struct Place {
  int64_t pos, page;
  int code;
  bool absent;  // behind the last sequence
};
__device__ __forceinline__ Place place_row(const llx_paged_append_args& a, int r) {
  Place p{-1, -1, 0, false};
  const int i = find_sequence(a.q_start, (int)a.n_seqs, r);
  if (i < 0) {
    p.absent = true;
    return p;
  }
  const int slot = a.seqs ? a.seqs[i] : i;
  if (slot < 0 || slot >= a.max_seqs) {
    p.code = LLX_STATUS_BAD_SLOT;
    return p;
  }
  p.pos = (int64_t)a.length[slot] - (a.q_start[i + 1] - r);
  const int shift = __ffs((int)a.page_size) - 1;
  if (p.pos < 0 || p.pos >= a.n_positions || p.pos >> shift >= a.max_pages) {
    p.code = LLX_STATUS_BAD_POSITION;
    return p;
  }
  p.page = a.table[slot * a.table_stride + (p.pos >> shift)];
  if (p.page < 0 || p.page >= a.n_pages) p.code = LLX_STATUS_BAD_PAGE;
  return p;
}

// Any geometry, constants and alignment: one block per row, one warp per head at a time.
__global__ void __launch_bounds__(256) k_paged_append_any(const llx_paged_append_args a) {
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x;
  const Place at = place_row(a, r);
  if (at.absent) return;
  const int D = (int)a.head_dim, half = D / 2, H = (int)a.n_heads, Hkv = (int)a.n_kv_heads;
  const int64_t pos = at.pos, page = at.page;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  int8_t* q8 = a.q8 + r * a.q8_stride;
  if (at.code) {
    if (threadIdx.x == 0) raise_status(a.status, at.code);
    for (int e = threadIdx.x; e < H * D; e += blockDim.x) q8[e] = 0;
    return;
  }
  const int row = (int)(pos % a.page_size);
  const int64_t head0 = page * a.page_stride + (int64_t)row * D;  // key / value row of head 0
  const int64_t head_step = a.page_size * D;
  const int16_t* ct = a.cos + pos * half;
  const int16_t* sn = a.sin + pos * half;
  for (int h = warp; h < H + Hkv; h += warps) {
    const bool is_q = h < H;
    const int hh = is_q ? h : h - H;
    const int16_t* x = is_q ? a.q + r * a.q_stride + (int64_t)hh * D : a.k + r * a.k_stride + (int64_t)hh * D;
    const int16_t* gamma = is_q ? a.q_gamma : a.k_gamma;
    int64_t inv = 0;
    if (gamma) {
      uint64_t ss = 0;
      for (int e = lane; e < D; e += 32) ss += (uint64_t)((int64_t)x[e] * x[e]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const uint32_t root = isqrt48_fast(ss + (uint64_t)(is_q ? a.q_eps : a.k_eps));
      const uint64_t v = udiv_fast((uint64_t)(is_q ? a.q_C : a.k_C), root ? root : 1);
      inv = v < 65535 ? (int64_t)v : 65535;
    }
    const int sh = (int)(is_q ? a.q_shift : a.k_shift);
    const int64_t M = is_q ? a.q_M : a.k_M;
    const int S = (int)(is_q ? a.q_S : a.k_S);
    int8_t* dst = is_q ? q8 + (int64_t)hh * D : a.k_pages + head0 + hh * head_step;
    for (int e = lane; e < half; e += 32) {
      int64_t x1 = x[e], x2 = x[e + half];
      if (gamma) {
        x1 = sat16(rshr(x1 * gamma[e] * inv, sh));
        x2 = sat16(rshr(x2 * gamma[e + half] * inv, sh));
      }
      const int64_t c = ct[e], s = sn[e];
      dst[e] = (int8_t)sat8(mulshift(sat16(rshr(x1 * c - x2 * s, 14)), M, S));
      dst[e + half] = (int8_t)sat8(mulshift(sat16(rshr(x2 * c + x1 * s, 14)), M, S));
    }
  }
  const int8_t* v = a.v + r * a.v_stride;
  for (int e = threadIdx.x; e < Hkv * D; e += blockDim.x) a.v_pages[head0 + (e / D) * head_step + e % D] = v[e];
}

// The usual case: head_dim D a power of two, 16-byte aligned rows, multipliers below 2^31 with shifts
// of 32 and more (how the quantizer normalises them), norm shifts of 18 to 46.  D / 16 lanes share a
// head, each with 8 neighbouring values and their 8 partners half a head away: one 16-byte load each,
// and a rotation without exchange.  The row's place is looked up while those loads are under way.
// Per row 2 (H + Hkv) D + Hkv D bytes read, H D + 2 Hkv D written.  8,000 rows of 16 + 8 heads of 128 with
// norms: 92 MB in 37 us, 2.5 TB/s; the copy rate would allow 14 us.  No limit is reached: 65 % of the issue
// slots, 17 % of DRAM.  64-bit products of norm and requantization make some 40 instructions a value; 80
// registers leave five warps a scheduler, which wait 1.6 cycles an instruction for results, 1.3 for the
// integer multipliers and 0.8 for loads, over 2.3 waves.  A block per row and a warp per head with single
// loads took 166; one lane per head for square root and quotient, after a first reading of the row, 47.  A
// single row takes 3.2 us inside a graph, most of it latency.  Other head sizes and alignments:
// k_paged_append_any, 8,000 rows of 16 + 8 heads of 96 in 178 us (68 MB).
struct AppendSide {
  const int16_t *x, *gamma;
  int64_t eps, C, stride;
  int shift;
  int32_t M;
  int S;
};

__device__ __forceinline__ void unpack8(const uint4& v, int (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = (int)(int16_t)(w[j] & 0xffffu);
    x[2 * j + 1] = (int)w[j] >> 16;
  }
}
__device__ __forceinline__ int clamp32(int v, int lo, int hi) { return max(lo, min(hi, v)); }

// floor(sqrt(t)) for t < 2^48: an approximate root is off by a few at most, integer products settle it
__device__ __forceinline__ uint32_t root48(uint64_t t) {
  float f;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"((float)t));
  uint32_t r = (uint32_t)f;
  while ((uint64_t)r * r > t) --r;
  while ((uint64_t)(r + 1) * (r + 1) <= t) ++r;
  return r;
}
// min(65535, C / r) for C < 2^40, 1 <= r < 2^24: below 2^17 an approximate quotient (2 ulp) is off by less than 1
__device__ __forceinline__ uint32_t inverse16(uint64_t C, uint32_t r) {
  const float f = __fdividef((float)C, (float)r);
  uint32_t q = f >= 65536.0f ? 65536u : (uint32_t)f;
  while ((uint64_t)q * r > C) --q;
  while (q < 65536u && (uint64_t)(q + 1) * r <= C) ++q;
  return q < 65535u ? q : 65535u;
}

// two 32-bit values saturated to 8 bits, above the lower two bytes of `rest`
__device__ __forceinline__ uint32_t pack_sat8(int b, int a, uint32_t rest) {
  uint32_t d;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(b), "r"(a), "r"(rest));
  return d;
}

template <int D>
__global__ void __launch_bounds__(128) k_paged_append(const llx_paged_append_args a, const AppendSide sq, const AppendSide sk,
                                                      const int warps_per_row) {
  constexpr int L = D / 16, kHalf = D / 2, G = 32 / L;  // lanes per head; heads a warp takes at a time
  pdl_trigger();
  pdl_wait();
  const int64_t w = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int r = (int)(w / warps_per_row), first = (int)(w - (int64_t)r * warps_per_row);
  if (r >= a.rows) return;
  const int lane = threadIdx.x & 31, sub = lane % L;
  const int H = (int)a.n_heads, Hkv = (int)a.n_kv_heads;
  // groups of query heads, then of key heads, then 512-byte pieces of the values
  const int nq = (H + G - 1) / G, nk = nq + (Hkv + G - 1) / G, groups = nk + (Hkv * D + 511) / 512;
  auto fetch = [&](int g, uint4& lo, uint4& hi) {
    lo = hi = make_uint4(0, 0, 0, 0);
    if (g < nk) {
      const bool is_q = g < nq;
      const int h = (is_q ? g : g - nq) * G + lane / L;
      if (h < (is_q ? H : Hkv)) {
        const int16_t* x = (is_q ? sq.x + r * sq.stride : sk.x + r * sk.stride) + (int64_t)h * D + sub * 8;
        lo = *reinterpret_cast<const uint4*>(x);
        hi = *reinterpret_cast<const uint4*>(x + kHalf);
      }
    } else if (g < groups && (g - nk) * 512 + lane * 16 < Hkv * D) {
      lo = *reinterpret_cast<const uint4*>(a.v + r * a.v_stride + (g - nk) * 512 + lane * 16);
    }
  };
  uint4 lo, hi;
  fetch(first, lo, hi);
  const Place at = place_row(a, r);
  if (at.absent) return;
  int8_t* q8 = a.q8 + r * a.q8_stride;
  if (at.code) {
    if (first == 0 && lane == 0) raise_status(a.status, at.code);
    for (int x = first * 32 + lane; x < H * L; x += warps_per_row * 32) reinterpret_cast<uint4*>(q8)[x] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int P = (int)a.page_size, prow = (int)at.pos & (P - 1);
  const int64_t page0 = at.page * a.page_stride + (int64_t)prow * D;  // row of head 0
  int c[8], n[8];
  unpack8(*reinterpret_cast<const uint4*>(a.cos + at.pos * kHalf + sub * 8), c);
  unpack8(*reinterpret_cast<const uint4*>(a.sin + at.pos * kHalf + sub * 8), n);
  for (int g = first; g < groups; g += warps_per_row) {
    uint4 next_lo, next_hi;
    fetch(g + warps_per_row, next_lo, next_hi);
    if (g >= nk) {
      const int x = (g - nk) * 512 + lane * 16;
      if (x < Hkv * D) *reinterpret_cast<uint4*>(a.v_pages + page0 + (int64_t)(x / D) * P * D + x % D) = lo;
      lo = next_lo;
      continue;
    }
    const bool is_q = g < nq;
    const AppendSide& s = is_q ? sq : sk;
    const int h = (is_q ? g : g - nq) * G + lane / L;
    int x1[8], x2[8];
    unpack8(lo, x1);
    unpack8(hi, x2);
    if (s.gamma) {
      uint64_t ss = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += (uint32_t)(x1[j] * x1[j]) + (uint32_t)(x2[j] * x2[j]);  // 2^31 at most
#pragma unroll
      for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const uint32_t root = root48(ss + (uint64_t)s.eps);
      // |x g inv| < 2^46: 14 bits more keep it in 64 and put the result into the upper word
      const int inv = (int)(inverse16((uint64_t)s.C, root ? root : 1u) << 14), sh = s.shift + 14 - 32;
      int g1[8], g2[8];
      unpack8(*reinterpret_cast<const uint4*>(s.gamma + sub * 8), g1);
      unpack8(*reinterpret_cast<const uint4*>(s.gamma + kHalf + sub * 8), g2);
      const int64_t half = 1ll << (s.shift + 13);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x1[j] = clamp32((int)(((int64_t)(x1[j] * g1[j]) * inv + half) >> 32) >> sh, -32768, 32767);
        x2[j] = clamp32((int)(((int64_t)(x2[j] * g2[j]) * inv + half) >> 32) >> sh, -32768, 32767);
      }
    }
    // the rotated value saturates as y + 2^15 in [0, 2^16); the requantization takes the 2^15 back
    const int64_t half = (1ll << (s.S - 1)) - ((int64_t)s.M << 15);
    const int sh = s.S - 32;
    int z1[8], z2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // of 16-bit values x1 c - x2 s stays in 32 bits with the rounding; x2 c + x1 s can be 2^31, but not
      // with 2^14 less (and is -2^31 + 2^16 at least), which its quotient gets back as 1
      const int y1 = __viaddmin_s32_relu((x1[j] * c[j] - x2[j] * n[j] + 8192) >> 14, 32768, 65535);
      const int y2 = __viaddmin_s32_relu((x2[j] * c[j] - 8192 + x1[j] * n[j]) >> 14, 32769, 65535);
      z1[j] = (int)(((int64_t)y1 * s.M + half) >> 32) >> sh;
      z2[j] = (int)(((int64_t)y2 * s.M + half) >> 32) >> sh;
    }
    if (h < (is_q ? H : Hkv)) {
      uint32_t o1[2], o2[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        o1[j] = pack_sat8(z1[4 * j + 1], z1[4 * j], pack_sat8(z1[4 * j + 3], z1[4 * j + 2], 0));
        o2[j] = pack_sat8(z2[4 * j + 1], z2[4 * j], pack_sat8(z2[4 * j + 3], z2[4 * j + 2], 0));
      }
      int8_t* dst = is_q ? q8 + (int64_t)h * D : a.k_pages + page0 + (int64_t)h * P * D;
      *reinterpret_cast<uint2*>(dst + sub * 8) = make_uint2(o1[0], o1[1]);
      *reinterpret_cast<uint2*>(dst + kHalf + sub * 8) = make_uint2(o2[0], o2[1]);
    }
    lo = next_lo;
    hi = next_hi;
  }
}

template <int D>
static cudaError_t launch_append_t(const llx_paged_append_args& a, const AppendSide& q, const AppendSide& k, cudaStream_t st) {
  const int64_t G = 512 / D, groups = (a.n_heads + G - 1) / G + (a.n_kv_heads + G - 1) / G + (a.n_kv_heads * D + 511) / 512;
  // With many rows a warp takes several groups of one: the row's place is looked up and its rotation
  // unpacked once for them.
  int64_t per_row = groups;
  while (per_row > 1 && a.rows * per_row > 148 * 64) per_row = (per_row + 1) / 2;
  const int64_t blocks = (a.rows * per_row + 3) / 4;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_k(k_paged_append<D>, dim3((unsigned)blocks), dim3(128), 0, st, a, q, k, (int)per_row);
}

cudaError_t launch_paged_append(const llx_paged_append_args& a, cudaStream_t st) {
  if (a.rows == 0 || a.n_seqs == 0) return cudaSuccess;
  const AppendSide q{a.q, a.q_gamma, a.q_eps, a.q_C, a.q_stride, (int)a.q_shift, (int32_t)a.q_M, (int)a.q_S};
  const AppendSide k{a.k, a.k_gamma, a.k_eps, a.k_C, a.k_stride, (int)a.k_shift, (int32_t)a.k_M, (int)a.k_S};
  const void* ptrs[] = {a.q, a.k, a.v, a.q8, a.q_gamma, a.k_gamma, a.cos, a.sin, a.k_pages, a.v_pages};
  bool usual = a.q_stride % 8 == 0 && a.k_stride % 8 == 0 && a.v_stride % 16 == 0 && a.q8_stride % 16 == 0;
  for (const void* p : ptrs) usual = usual && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  for (const AppendSide* s : {&q, &k}) {
    usual = usual && s->S >= 32 && (s == &q ? a.q_M : a.k_M) < (1ll << 31);
    if (s->gamma) usual = usual && s->shift >= 18 && s->shift <= 46;
  }
  if (usual) switch (a.head_dim) {
      case 16: return launch_append_t<16>(a, q, k, st);
      case 32: return launch_append_t<32>(a, q, k, st);
      case 64: return launch_append_t<64>(a, q, k, st);
      case 128: return launch_append_t<128>(a, q, k, st);
      case 256: return launch_append_t<256>(a, q, k, st);
    }
  return launch_k(k_paged_append_any, dim3((unsigned)a.rows), dim3(256), 0, st, a);
}

// ---------------------------------------------------------------------------------------
// Page management.  One block plans (checks, counts, renames; a few thousand integers), then
// a grid copies the pages' rows.  Whatever the order of threads, the result is the same: new
// pages are the lowest free ids, handed out in the order of the lists.
// ---------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kMaxSlots = 1 << 18;  // slots of a table (bitmap of 32 KB)

// exclusive sum over the block; *total gets the whole
template <class T>
__device__ __forceinline__ T block_scan_of(T v, T* total) {
  __shared__ T part[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // part may still be read by an earlier call
  if (lane == 31) part[w] = x;
  __syncthreads();
  if (w == 0) {
    T y = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    part[lane] = y;
  }
  __syncthreads();
  *total = part[kPlanThreads / 32 - 1];
  return x - v + (w ? part[w - 1] : 0);
}
// of what slots ask for: 2^24 pages each, so the threads of one round for 2^34, and a request must not wrap
// into one that can be met
__device__ int64_t block_scan(int64_t v, int64_t* total) { return block_scan_of(v, total); }
// of what is known to be at most the cache's pages
__device__ int page_scan(int v, int* total) { return block_scan_of(v, total); }

__device__ __forceinline__ int64_t pages_for(int64_t len, int64_t P) { return (len + P - 1) / P; }

// positions of a slot as the table can hold them
__device__ __forceinline__ int64_t slot_length(const llx_pages_args& a, int slot) {
  const int64_t len = a.length[slot];
  return len < 0 ? 0 : (len > a.max_pages * a.page_size ? a.max_pages * a.page_size : len);
}

// The lists name slots of the table, each at most once in `once` (and, for a fork, none of
// them among `others`): checked with a bitmap of the slots.
__device__ bool lists_fine(const llx_pages_args& a, const int32_t* once, const int32_t* others) {
  __shared__ uint32_t seen[kMaxSlots / 32];
  __shared__ int bad;
  const int words = (int)((a.max_seqs + 31) / 32);
  for (int w = threadIdx.x; w < words; w += blockDim.x) seen[w] = 0;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.n; i += blockDim.x) {
    const int s = once[i];
    if (s < 0 || s >= a.max_seqs || (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1u) bad = 1;
  }
  __syncthreads();
  if (others)
    for (int64_t i = threadIdx.x; i < a.n; i += blockDim.x) {
      const int s = others[i];
      if (s < 0 || s >= a.max_seqs || (seen[s >> 5] >> (s & 31)) & 1u) bad = 1;
    }
  __syncthreads();
  return bad == 0;
}

// Releases (sign -1) or takes back (+1) every page of the listed slots; the entries stay.
__device__ void count_pages(const llx_pages_args& a, const int32_t* slots, int sign) {
  for (int64_t i = threadIdx.x >> 5; i < a.n; i += blockDim.x >> 5) {
    const int32_t* row = a.table + slots[i] * a.table_stride;
    for (int64_t j = threadIdx.x & 31; j < a.max_pages; j += 32) {
      const int id = row[j];
      if (id >= 0 && id < a.n_pages) atomicAdd(&a.refs[id], sign);
    }
  }
  __syncthreads();
}

// Writes the ids of the `need` lowest free pages to scratch; false if there are fewer.
__device__ bool take_free(const llx_pages_args& a, int64_t need) {
  const int64_t per = (a.n_pages + kPlanThreads - 1) / kPlanThreads;
  const int64_t p0 = threadIdx.x * per, p1 = p0 + per < a.n_pages ? p0 + per : a.n_pages;
  int mine = 0, have;
  for (int64_t p = p0; p < p1; ++p) mine += a.refs[p] <= 0;
  int at = page_scan(mine, &have);
  if (have < need) return false;
  for (int64_t p = p0; p < p1 && at < need; ++p)
    if (a.refs[p] <= 0) a.scratch[at++] = (int32_t)p;
  __syncthreads();
  return true;
}

// 64 slots, one position each, of 8,192 pages: 6.1 us in a graph, 10.8 a call from Python; the same block's
// chain as a fork's.
__global__ void __launch_bounds__(kPlanThreads) k_pages_reserve(const llx_pages_args a) {
  pdl_trigger();
  pdl_wait();
  __shared__ int code;
  if (threadIdx.x == 0) code = 0;
  __syncthreads();
  if (!lists_fine(a, a.list_a, nullptr)) {
    if (threadIdx.x == 0) raise_status(a.status, LLX_STATUS_BAD_SLOT);
    return;
  }
  const int64_t P = a.page_size;
  int64_t need = 0;
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int64_t i = i0 + threadIdx.x;
    int64_t mine = 0, sum;
    if (i < a.n) {
      const int s = a.list_a[i];
      const int64_t len = a.length[s], more = a.list_b[i];
      if (len < 0 || more < 0 || len + more > a.max_pages * P || len + more > INT32_MAX) {
        atomicOr(&code, LLX_STATUS_BAD_POSITION);
      } else {
        mine = pages_for(len + more, P) - pages_for(len, P);
        if (more && len % P) {
          const int id = a.table[s * a.table_stride + len / P];
          if (id < 0 || id >= a.n_pages) atomicOr(&code, LLX_STATUS_BAD_PAGE);
          else if (a.refs[id] > 1) atomicOr(&code, LLX_STATUS_SHARED_PAGE);
        }
      }
    }
    block_scan(mine, &sum);
    need += sum;
  }
  __syncthreads();
  if (code || !take_free(a, need)) {
    if (threadIdx.x == 0) raise_status(a.status, code ? code : LLX_STATUS_NO_PAGES);
    return;
  }
  int64_t base = 0;
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int64_t i = i0 + threadIdx.x;
    int s = 0, mine = 0, sum;
    int64_t len = 0;
    if (i < a.n) {
      s = a.list_a[i];
      len = a.length[s];
      mine = (int)(pages_for(len + a.list_b[i], P) - pages_for(len, P));
    }
    const int64_t at = base + page_scan(mine, &sum);
    for (int j = 0; j < mine; ++j) {
      const int id = a.scratch[at + j];
      a.table[s * a.table_stride + pages_for(len, P) + j] = id;
      a.refs[id] = 1;
    }
    if (i < a.n) a.length[s] = (int32_t)(len + a.list_b[i]);
    base += sum;
  }
}

// Not all or nothing: the good slots of a list are freed, the others noted.  2.2 us in a graph for 64 slots.
__global__ void __launch_bounds__(kPlanThreads) k_pages_free(const llx_pages_args a) {
  pdl_trigger();
  pdl_wait();
  const int64_t total = a.n * a.max_pages;
  for (int64_t x = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; x < total; x += (int64_t)gridDim.x * blockDim.x) {
    const int s = a.list_a[x / a.max_pages];
    if (s < 0 || s >= a.max_seqs) {
      raise_status(a.status, LLX_STATUS_BAD_SLOT);
      continue;
    }
    // a slot listed twice still gives each page back once
    const int id = atomicExch(&a.table[s * a.table_stride + x % a.max_pages], -1);
    if (id >= 0 && id < a.n_pages) atomicSub(&a.refs[id], 1);
    a.length[s] = 0;
  }
}

// Children become copies of their parents; the copying itself is k_pages_copy's.  One block decides, so
// the call is all or nothing without a wait between blocks: 48 children of sequences of 500 to 1,100
// positions take 16.1 us with the copying (20 MB, 3 us), most of it this block's chain of scans.
__global__ void __launch_bounds__(kPlanThreads) k_pages_fork(const llx_pages_args a) {
  pdl_trigger();
  pdl_wait();
  // scratch: the copies' targets [0, N), sources [N, 2N) and rows [2N, 3N), and [3N] their number
  int32_t* done = a.scratch + 3 * a.n_pages;
  __shared__ int bad;  // a page to be copied is not there
  if (threadIdx.x == 0) bad = 0;
  if (!lists_fine(a, a.list_b, a.list_a)) {
    if (threadIdx.x == 0) {
      raise_status(a.status, LLX_STATUS_BAD_SLOT);
      *done = 0;
    }
    return;
  }
  const int64_t P = a.page_size;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // what is to be copied has to be there, before anything is changed
  auto there = [&](int slot, int64_t j) {
    const int id = a.table[slot * a.table_stride + j];
    if (id < 0 || id >= a.n_pages) bad = 1;
  };
  int64_t need = 0;
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int64_t i = i0 + threadIdx.x;
    int64_t mine = 0, sum;
    if (i < a.n) {
      const int64_t len = slot_length(a, a.list_a[i]);
      mine = pages_for(len, P) - (a.share ? len / P : 0);
      if (a.share && mine) there(a.list_a[i], len / P);
    }
    block_scan(mine, &sum);
    need += sum;
  }
  if (!a.share) {
    for (int64_t i = warp; i < a.n; i += kPlanThreads / 32) {
      const int64_t held = pages_for(slot_length(a, a.list_a[i]), P);
      for (int64_t j = lane; j < held; j += 32) there(a.list_a[i], j);
    }
    __syncthreads();
  }
  if (bad) {  // block_scan's barriers lie between
    if (threadIdx.x == 0) {
      raise_status(a.status, LLX_STATUS_BAD_PAGE);
      *done = 0;
    }
    return;
  }
  count_pages(a, a.list_b, -1);
  if (!take_free(a, need)) {
    count_pages(a, a.list_b, 1);
    if (threadIdx.x == 0) {
      raise_status(a.status, LLX_STATUS_NO_PAGES);
      *done = 0;
    }
    return;
  }
  __shared__ int first[kPlanThreads];
  int64_t base = 0;
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int64_t i = i0 + threadIdx.x;
    int mine = 0, sum;
    if (i < a.n) {
      const int64_t len = slot_length(a, a.list_a[i]);
      mine = (int)(pages_for(len, P) - (a.share ? len / P : 0));
    }
    first[threadIdx.x] = page_scan(mine, &sum);
    __syncthreads();
    for (int64_t x = warp; x < kPlanThreads && i0 + x < a.n; x += kPlanThreads / 32) {
      const int from = a.list_a[i0 + x], to = a.list_b[i0 + x];
      const int64_t len = slot_length(a, from), held = pages_for(len, P), kept = a.share ? len / P : 0;
      for (int64_t j = lane; j < a.max_pages; j += 32) {
        int id = -1;
        if (j < kept) {
          id = a.table[from * a.table_stride + j];
          if (id >= 0 && id < a.n_pages) atomicAdd(&a.refs[id], 1);
        } else if (j < held) {
          const int64_t m = base + first[x] + j - kept;
          id = a.scratch[m];
          a.refs[id] = 1;
          a.scratch[a.n_pages + m] = a.table[from * a.table_stride + j];
          a.scratch[2 * a.n_pages + m] = (int)min(P, len - j * P);
        }
        a.table[to * a.table_stride + j] = id;
      }
      if (lane == 0) a.length[to] = (int32_t)len;
    }
    base += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) *done = (int32_t)need;
}

// Copies pages: block (x, y) takes moves x, x + gridDim.x, ... of layer y / 2, k or v.  `rows` null:
// whole pages.  Four 16-byte loads per thread are under way before the first is stored; a page of 16 KB
// per layer is one round.  Bytes bound it: 359 MB copied in 59 us, 0.94 of the copy rate; in place, where
// pages move within one range (compact, 405 MB), 75 us, 0.82.
__global__ void __launch_bounds__(256) k_pages_copy(const llx_pages_args a, const int32_t* src, const int32_t* dst,
                                                    const int32_t* rows, const int32_t* number,
                                                    const int32_t* names) {
  pdl_trigger();
  pdl_wait();
  const int moves = *number;
  if (names && blockIdx.y == 0) {  // the table with the pages' new names
    const int64_t entries = a.max_seqs * a.max_pages;
    for (int64_t x = blockIdx.x * 256ll + threadIdx.x; x < entries; x += gridDim.x * 256ll) {
      const int64_t at = x / a.max_pages * a.table_stride + x % a.max_pages;
      const int id = a.table[at];
      a.new_table[at] = id >= 0 && id < a.n_pages ? names[id] : id;
    }
  }
  const int64_t head = a.page_size * a.head_dim;
  const int whole = (int)(a.n_kv_heads * head / 16);
  for (int64_t y = blockIdx.y; y < 2 * a.n_layers; y += gridDim.y) {
    int8_t* pool = ((y & 1) ? a.v : a.k) + (y >> 1) * a.layer_stride;
    for (int m = blockIdx.x; m < moves; m += gridDim.x) {
      const int from = src[m], to = dst[m], held = rows ? rows[m] : (int)a.page_size;
      if (from < 0 || from >= a.n_pages) {
        if (threadIdx.x == 0) raise_status(a.status, LLX_STATUS_BAD_PAGE);
        continue;
      }
      auto copy = [&](const int8_t* s8, int8_t* d8, int vecs) {
        const uint4* s = reinterpret_cast<const uint4*>(s8);
        uint4* d = reinterpret_cast<uint4*>(d8);
        for (int e = threadIdx.x; e < vecs; e += 4 * 256) {
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (e + j * 256 < vecs) v[j] = s[e + j * 256];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (e + j * 256 < vecs) d[e + j * 256] = v[j];
        }
      };
      const int8_t* s = pool + from * a.page_stride;
      int8_t* d = pool + to * a.page_stride;
      if (held == a.page_size)
        copy(s, d, whole);
      else
        for (int h = 0; h < a.n_kv_heads; ++h) copy(s + h * head, d + h * head, (int)(held * a.head_dim / 16));
    }
  }
}

// The pages from id `live` on move, in order, into the free pages below; the others stay where they are.
// scratch: [0, N) new id of each page, [N, 2N) holes then sources of the moves, [2N, 3N) their
// targets, [3N] number of moves
__global__ void __launch_bounds__(kPlanThreads) k_pages_compact(const llx_pages_args a) {
  pdl_trigger();
  pdl_wait();
  const int64_t N = a.n_pages, per = (N + kPlanThreads - 1) / kPlanThreads;
  const int64_t p0 = min(N, threadIdx.x * per), p1 = min(N, p0 + per);
  int32_t *to = a.scratch, *src = to + N, *dst = src + N;
  int used = 0, live;
  for (int64_t p = p0; p < p1; ++p) used += a.refs[p] > 0;
  const int before = page_scan(used, &live);  // live pages below p0
  // movers: live pages from id `live` on; holes: free pages below it; as many of each.  Of the pages
  // below `live`, those that are not live are holes; of the live pages, those past the ones below it move.
  __shared__ int live_below;  // live pages with an id below `live`
  if (p0 <= live && live < p1 + (p1 == N)) {
    int n = before;
    for (int64_t p = p0; p < p1 && p < live; ++p) n += a.refs[p] > 0;
    live_below = n;
  }
  __syncthreads();
  const int moves = live - live_below;
  int n = before;
  for (int64_t p = p0; p < p1; ++p) {
    const bool l = a.refs[p] > 0;
    if (!l && p < live) dst[p - n] = (int32_t)p;  // free pages below p
    if (l && p >= live) src[n - live_below] = (int32_t)p;
    n += l;
    to[p] = (int32_t)p;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < moves; x += blockDim.x) to[src[x]] = dst[x];
  // counts: every page reads its old count before any is written (new_refs may be refs)
  for (int x = threadIdx.x; x < moves; x += blockDim.x) a.new_refs[dst[x]] = a.refs[src[x]];
  for (int64_t p = p0; p < p1; ++p)
    if (a.refs[p] > 0 && p < live && to[p] == p) a.new_refs[p] = a.refs[p];
  __syncthreads();
  for (int64_t p = live + threadIdx.x; p < N; p += blockDim.x) a.new_refs[p] = 0;
  if (threadIdx.x == 0) to[3 * N] = moves;
}

static unsigned copy_grid(int64_t units) { return (unsigned)(units < 1 ? 1 : units > 148 * 8 ? 148 * 8 : units); }

cudaError_t launch_pages_reserve(const llx_pages_args& a, cudaStream_t st) {
  if (a.n == 0) return cudaSuccess;
  return launch_k(k_pages_reserve, dim3(1), dim3(kPlanThreads), 0, st, a);
}

cudaError_t launch_pages_free(const llx_pages_args& a, cudaStream_t st) {
  if (a.n == 0) return cudaSuccess;
  const int64_t blocks = (a.n * a.max_pages + kPlanThreads - 1) / kPlanThreads;
  return launch_k(k_pages_free, dim3(copy_grid(blocks)), dim3(kPlanThreads), 0, st, a);
}

// enough blocks for 8 on an SM, whichever of moves and layers there are more of
static dim3 copy_blocks(int64_t moves, int64_t layers) {
  const int64_t y = 2 * layers < 65535 ? 2 * layers : 65535, most = (148 * 8 + y - 1) / y;
  return dim3((unsigned)(moves < most ? (moves < 1 ? 1 : moves) : most), (unsigned)y);
}

cudaError_t launch_pages_fork(const llx_pages_args& a, cudaStream_t st) {
  if (a.n == 0) return cudaSuccess;
  const cudaError_t e = launch_k(k_pages_fork, dim3(1), dim3(kPlanThreads), 0, st, a);
  if (e != cudaSuccess) return e;
  const int64_t N = a.n_pages, most = a.share ? a.n : a.n * a.max_pages;
  return launch_k(k_pages_copy, copy_blocks(most < N ? most : N, a.n_layers), dim3(256), 0, st, a,
                  (const int32_t*)a.scratch + N, (const int32_t*)a.scratch, (const int32_t*)a.scratch + 2 * N,
                  (const int32_t*)a.scratch + 3 * N, (const int32_t*)nullptr);
}

cudaError_t launch_pages_compact(const llx_pages_args& a, cudaStream_t st) {
  const cudaError_t e = launch_k(k_pages_compact, dim3(1), dim3(kPlanThreads), 0, st, a);
  if (e != cudaSuccess) return e;
  const int64_t N = a.n_pages;
  return launch_k(k_pages_copy, copy_blocks(N / 2, a.n_layers), dim3(256), 0, st, a, (const int32_t*)a.scratch + N,
                  (const int32_t*)a.scratch + 2 * N, (const int32_t*)nullptr, (const int32_t*)a.scratch + 3 * N, (const int32_t*)a.scratch);
}

}  // namespace llx
