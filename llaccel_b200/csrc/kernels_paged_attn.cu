// Causal GQA integer-softmax attention of a ragged launch over a paged int8 cache
// (numerics.h:88-120, golden.py:353-366): every row's maximum over all its keys, then the sum of
// the table exponentials, then the normalised integer weights times the values.  Max and sums are
// integer, so any split of the keys gives the reference's bits.
#include <cuda_runtime.h>

#include "paged_attn.cuh"

namespace llx {

template <typename T, typename Op>
__device__ __forceinline__ T reduce_block(T v, T* scratch, Op op) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) scratch[w] = v;
  __syncthreads();
  T r = scratch[0];
  for (int i = 1; i < nw; ++i) r = op(r, scratch[i]);
  return r;
}

// Any geometry (head sizes other than 64 and 128, more sequences than a grid axis holds): one block per
// (row, query head), three passes over the keys, scores recomputed.  It reads a row's keys three times for
// every query head and has no reuse between rows: 57.7 ms where the chunk kernel takes 0.27; 64 single tokens
// of 1,000 keys, 14 heads on 2 of 80, 184 us for 20 MB.
__global__ void __launch_bounds__(256) k_paged_attention_any(const llx_paged_attention_args a) {
  pdl_trigger();
  pdl_wait();
  __shared__ __align__(16) int8_t q_s[256];
  __shared__ int32_t pn_s[256];
  __shared__ int32_t acc_s[256];
  __shared__ long long red[8];
  __shared__ uint16_t expi[16], expf[256];
  const int r = blockIdx.x, h = blockIdx.y;
  const int D = (int)a.head_dim, rep = (int)(a.n_heads / a.n_kv_heads), kvh = h / rep;
  const int i = find_sequence(a.q_start, (int)a.n_seqs, r);
  if (i < 0) return;
  const SeqView sv = view_sequence(a, i);
  const int64_t P = a.page_size;
  int code = sv.code;
  // keys 0 .. T - 1; the bounds of the call and of the page table cut both
  int64_t T = sv.slot < 0 ? 0 : (int64_t)sv.len - sv.rows + (r - sv.first) + 1;
  if (T <= 0 && !code) code = LLX_STATUS_BAD_POSITION;
  if (r - sv.first >= a.max_rows) {
    if (threadIdx.x == 0) raise_status(a.status, LLX_STATUS_BAD_BOUND);
    return;
  }
  const int64_t cap = min(a.max_len, a.max_pages * P);
  if (T > cap) {
    code |= LLX_STATUS_BAD_BOUND;
    T = cap;
  }
  for (int e = threadIdx.x; e < D; e += blockDim.x) q_s[e] = a.q8[r * a.q8_stride + h * D + e];
  expf[threadIdx.x] = kDevExpF[threadIdx.x];
  if (threadIdx.x < 16) expi[threadIdx.x] = kDevExpI[threadIdx.x];
  acc_s[threadIdx.x] = 0;
  __syncthreads();
  const int32_t* pages = a.table + (sv.slot < 0 ? 0 : sv.slot) * a.table_stride;
  bool bad = false;
  auto page_of = [&](int64_t t) {
    const int id = pages[t / P];
    return id < 0 || id >= a.n_pages ? (int64_t)-1 : id * a.page_stride + (kvh * P + t % P) * D;
  };
  auto score = [&](int64_t at) {
    const uint4* k = reinterpret_cast<const uint4*>(a.k_pages + at);
    int s = 0;
    for (int c = 0; c < D / 16; ++c) {
      const uint4 x = k[c], y = reinterpret_cast<const uint4*>(q_s)[c];
      s = __dp4a((int)x.x, (int)y.x, s);
      s = __dp4a((int)x.y, (int)y.y, s);
      s = __dp4a((int)x.z, (int)y.z, s);
      s = __dp4a((int)x.w, (int)y.w, s);
    }
    return s;
  };
  long long mx = LLONG_MIN;
  for (int64_t t = threadIdx.x; t < T; t += blockDim.x) {
    const int64_t at = page_of(t);
    if (at < 0)
      bad = true;
    else
      mx = max(mx, (long long)score(at));
  }
  if (bad) code |= LLX_STATUS_BAD_PAGE;
  if (code) raise_status(a.status, code);
  mx = reduce_block<long long>(mx, red, [](long long x, long long y) { return x > y ? x : y; });
  long long sum = 0;
  for (int64_t t = threadIdx.x; t < T; t += blockDim.x) {
    const int64_t at = page_of(t);
    if (at >= 0) sum += exp_prob(mulshift(mx - score(at), a.Ms, (int)a.Ss), expi, expf);
  }
  sum = reduce_block<long long>(sum, red, [](long long x, long long y) { return x + y; });
  const int64_t inv = (int64_t)(((uint64_t)1 << 31) / (uint64_t)(sum ? sum : 1));
  const int64_t pmax = (1 << a.prob_bits) - 1;
  const int groups = 256 / D, d = threadIdx.x % D, g = threadIdx.x / D;
  int32_t acc = 0;
  for (int64_t t0 = 0; t0 < T; t0 += 256) {
    const int64_t t = t0 + threadIdx.x;
    int32_t pn = 0;
    if (t < T) {
      const int64_t at = page_of(t);
      if (at >= 0) {
        const int64_t p = exp_prob(mulshift(mx - score(at), a.Ms, (int)a.Ss), expi, expf);
        pn = (int32_t)min(rshr(p * inv, 31 - (int)a.prob_bits), pmax);
      }
    }
    __syncthreads();
    pn_s[threadIdx.x] = pn;
    __syncthreads();
    if (g < groups)
      for (int x = g; x < 256 && t0 + x < T; x += groups)
        if (pn_s[x]) acc += pn_s[x] * a.v_pages[page_of(t0 + x) + d];  // pn > 0: its page is there
  }
  __syncthreads();
  if (g < groups) atomicAdd(&acc_s[d], acc);  // integer: any order
  __syncthreads();
  for (int e = threadIdx.x; e < D; e += blockDim.x) {
    int64_t o = acc_s[e];
    if (a.prob_bits == 15) o = rshr(o, 7);
    a.out[r * a.out_stride + h * D + e] = (int8_t)sat8(mulshift(o, a.Mo, (int)a.So));
  }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t make_page_map(CUtensorMap* map, const void* base, const llx_paged_attention_args& a, int box_rows) {
  static const EncodeTiled encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)(a.n_kv_heads * a.page_size), (cuuint64_t)a.n_pages};
  const cuuint64_t strides[2] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.page_stride};
  const cuuint32_t box[3] = {(cuuint32_t)a.head_dim, (cuuint32_t)box_rows, 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            a.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t launch_paged_attention(const llx_paged_attention_args& args, cudaStream_t st) {
  llx_paged_attention_args a = args;
  if (a.max_rows > a.rows) a.max_rows = a.rows;  // grids follow it
  if (a.rows == 0 || a.n_seqs == 0 || a.max_rows == 0) return cudaSuccess;
  const int64_t pairs = a.max_rows * (a.n_heads / a.n_kv_heads);
  // Up to 32 stacked pairs the cache is read once per 8 of them by the few-row kernel; from there on, and in
  // launches that mix prompt chunks with single tokens, the chunk kernel takes every sequence.  For mixed
  // launches two were measured: 30 single tokens of at most 2,300 keys beside 2 chunks, 2 KV heads of 64, 74 us
  // against 102 for a kernel each; 30 of 4,500 keys beside a chunk of 500, 8 KV heads of 128, 275 against 156
  // (84 and 72 alone).  So the rule loses where single tokens have long contexts.
  // It also steps at both of its bounds: 4 sequences of 4 draft rows (28 pairs) over 1,100 keys take 12 us,
  // of 5 rows (35 pairs) 26; and see paged_decode_fits for max_len.
  constexpr int kFew = 32;
  if (paged_chunk_fits(a)) return pairs <= kFew && paged_decode_fits(a, pairs) ? launch_paged_decode(a, st) : launch_paged_chunk(a, st);
  return launch_k(k_paged_attention_any, dim3((unsigned)a.rows, (unsigned)a.n_heads), dim3(256), 0, st, a);
}

}  // namespace llx
