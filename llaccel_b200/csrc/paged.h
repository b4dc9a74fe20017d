// Launch wrappers of the paged-serving kernels: appending a launch's rows to a paged int8 cache,
// chunk attention over the pages, page management, and sampling from integer logits.
// Arguments are the C structs of include/llx.h, checked by the entry points in paged.cu.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/llx.h"

namespace llx {

cudaError_t launch_paged_append(const llx_paged_append_args& a, cudaStream_t st);
cudaError_t launch_paged_attention(const llx_paged_attention_args& a, cudaStream_t st);
cudaError_t launch_pages_reserve(const llx_pages_args& a, cudaStream_t st);
cudaError_t launch_pages_fork(const llx_pages_args& a, cudaStream_t st);
cudaError_t launch_pages_free(const llx_pages_args& a, cudaStream_t st);
cudaError_t launch_pages_compact(const llx_pages_args& a, cudaStream_t st);
cudaError_t launch_sample(const llx_sample_args& a, cudaStream_t st);

// vocabulary entries one sampling launch can hold on chip
int64_t sample_max_vocab();

// ---- device helpers shared by append and attention ------------------------------------------
// A launch row's place: sequence i with q_start[i] <= r < q_start[i + 1]; -1 behind the last one.
__device__ __forceinline__ int find_sequence(const int32_t* q_start, int n, int r) {
  if (r >= q_start[n] || r < q_start[0]) return -1;
  int lo = 0, hi = n;  // q_start[lo] <= r < q_start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (q_start[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void raise_status(int32_t* status, int code) {
  if (status) atomicOr(status, code);
}

}  // namespace llx
