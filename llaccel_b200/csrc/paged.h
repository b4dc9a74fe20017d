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
// A warp's lanes try 32 entries a round: one round of loads for 32 sequences, two for 1024.
__device__ __forceinline__ int find_sequence(const int32_t* q_start, int n, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, width = 1;  // entries lo, lo + width, ... are tried; q_start[lo] <= r from the second round on
  while (width * 32 <= n) width *= 32;
  for (;;) {
    const int at = lo + lane * width;
    const uint32_t below = __ballot_sync(0xffffffffu, at <= n && q_start[at] <= r);
    if (!below) return -1;
    // starts ascend, so the tries that are at most r come first
    lo += (31 - __clz(below)) * width;
    if (width == 1) break;
    width /= 32;
  }
  return lo < n ? lo : -1;
}

__device__ __forceinline__ void raise_status(int32_t* status, int code) {
  if (status) atomicOr(status, code);
}

}  // namespace llx
