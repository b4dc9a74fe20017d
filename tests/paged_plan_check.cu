// Compiles the real page-management kernels: a launch's page counts add up in 64 bits.
#include "kernels_paged.cu"

#include <type_traits>

// 1,024 slots of a round may ask for 2^24 pages each
static_assert(std::is_same<decltype(&llx::block_scan), int64_t (*)(int64_t, int64_t*)>::value, "page counts wrap");
static_assert(1024ll << 24 > INT32_MAX, "");
