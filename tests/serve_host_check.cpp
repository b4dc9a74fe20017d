// The serving calls' host code (runtime.cu) over a fake CUDA runtime: device memory is host memory, kernels
// do nothing, and the n-th operation of a call can be made to fail.  test_serve_host.py builds it.
#include <cuda_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "llx.h"

static int ops = 0, fail_at = 0;  // operations of the call under test; the one that fails (0: none)
static cudaError_t fail_with = cudaSuccess;
static bool reserved;  // the call under test has begun to change slots
static bool no_pages, bad_page, lost;

static cudaError_t tick() { return ++ops == fail_at ? fail_with : cudaSuccess; }

extern "C" {
int fake_launch() { return (int)tick(); }
cudaError_t cudaGetDeviceCount(int* n) { return *n = 1, cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) {
  *v = a == cudaDevAttrMultiProcessorCount ? 148 : a == cudaDevAttrComputeCapabilityMajor ? 10 : 1 << 18;
  return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t n) {
  const cudaError_t e = tick();
  *p = e == cudaSuccess ? calloc(1, n) : nullptr;
  return e;
}
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { return cudaMalloc(p, n); }
cudaError_t cudaFree(void* p) { return free(p), cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { return free(p), cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) {
  const cudaError_t e = n && !(d && s) ? cudaErrorInvalidValue : tick();
  if (e == cudaSuccess && n) memcpy(d, s, n);
  return e;
}
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind k) { return cudaMemcpyAsync(d, s, n, k, nullptr); }
cudaError_t cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t) {
  const cudaError_t e = tick();
  if (e == cudaSuccess) memset(d, v, n);
  return e;
}
cudaError_t cudaMemset(void* d, int v, size_t n) { return cudaMemsetAsync(d, v, n, nullptr); }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return tick(); }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { return *s = nullptr, cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "injected"; }
size_t llx_pages_scratch(int64_t n) { return (size_t)(3 * n + 4) * sizeof(int32_t); }
}

namespace llx {
int g_pdl = 0;
int64_t sample_max_vocab() { return 1 << 18; }
int sab_rows_per_tile(int) { return 64; }
cudaError_t launch_pages_reserve(const llx_pages_args& a, cudaStream_t) {
  const cudaError_t e = tick();
  if (e != cudaSuccess) return e;
  if (lost) *a.status |= LLX_STATUS_LOST;
  if (no_pages)
    *a.status |= LLX_STATUS_NO_PAGES;
  else
    reserved = true;
  return e;
}
cudaError_t launch_pages_fork(const llx_pages_args& a, cudaStream_t) {
  const cudaError_t e = tick();
  if (e != cudaSuccess) return e;
  if (bad_page)
    *a.status |= LLX_STATUS_BAD_PAGE;
  else
    reserved = true;
  return e;
}
}  // namespace llx

static int failures = 0;
#define CHECK(x)                                                                                   \
  do {                                                                                             \
    if (!(x)) {                                                                                    \
      ++failures;                                                                                  \
      printf("line %d, operation %d, error %d: %s (%s)\n", __LINE__, fail_was, with, #x, llx_last_error()); \
    }                                                                                              \
  } while (0)

static int fail_was = 0, with = 0;

// runs f with its n-th operation failing
template <class F>
static llx_status failing(int n, cudaError_t e, F f) {
  ops = 0;
  fail_was = fail_at = n;
  fail_with = e;
  with = (int)e;
  reserved = false;
  const llx_status r = f();
  fail_at = 0;
  return r;
}

struct Serve {
  llx_serve* h = nullptr;
  llx_model* m;
  int vp;
  std::vector<int16_t> logits;
  explicit Serve(llx_model* model, int pages = 32) : m(model) {
    llx_model_info i;
    llx_model_get_info(m, &i);
    vp = i.vocab_padded;
    if (llx_serve_create(m, 5, pages, 16, 64, &h) != LLX_OK) printf("create: %s\n", llx_last_error()), exit(1);
  }
  ~Serve() { llx_serve_destroy(h); }
  llx_status step(std::vector<int32_t> slots, int count = 3, bool sampled = true, bool with_logits = true) {
    const int n = (int)slots.size();
    std::vector<int32_t> counts(n, count), tokens(n * count, 1), next(n);
    std::vector<double> u(n, 0.5);
    std::vector<float> t(n, 1.0f), prob(n);
    llx_sampling how{u.data(), t.data(), nullptr, t.data(), nullptr};
    logits.resize((size_t)n * vp);
    return llx_serve_step(h, n, slots.data(), counts.data(), tokens.data(), sampled ? &how : nullptr, next.data(),
                          sampled ? prob.data() : nullptr, with_logits ? logits.data() : nullptr);
  }
  llx_status fork(std::vector<int32_t> p, std::vector<int32_t> c, int share = 1) {
    return llx_serve_fork(h, (int)p.size(), p.data(), c.data(), share);
  }
  llx_status release(std::vector<int32_t> s) { return llx_serve_free(h, (int)s.size(), s.data()); }
  int len(int slot) {
    int32_t l[5];
    return llx_serve_usage(h, l, nullptr) == LLX_OK ? l[slot] : -1;
  }
};

// a step that fails after its pages were taken leaves its slots closed until they are freed, and nothing else
static void steps(llx_model* m, cudaError_t e, bool sampled) {
  for (int n = 1;; ++n) {
    Serve s(m);
    CHECK(s.step({0, 2}) == LLX_OK);
    const llx_status r = failing(n, e, [&] { return s.step({0, 1}, 3, sampled); });
    if (r == LLX_OK) {
      CHECK(n > 20 && s.len(0) == 6 && s.len(1) == 3);  // every operation has had its turn
      return;
    }
    if (!reserved) {
      CHECK(s.len(0) == 3 && s.len(1) == 0);
      CHECK(s.step({0, 1}) == LLX_OK && s.len(0) == 6 && s.len(1) == 3);
      continue;
    }
    CHECK(r != LLX_ERR_OOM);  // it says that nothing was changed
    CHECK(s.step({0}) == LLX_ERR_INVALID && s.step({1, 2}) == LLX_ERR_INVALID);
    CHECK(s.fork({0}, {3}) == LLX_ERR_INVALID);
    CHECK(s.step({2}) == LLX_OK && s.len(2) == 6);
    CHECK(s.fork({2}, {1}) == LLX_OK && s.step({1}) == LLX_OK && s.len(1) == 9);  // a copy of another sequence
    CHECK(s.step({0}) == LLX_ERR_INVALID);
    CHECK(s.release({0}) == LLX_OK && s.len(0) == 0 && s.step({0}) == LLX_OK && s.len(0) == 3);
  }
}

static void too_few_pages(llx_model* m) {
  Serve s(m, 2);
  CHECK(s.step({0, 1}) == LLX_OK);
  no_pages = true;
  CHECK(s.step({0, 2}) == LLX_ERR_OOM && s.len(0) == 3 && s.len(2) == 0);
  no_pages = false;
  CHECK(s.step({0, 1}) == LLX_OK && s.len(0) == 6);
}

static void forks(llx_model* m, cudaError_t e) {
  for (int n = 1;; ++n) {
    Serve s(m);
    CHECK(s.step({0, 1}) == LLX_OK);
    const llx_status r = failing(n, e, [&] { return s.fork({0}, {3}); });
    const bool begun = reserved;
    if (r == LLX_OK) {
      CHECK(n > 3 && s.len(3) == 3);
      break;
    }
    CHECK(s.step({0, 1}) == LLX_OK);
    if (!begun) {
      CHECK(s.fork({1}, {3}) == LLX_OK && s.len(3) == 6);
      continue;
    }
    CHECK(r != LLX_ERR_OOM);
    CHECK(s.step({3}) == LLX_ERR_INVALID && s.fork({3}, {4}) == LLX_ERR_INVALID);
    CHECK(s.release({3}) == LLX_OK && s.step({3}) == LLX_OK && s.len(3) == 3);
  }
  Serve s(m);  // refused on the device: the fork itself says so, and the child is as it was
  CHECK(s.step({0, 3}) == LLX_OK && s.step({3}) == LLX_OK);
  bad_page = true;
  CHECK(s.fork({0}, {3}) == LLX_ERR_DEVICE);
  bad_page = false;
  CHECK(s.len(3) == 6 && s.step({0, 3}) == LLX_OK && s.len(3) == 9);
}

// pages may have moved and the table not: the handle is of no more use
static void compactions(llx_model* m, cudaError_t e) {
  for (int n = 1;; ++n) {
    Serve s(m);
    CHECK(s.step({0}) == LLX_OK);
    const llx_status r = failing(n, e, [&] { return llx_serve_compact(s.h); });
    if (r == LLX_OK) {
      CHECK(n > 1 && s.step({0}) == LLX_OK);
      return;
    }
    CHECK(r != LLX_ERR_OOM);
    CHECK(s.step({0}) == LLX_ERR_INVALID && s.step({1}) == LLX_ERR_INVALID && s.fork({0}, {1}) == LLX_ERR_INVALID);
    CHECK(llx_serve_compact(s.h) == LLX_ERR_INVALID && s.release({0}) == LLX_ERR_INVALID);
  }
}

// what a failed step's kernels have noted is its own: the calls after it neither fail by it nor take it for
// a refusal of theirs
static void notes(llx_model* m) {
  for (int fork = 0; fork < 2; ++fork)
    for (int n = 1; n < 60; ++n) {
      Serve s(m);
      CHECK(s.step({0, 2}) == LLX_OK);
      lost = true;
      CHECK(failing(n, cudaErrorLaunchOutOfResources, [&] { return s.step({0, 1}); }) != LLX_OK);
      lost = false;
      if (fork)
        CHECK(s.fork({2}, {3}) == LLX_OK && s.len(3) == 3 && s.step({3}) == LLX_OK);
      else
        CHECK(s.step({2}) == LLX_OK && s.len(2) == 6);
    }
}

// a buffer that could not be made larger is not taken for the one it was
static void logits_buffer(llx_model* m) {
  for (int n = 1; n < 5; ++n) {
    Serve s(m);
    CHECK(s.step({0}) == LLX_OK);
    if (failing(n, cudaErrorMemoryAllocation, [&] { return s.step({0, 1}); }) == LLX_OK) break;
    CHECK(!reserved && s.step({0}) == LLX_OK && s.step({0, 1}) == LLX_OK);
  }
}

int main(int argc, char** argv) {
  llx_model* m = nullptr;
  if (argc < 2 || llx_model_load(argv[1], nullptr, &m) != LLX_OK) return printf("load: %s\n", llx_last_error()), 1;
  for (const cudaError_t e : {cudaErrorMemoryAllocation, cudaErrorLaunchOutOfResources}) {
    steps(m, e, true);
    steps(m, e, false);
    forks(m, e);
    compactions(m, e);
  }
  too_few_pages(m);
  logits_buffer(m);
  notes(m);
  llx_model_destroy(m);
  printf("%d failures\n", failures);
  return failures != 0;
}
