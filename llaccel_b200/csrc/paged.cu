// C entry points of the paged-serving calls (include/llx.h): argument checks, then one enqueue on
// the caller's stream.  Nothing is allocated, synchronised or remembered between calls.
#include "paged.h"

#include <climits>
#include <string>

namespace llx {

void noalloc_set_error(const std::string& msg);  // the thread's llx_last_error text

namespace {

struct Refused {
  llx_status code;
  std::string what;
};

void need(bool ok, const char* what, llx_status code = LLX_ERR_INVALID) {
  if (!ok) throw Refused{code, what};
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void need_rq(int64_t M, int64_t S, const char* what) {
  need(M >= 0 && M <= 0xFFFFFFFFll && S >= 0 && S <= 63, what);
}

void need_cache(int64_t n_pages, int64_t page_size, int64_t n_kv_heads, int64_t head_dim, int64_t page_stride) {
  need(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0, "head_dim must be a multiple of 16 up to 256");
  need(page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0,
       "page_size must be a power of two of 16 to 256");
  need(n_kv_heads >= 1 && n_kv_heads <= 1024, "n_kv_heads must be 1 to 1024");
  need(n_pages >= 1 && n_pages <= 0x7FFFFFFF, "n_pages must be at least 1");
  need(page_stride >= n_kv_heads * page_size * head_dim && page_stride % 16 == 0,
       "page_stride must cover a page and be a multiple of 16 bytes");
}

void need_table(const void* table, int64_t stride, int64_t max_seqs, int64_t max_pages) {
  need(table != nullptr, "null page table");
  need(max_seqs >= 1 && max_seqs <= (1 << 18), "max_seqs must be 1 to 262144");
  need(max_pages >= 1 && max_pages <= (1 << 24) && stride >= max_pages, "the page table needs 1 to 2^24 pages a row and its stride to cover them");
}

// the launch's rows: every count the kernels index with 32 bits
void need_rows(int64_t rows, int64_t n_heads, int64_t n_kv_heads, int64_t n_seqs, const void* q_start, const void* length) {
  need(rows >= 0 && rows < (1ll << 30), "rows must be 0 to 2^30");
  need(n_seqs >= 0 && n_seqs <= (1 << 20), "n_seqs must be 0 to 2^20");
  need(n_heads >= 1 && n_heads <= 65535 && n_kv_heads >= 1 && n_heads % n_kv_heads == 0,
       "n_heads must be a multiple of n_kv_heads, at most 65535");
  need(q_start != nullptr && length != nullptr, "null q_start or length");
}

// makes `device` current; the caller's is put back when the call ends
class OnDevice {
 public:
  explicit OnDevice(int64_t device) {
    int now = -1;
    error = cudaGetDevice(&now);
    if (error != cudaSuccess || now == device) return;
    error = cudaSetDevice((int)device);
    if (error == cudaSuccess) back_ = now;
  }
  ~OnDevice() {
    if (back_ >= 0) cudaSetDevice(back_);
  }
  cudaError_t error;

 private:
  int back_ = -1;
};

template <class Args, class Check, class Launch>
llx_status call(const char* name, const Args* a, void* stream, Check check, Launch launch) {
  try {
    need(a != nullptr, "null argument");
    need(a->device >= 0 && a->device <= INT_MAX, "no such device");
    check(*a);
    OnDevice on(a->device);
    const cudaError_t e = on.error != cudaSuccess ? on.error : launch(*a, static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) return LLX_OK;
    cudaGetLastError();  // reported here, not by the caller's next call
    noalloc_set_error(std::string(name) + ": " + cudaGetErrorString(e));
    return e == cudaErrorMemoryAllocation ? LLX_ERR_OOM : LLX_ERR_CUDA;
  } catch (const Refused& r) {
    try {
      noalloc_set_error(std::string(name) + ": " + r.what);
    } catch (...) {
    }
    return r.code;
  } catch (...) {
    return LLX_ERR_OOM;  // the error text could not be kept
  }
}

void check_pages(const llx_pages_args& a) {
  need_cache(a.n_pages, a.page_size, a.n_kv_heads, a.head_dim, a.page_stride);
  need_table(a.table, a.table_stride, a.max_seqs, a.max_pages);
  need(a.n >= 0 && a.n <= a.max_seqs, "a list may name every slot once at most");
  need(a.refs != nullptr, "null refs");
}

void check_pools(const llx_pages_args& a) {
  need(a.k && a.v && aligned16(a.k) && aligned16(a.v), "k and v must be 16-byte aligned");
  need(a.n_layers >= 1 && a.n_layers <= 65535, "n_layers must be 1 to 65535");
  need(a.n_layers == 1 || (a.layer_stride % 16 == 0 && a.layer_stride != 0), "layer_stride must be a multiple of 16 bytes");
}

}  // namespace
}  // namespace llx

using namespace llx;

extern "C" {

llx_status llx_paged_append(const llx_paged_append_args* args, void* stream) {
  return call(
      "llx_paged_append", args, stream,
      [](const llx_paged_append_args& a) {
        need_cache(a.n_pages, a.page_size, a.n_kv_heads, a.head_dim, a.page_stride);
        need_table(a.table, a.table_stride, a.max_seqs, a.max_pages);
        need_rows(a.rows, a.n_heads, a.n_kv_heads, a.n_seqs, a.q_start, a.length);
        need(a.q && a.k && a.v && a.q8 && a.k_pages && a.v_pages && a.cos && a.sin, "null pointer");
        need(a.n_positions >= 1, "the rotation tables need a position");
        need(a.q_stride >= a.n_heads * a.head_dim && a.q8_stride >= a.n_heads * a.head_dim &&
                 a.k_stride >= a.n_kv_heads * a.head_dim && a.v_stride >= a.n_kv_heads * a.head_dim,
             "a row stride is smaller than the row");
        need_rq(a.q_M, a.q_S, "q requantization outside M [0, 2^32), S [0, 63]");
        need_rq(a.k_M, a.k_S, "k requantization outside M [0, 2^32), S [0, 63]");
        for (int i = 0; i < 2; ++i) {
          if (!(i ? a.k_gamma : a.q_gamma)) continue;
          const int64_t eps = i ? a.k_eps : a.q_eps, C = i ? a.k_C : a.q_C, sh = i ? a.k_shift : a.q_shift;
          need(eps >= 0 && eps < (1ll << 32) && C >= 0 && C < (1ll << 40) && sh >= 0 && sh <= 63,
               "norm constants outside eps [0, 2^32), C [0, 2^40), shift [0, 63]");
        }
      },
      launch_paged_append);
}

llx_status llx_paged_attention(const llx_paged_attention_args* args, void* stream) {
  return call(
      "llx_paged_attention", args, stream,
      [](const llx_paged_attention_args& a) {
        need_cache(a.n_pages, a.page_size, a.n_kv_heads, a.head_dim, a.page_stride);
        need_table(a.table, a.table_stride, a.max_seqs, a.max_pages);
        need_rows(a.rows, a.n_heads, a.n_kv_heads, a.n_seqs, a.q_start, a.length);
        need(a.q8 && a.out && a.k_pages && a.v_pages, "null pointer");
        need(aligned16(a.q8) && aligned16(a.out) && aligned16(a.k_pages) && aligned16(a.v_pages) &&
                 a.q8_stride % 16 == 0 && a.out_stride % 16 == 0,
             "q8, out and the pages must be 16-byte aligned, row for row");
        need(a.q8_stride >= a.n_heads * a.head_dim && a.out_stride >= a.n_heads * a.head_dim,
             "a row stride is smaller than the row");
        need(a.max_rows >= 0 && a.max_len >= 0, "max_rows and max_len must not be negative");
        need(a.prob_bits == 8 || a.prob_bits == 15, "attention prob_bits must be 8 or 15");
        need_rq(a.Ms, a.Ss, "score scaling outside M [0, 2^32), S [0, 63]");
        need_rq(a.Mo, a.So, "output requantization outside M [0, 2^32), S [0, 63]");
      },
      launch_paged_attention);
}

size_t llx_pages_scratch(int64_t n_pages) { return n_pages < 0 ? 0 : (size_t)(3 * n_pages + 4) * sizeof(int32_t); }

llx_status llx_pages_reserve(const llx_pages_args* args, void* stream) {
  return call(
      "llx_pages_reserve", args, stream,
      [](const llx_pages_args& a) {
        check_pages(a);
        need(a.length && a.scratch && (a.n == 0 || (a.list_a && a.list_b)), "null pointer");
      },
      launch_pages_reserve);
}

llx_status llx_pages_fork(const llx_pages_args* args, void* stream) {
  return call(
      "llx_pages_fork", args, stream,
      [](const llx_pages_args& a) {
        check_pages(a);
        check_pools(a);
        need(a.length && a.scratch && (a.n == 0 || (a.list_a && a.list_b)), "null pointer");
      },
      launch_pages_fork);
}

llx_status llx_pages_free(const llx_pages_args* args, void* stream) {
  return call(
      "llx_pages_free", args, stream,
      [](const llx_pages_args& a) {
        check_pages(a);
        need(a.length && (a.n == 0 || a.list_a), "null pointer");
      },
      launch_pages_free);
}

llx_status llx_pages_compact(const llx_pages_args* args, void* stream) {
  return call(
      "llx_pages_compact", args, stream,
      [](const llx_pages_args& a) {
        check_pages(a);
        check_pools(a);
        need(a.scratch && a.new_table && a.new_refs, "null pointer");
      },
      launch_pages_compact);
}

llx_status llx_sample(const llx_sample_args* args, void* stream) {
  return call(
      "llx_sample", args, stream,
      [](const llx_sample_args& a) {
        need(a.rows >= 0 && a.rows <= (1ll << 26), "rows must be 0 to 2^26");
        need(a.vocab >= 1, "an empty vocabulary");
        need(a.vocab <= sample_max_vocab(), "the vocabulary exceeds 262144 tokens", LLX_ERR_UNSUPPORTED);
        need(a.logits_stride >= a.vocab, "the row stride is smaller than the vocabulary");
        need(a.exponent >= -31 && a.exponent <= 15, "exponent outside [-31, 15]");
        need(a.rows == 0 || (a.logits && a.random && a.token), "null pointer");
      },
      launch_sample);
}

}  // extern "C"
