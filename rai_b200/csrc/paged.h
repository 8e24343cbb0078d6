// Paged-cache and beam-search kernels (internal launch API).
//
// A paged cache keeps the tokens of many sequences in pages of page_size
// slots: token t of sequence s is slot t % page_size of page
// table[s][t / page_size]. Sequences may share pages (refs[page] counts the
// table cells that name it; 0 = free).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "common.cuh"

// Kernels here are launched while their predecessors still run, so what these
// write (tables, lists of copies) is read by plain loads behind the wait, not by
// __ldg or through __restrict__: read-only loads want memory that does not
// change while the kernel runs, and may be moved ahead of the wait.
namespace rai {

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };  // RAI_F32, RAI_F16, RAI_BF16

// Unsigned division by a runtime constant: n / d for n < 2^31 as a multiply
// and a shift (Granlund and Montgomery's round-up method, d < 2^31).
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << shift) < div) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - div)) / div + 1);
  }
  __host__ __device__ uint32_t quot(uint32_t n) const {
#ifdef __CUDA_ARCH__
    const uint32_t hi = __umulhi(n, mul);
#else
    const uint32_t hi = (uint32_t)(((uint64_t)n * mul) >> 32);
#endif
    return (uint32_t)(((uint64_t)hi + n) >> shift);
  }
};

// One layer's pages and a ragged chunk of new rows: sequence s has rows
// q_start[s] .. q_start[s + 1] - 1, the last of its kv_len[s] tokens.
struct PagedChunk {
  void* k = nullptr;
  void* v = nullptr;
  long long k_page = 0, k_head = 0, k_slot = 0, v_page = 0, v_head = 0, v_slot = 0;  // strides in elements
  const int* table = nullptr;
  long long table_stride = 0;
  const int* kv_len = nullptr;
  const int* q_start = nullptr;
  uint32_t* err = nullptr;
  int n_seqs = 0, max_pages = 0, n_pages = 0, nkv = 0, hd = 0, rows = 0, max_rows = 0;
  FastDiv page;
};

// Row range and length of a sequence. Values outside the call's bounds are
// cut to them and reported, so that no access leaves the tensors.
struct SeqRows {
  int start, n, len;
};
__device__ __forceinline__ SeqRows seq_rows(const PagedChunk& c, int s) {
  const int a = c.q_start[s], b = c.q_start[s + 1], t = c.kv_len[s];
  const int cap = (int)min((long long)c.max_pages * c.page.d, (long long)(INT_MAX - 1024));
  SeqRows r;
  r.start = min(max(a, 0), c.rows);
  r.n = min(min(max(b, r.start), c.rows) - r.start, c.max_rows);
  r.len = min(max(t, 0), cap);
  if (r.start != a || r.start + r.n != b || r.len != t) atomicOr(c.err, kErrBadInput);
  return r;
}

// Page of token t of sequence s, or -1 (reported) if the table names none.
__device__ __forceinline__ int page_of(const PagedChunk& c, int s, int page_index) {
  const int page = c.table[(long long)s * c.table_stride + page_index];
  if ((unsigned)page < (unsigned)c.n_pages) return page;
  atomicOr(c.err, kErrBadInput);
  return -1;
}

struct AttnArgs {
  PagedChunk c;
  const void* q = nullptr;
  void* out = nullptr;
  float* lse = nullptr;  // [rows][heads], may be null
  long long q_row = 0, q_head = 0, o_row = 0, o_head = 0;
  int group = 1;     // query heads per KV head
  int window = 0;    // 0 = no window
  float scale = 1.f, softcap = 0.f;
  int dtype = kF32;
  float* part = nullptr;  // workspace
  size_t part_bytes = 0;
};
size_t paged_attention_workspace(const AttnArgs& a);
cudaError_t paged_attention(const AttnArgs& a, cudaStream_t s);

struct RopeArgs {
  PagedChunk c;
  const void *q = nullptr, *k = nullptr, *v = nullptr;  // rows of any dtype
  void* q_out = nullptr;                                // in the cache's dtype
  long long q_row = 0, q_head = 0, k_row = 0, k_head = 0, v_row = 0, v_head = 0, o_row = 0, o_head = 0;
  const float* inv_freq = nullptr;  // [rot / 2]
  int heads = 0, rot = 0, interleaved = 0, in_dtype = kF32, cache_dtype = kF32;
  float mscale = 1.f;
};
cudaError_t rope_append(const RopeArgs& a, cudaStream_t s);

// A pool of pages: `layers` planes of K and V, page p of plane l at
// base + l * layer_bytes + p * page_bytes, page_bytes long.
struct PagePool {
  char *k = nullptr, *v = nullptr;
  long long k_layer = 0, v_layer = 0, k_page = 0, v_page = 0;  // bytes
  long long bytes = 0;                                         // of one page of one plane
  int layers = 0, n_pages = 0;
};
struct TableArgs {
  int* table = nullptr;
  long long stride = 0;
  int* lens = nullptr;
  int* refs = nullptr;
  int n_seqs = 0, max_pages = 0, n_pages = 0, page_size = 1;
  uint32_t* err = nullptr;
};
constexpr int kMaxTableSeqs = 4096;
cudaError_t kv_fork(const TableArgs& in, const TableArgs& out, const int* parents, cudaStream_t s);
size_t kv_resize_workspace(int n_seqs);
cudaError_t kv_resize(const TableArgs& t, const PagePool& pool, const int* new_lens, int delta, int* status, void* ws,
                      cudaStream_t s);
size_t kv_compact_workspace(int n_pages);
cudaError_t kv_compact(const TableArgs& t, const PagePool& pool, int* used, void* ws, cudaStream_t s);
// Copies page src[i] to page dst[i] for i < n (n_dev, when set, holds n on
// the device, at most n).
cudaError_t kv_copy(const PagePool& pool, const int* src, const int* dst, const int* n_dev, int n, uint32_t* err,
                    cudaStream_t s);

struct BeamArgs {
  const void* logits = nullptr;
  long long row = 0;  // stride between (batch, beam) rows in elements
  const float* scores = nullptr;
  float *cand_score = nullptr, *score = nullptr;
  int *cand_beam = nullptr, *cand_token = nullptr, *parent = nullptr, *token = nullptr;
  const int* history = nullptr;
  int* out_history = nullptr;
  const int* hist_len = nullptr;
  int* out_len = nullptr;
  long long hist_stride = 0, out_stride = 0;
  int hist_cap = 0;
  int batch = 0, beams = 0, vocab = 0, keep = 0, eos = -1, dtype = kF32;
  uint32_t* err = nullptr;
  void* ws = nullptr;
};
constexpr int kMaxBeams = 32, kMaxKeep = 64;
size_t beam_workspace(int batch, int beams, int vocab, int keep);
cudaError_t beam_select(const BeamArgs& a, cudaStream_t s);

}  // namespace rai
