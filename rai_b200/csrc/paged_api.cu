// C ABI of the paged cache and beam search: checks of arguments, then the
// launches of kernels_paged_*.cu and kernels_beam.cu.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/rai_gpu.h"
#include "errors.h"
#include "paged.h"

namespace {

int bad(const char* msg) { return rai::set_error(RAI_ERR_INVALID, msg); }
int unsupported(const char* msg) { return rai::set_error(RAI_ERR_UNSUPPORTED, msg); }

int done(cudaError_t e) {
  if (e == cudaSuccess) return RAI_OK;
  (void)cudaGetLastError();
  return rai::set_error(e == cudaErrorMemoryAllocation ? RAI_ERR_OOM : RAI_ERR_DEVICE, cudaGetErrorString(e));
}

// No C++ exception (a failed allocation of a message or a lock) passes the
// C boundary.
template <typename F>
int guarded(F f) noexcept {
  try {
    return f();
  } catch (...) {
    return RAI_ERR_OOM;
  }
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
int size_of(uint32_t dtype) { return dtype == RAI_F32 ? 4 : 2; }

// A stride in elements whose rows start on 16-byte boundaries.
bool vec_stride(int64_t s, int elt) { return s >= 0 && s < ((int64_t)1 << 48) && s * elt % 16 == 0; }

int check_chunk(const rai_paged_chunk& c, rai::PagedChunk* out) {
  if (!c.k || !c.v || !c.table || !c.kv_len || !c.q_start) return bad("null argument");
  if (c.dtype > RAI_BF16) return unsupported("dtype");
  if (!c.n_seqs || !c.max_pages || !c.n_pages || !c.page_size || !c.n_kv_heads || !c.head_dim || !c.rows || !c.max_rows)
    return bad("a size is zero");
  const int elt = size_of(c.dtype);
  if (c.head_dim > 256 || c.head_dim * elt % 16) return unsupported("head_dim: up to 256, a multiple of 16 bytes");
  const uint32_t top = 1u << 30;
  if (c.n_seqs > top || c.max_pages > top || c.n_pages > top || c.page_size > top || c.rows > top || c.n_kv_heads > 65535)
    return bad("a size is out of range");
  if (c.max_rows > c.rows) return bad("max_rows is more than the rows of the tensors");
  if ((uint64_t)c.max_pages * c.page_size > (uint64_t)INT_MAX - 1024) return bad("max_pages * page_size passes 2^31 tokens");
  if (c.table_stride < c.max_pages) return bad("table_stride");
  if (!vec_stride(c.k_page, elt) || !vec_stride(c.k_head, elt) || !vec_stride(c.k_slot, elt) ||
      !vec_stride(c.v_page, elt) || !vec_stride(c.v_head, elt) || !vec_stride(c.v_slot, elt) || !aligned(c.k, 16) ||
      !aligned(c.v, 16))
    return bad("pages: every vector has to start on a 16-byte boundary");
  rai::PagedChunk o;
  o.k = c.k, o.v = c.v;
  o.k_page = c.k_page, o.k_head = c.k_head, o.k_slot = c.k_slot;
  o.v_page = c.v_page, o.v_head = c.v_head, o.v_slot = c.v_slot;
  o.table = c.table, o.table_stride = c.table_stride;
  o.kv_len = c.kv_len, o.q_start = c.q_start;
  o.n_seqs = (int)c.n_seqs, o.max_pages = (int)c.max_pages, o.n_pages = (int)c.n_pages;
  o.nkv = (int)c.n_kv_heads, o.hd = (int)c.head_dim, o.rows = (int)c.rows, o.max_rows = (int)c.max_rows;
  o.page = rai::FastDiv(c.page_size);
  *out = o;
  return RAI_OK;
}

int check_heads(uint32_t heads, const rai::PagedChunk& c) {
  if (!heads || heads % c.nkv) return bad("n_heads has to be a multiple of n_kv_heads");
  if ((uint64_t)heads * c.rows > (1u << 30)) return bad("rows * n_heads is out of range");
  return RAI_OK;
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}
// Whether the rows of `inner` elements of a tensor that is written lie apart:
// each stride, from the smallest, passes what lies below it.
struct Dim {
  int64_t stride, count;
};
template <int N>
bool apart(int64_t inner, Dim (&&dims)[N]) {
  std::sort(dims, dims + N, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  for (const Dim& d : dims) {
    if (d.count <= 1) continue;
    if (d.stride < inner) return false;
    inner += (d.count - 1) * d.stride;
  }
  return true;
}
size_t table_bytes(const rai_page_table& t) { return ((size_t)(t.n_seqs - 1) * t.table_stride + t.max_pages) * 4; }

int attention_args(const rai_paged_attention* a, rai::AttnArgs* out) {
  if (!a || !a->q || !a->out) return bad("null argument");
  rai::AttnArgs o;
  if (int rc = check_chunk(a->chunk, &o.c)) return rc;
  if (int rc = check_heads(a->n_heads, o.c)) return rc;
  const int elt = size_of(a->chunk.dtype);
  if (!vec_stride(a->q_row, elt) || !vec_stride(a->q_head, elt) || !vec_stride(a->out_row, elt) ||
      !vec_stride(a->out_head, elt) || !aligned(a->q, 16) || !aligned(a->out, 16))
    return bad("q, out: every vector has to start on a 16-byte boundary");
  if (!apart(a->chunk.head_dim, {{a->out_row, a->chunk.rows}, {a->out_head, a->n_heads}})) return bad("out: rows share memory");
  if ((uint64_t)a->chunk.n_seqs * (((uint64_t)a->chunk.max_rows * (a->n_heads / a->chunk.n_kv_heads) + 15) / 16) > (1u << 30))
    return bad("n_seqs * max_rows is out of range");
  // (The kernels use scale * log2(e).)
  if (!(a->scale > 0.f) || !std::isfinite(a->scale * 1.4426950408889634f)) return bad("scale has to be positive, up to 2.3e38");
  if (!(a->softcap == 0.f || std::isnormal(a->softcap)) || a->softcap < 0.f) return bad("softcap: 0, or a positive normal number");
  if (a->window > (1u << 30)) return bad("window");
  o.q = a->q, o.out = a->out, o.lse = a->lse;
  o.q_row = a->q_row, o.q_head = a->q_head, o.o_row = a->out_row, o.o_head = a->out_head;
  o.group = (int)a->n_heads / o.c.nkv;
  o.window = (int)a->window;
  o.scale = a->scale, o.softcap = a->softcap, o.dtype = (int)a->chunk.dtype;
  o.part = static_cast<float*>(a->workspace), o.part_bytes = a->workspace_bytes;
  *out = o;
  return RAI_OK;
}

int check_table(const rai_page_table* t, rai::TableArgs* out) {
  if (!t || !t->table || !t->lens || !t->refs) return bad("null argument");
  if (!t->n_seqs || !t->max_pages || !t->n_pages || !t->page_size) return bad("a size is zero");
  const uint32_t top = 1u << 30;
  if (t->n_seqs > top || t->max_pages > top || t->n_pages > top || t->page_size > top) return bad("a size is out of range");
  if ((uint64_t)t->max_pages * t->page_size > (uint64_t)INT_MAX - 1024) return bad("max_pages * page_size passes 2^31 tokens");
  if (t->table_stride < t->max_pages) return bad("table_stride");
  rai::TableArgs o;
  o.table = t->table, o.stride = t->table_stride, o.lens = t->lens, o.refs = t->refs;
  o.n_seqs = (int)t->n_seqs, o.max_pages = (int)t->max_pages, o.n_pages = (int)t->n_pages, o.page_size = (int)t->page_size;
  *out = o;
  return RAI_OK;
}

int check_pool(const rai_page_pool* p, uint32_t n_pages, rai::PagePool* out) {
  if (!p || !p->k || !p->v) return bad("null argument");
  if (!p->n_layers || p->n_layers > 65535 || !p->n_pages || p->n_pages > (1u << 30) || p->page_bytes <= 0)
    return bad("pool size");
  if (n_pages && p->n_pages != n_pages) return bad("the pool and the table have different page counts");
  if ((p->k_layer | p->k_page | p->v_layer | p->v_page | p->page_bytes) % 16 || !aligned(p->k, 16) || !aligned(p->v, 16))
    return bad("pool: pages have to start on 16-byte boundaries and be a multiple of 16 bytes");
  if (p->k_page < p->page_bytes || p->v_page < p->page_bytes || p->k_layer < 0 || p->v_layer < 0) return bad("pool strides");
  rai::PagePool o;
  o.k = static_cast<char*>(p->k), o.v = static_cast<char*>(p->v);
  o.k_layer = p->k_layer, o.v_layer = p->v_layer, o.k_page = p->k_page, o.v_page = p->v_page;
  o.bytes = p->page_bytes, o.layers = (int)p->n_layers, o.n_pages = (int)p->n_pages;
  *out = o;
  return RAI_OK;
}

}  // namespace

extern "C" {

size_t rai_gpu_paged_attention_workspace_bytes(const rai_paged_attention* a) {
  // (Sizes that the call refuses need no workspace; the rules below divide by
  // some of them.)
  if (!a || !a->chunk.n_kv_heads || !a->n_heads || !a->chunk.page_size || !a->chunk.max_rows) return 0;
  rai::AttnArgs o;
  o.c.hd = (int)a->chunk.head_dim, o.c.max_rows = (int)a->chunk.max_rows;
  o.c.max_pages = (int)a->chunk.max_pages, o.c.page.d = a->chunk.page_size;
  o.c.n_seqs = (int)a->chunk.n_seqs, o.c.nkv = (int)a->chunk.n_kv_heads;
  o.group = (int)(a->n_heads / a->chunk.n_kv_heads);
  o.dtype = (int)a->chunk.dtype;
  return rai::paged_attention_workspace(o);
}

int rai_gpu_paged_attention(const rai_paged_attention* a, void* stream) {
  return guarded([&] {
    rai::AttnArgs o;
    if (int rc = attention_args(a, &o)) return rc;
    const size_t need = rai::paged_attention_workspace(o);
    if (need && (!o.part || !aligned(o.part, 16) || o.part_bytes < need))
      return bad("workspace is too small or not on a 16-byte boundary");
    if (int rc = rai::kernel_status_word(&o.c.err)) return rc;
    return done(rai::paged_attention(o, static_cast<cudaStream_t>(stream)));
  });
}

int rai_gpu_rope_append(const rai_rope_append* a, void* stream) {
  return guarded([&] {
    if (!a || !a->q || !a->k || !a->v || !a->q_out || !a->inv_freq) return bad("null argument");
    rai::RopeArgs o;
    if (int rc = check_chunk(a->chunk, &o.c)) return rc;
    if (int rc = check_heads(a->n_heads, o.c)) return rc;
    if (a->in_dtype > RAI_BF16) return unsupported("dtype");
    const int ei = size_of(a->in_dtype), eo = size_of(a->chunk.dtype);
    if (a->chunk.head_dim * ei % 16 || (a->chunk.head_dim % 8 && ei != eo))
      return unsupported("head_dim: a multiple of 16 bytes in both types");
    if (!a->rot_dim || a->rot_dim % 2 || a->rot_dim > a->chunk.head_dim) return bad("rot_dim: even, up to head_dim");
    if (!std::isfinite(a->mscale)) return bad("mscale");
    if (!vec_stride(a->q_row, ei) || !vec_stride(a->q_head, ei) || !vec_stride(a->k_row, ei) ||
        !vec_stride(a->k_head, ei) || !vec_stride(a->v_row, ei) || !vec_stride(a->v_head, ei) ||
        !vec_stride(a->out_row, eo) || !vec_stride(a->out_head, eo) || !aligned(a->q, 16) || !aligned(a->k, 16) ||
        !aligned(a->v, 16) || !aligned(a->q_out, 16))
      return bad("q, k, v, q_out: every vector has to start on a 16-byte boundary");
    o.q = a->q, o.k = a->k, o.v = a->v, o.q_out = a->q_out, o.inv_freq = a->inv_freq;
    o.q_row = a->q_row, o.q_head = a->q_head, o.k_row = a->k_row, o.k_head = a->k_head;
    o.v_row = a->v_row, o.v_head = a->v_head, o.o_row = a->out_row, o.o_head = a->out_head;
    if (a->q_out == a->q && (ei != eo || a->q_row != a->out_row || a->q_head != a->out_head || a->in_dtype != a->chunk.dtype))
      return bad("q_out is q with other strides or another type");
    const rai_paged_chunk& c = a->chunk;
    if (!apart(c.head_dim, {{a->out_row, c.rows}, {a->out_head, a->n_heads}})) return bad("q_out: rows share memory");
    if (!apart(c.head_dim, {{c.k_page, c.n_pages}, {c.k_head, c.n_kv_heads}, {c.k_slot, c.page_size}}) ||
        !apart(c.head_dim, {{c.v_page, c.n_pages}, {c.v_head, c.n_kv_heads}, {c.v_slot, c.page_size}}) || c.k == c.v)
      return bad("pages: vectors share memory");
    o.heads = (int)a->n_heads, o.rot = (int)a->rot_dim, o.interleaved = a->interleaved != 0;
    o.in_dtype = (int)a->in_dtype, o.cache_dtype = (int)a->chunk.dtype, o.mscale = a->mscale;
    if (int rc = rai::kernel_status_word(&o.c.err)) return rc;
    return done(rai::rope_append(o, static_cast<cudaStream_t>(stream)));
  });
}

int rai_rope_frequencies(int kind, uint32_t rot, double theta, double factor, double low, double high, double original,
                         float* inv_freq, float* mscale) {
  return guarded([&] {
    if (!inv_freq || !mscale) return bad("null argument");
    if (!rot || rot % 2 || rot > 256) return bad("rot_dim: even, up to 256");
    if (!(theta > 1.0) || !std::isfinite(theta)) return bad("theta");
    if (kind < RAI_ROPE_PLAIN || kind > RAI_ROPE_YARN) return unsupported("kind of rope scaling");
    if (kind != RAI_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return bad("factor: at least 1");
    if (kind >= RAI_ROPE_LLAMA3 && !(low > 0.0 && high > low && original > 0.0 && std::isfinite(high) && std::isfinite(original)))
      return bad("low, high and original positions of the scaling");
    if (kind == RAI_ROPE_NTK && rot <= 2) return bad("rot_dim: more than 2 with this scaling");
    const double two_pi = 6.283185307179586476925286766559;
    const double base = kind == RAI_ROPE_NTK ? theta * std::pow(factor, rot / (rot - 2.0)) : theta;
    // YaRN: the pair that turns n times within the original context.
    auto pair_of = [&](double n) { return rot * std::log(original / (n * two_pi)) / (2.0 * std::log(theta)); };
    const double from = std::fmax(0.0, std::floor(pair_of(high))), to = std::fmin(rot - 1.0, std::ceil(pair_of(low)));
    for (uint32_t i = 0; i < rot / 2; ++i) {
      double f = std::pow(base, -2.0 * i / rot);
      if (kind == RAI_ROPE_LINEAR) {
        f /= factor;
      } else if (kind == RAI_ROPE_LLAMA3) {
        const double turns = original * f / two_pi;  // within the original context
        const double keep = turns >= high ? 1.0 : turns <= low ? 0.0 : (turns - low) / (high - low);
        f = keep * f + (1.0 - keep) * f / factor;
      } else if (kind == RAI_ROPE_YARN) {
        const double gone = std::fmin(1.0, std::fmax(0.0, (i - from) / std::fmax(to - from, 1e-3)));
        f = (1.0 - gone) * f + gone * f / factor;
      }
      inv_freq[i] = (float)f;
    }
    *mscale = kind == RAI_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.f;
    return (int)RAI_OK;
  });
}

int rai_gpu_kv_fork(const rai_page_table* in, const rai_page_table* out, const int32_t* parents, void* stream) {
  return guarded([&] {
    rai::TableArgs a, b;
    if (int rc = check_table(in, &a)) return rc;
    if (int rc = check_table(out, &b)) return rc;
    if (!parents) return bad("null argument");
    if (a.refs != b.refs || a.n_pages != b.n_pages || a.page_size != b.page_size)
      return bad("fork: both tables have to be of one pool");
    if (b.max_pages < a.max_pages) return bad("fork: the new table is narrower than the old one");
    if (overlap(in->table, table_bytes(*in), out->table, table_bytes(*out)) ||
        overlap(in->lens, in->n_seqs * 4ull, out->lens, out->n_seqs * 4ull))
      return bad("fork: the new table and lengths need their own memory");
    if (overlap(parents, out->n_seqs * 4ull, out->table, table_bytes(*out)) ||
        overlap(parents, out->n_seqs * 4ull, out->lens, out->n_seqs * 4ull))
      return bad("fork: the new table and lengths need their own memory");
    if (int rc = rai::kernel_status_word(&a.err)) return rc;
    b.err = a.err;
    return done(rai::kv_fork(a, b, parents, static_cast<cudaStream_t>(stream)));
  });
}

size_t rai_gpu_kv_resize_workspace_bytes(uint32_t n_seqs) {
  return n_seqs > (uint32_t)rai::kMaxTableSeqs ? 0 : rai::kv_resize_workspace((int)n_seqs);
}

int rai_gpu_kv_resize(const rai_page_table* table, const rai_page_pool* pool, const int32_t* new_lens, int32_t delta,
                      int32_t* status, void* ws, size_t ws_bytes, void* stream) {
  return guarded([&] {
    rai::TableArgs t;
    rai::PagePool p;
    if (int rc = check_table(table, &t)) return rc;
    if (int rc = check_pool(pool, table->n_pages, &p)) return rc;
    if (!status) return bad("null argument");
    if (t.n_seqs > rai::kMaxTableSeqs) return unsupported("resize: at most 4096 sequences");
    if (!ws || !aligned(ws, 4) || ws_bytes < rai::kv_resize_workspace(t.n_seqs)) return bad("workspace is too small");
    if (new_lens && new_lens != t.lens && overlap(new_lens, t.n_seqs * 4ull, t.lens, t.n_seqs * 4ull))
      return bad("resize: the new lengths overlap the old ones");
    if (int rc = rai::kernel_status_word(&t.err)) return rc;
    return done(rai::kv_resize(t, p, new_lens, delta, status, ws, static_cast<cudaStream_t>(stream)));
  });
}

size_t rai_gpu_kv_compact_workspace_bytes(uint32_t n_pages) {
  return n_pages > (1u << 30) ? 0 : rai::kv_compact_workspace((int)n_pages);
}

int rai_gpu_kv_compact(const rai_page_table* table, const rai_page_pool* pool, int32_t* used, void* ws, size_t ws_bytes,
                       void* stream) {
  return guarded([&] {
    rai::TableArgs t;
    rai::PagePool p;
    if (int rc = check_table(table, &t)) return rc;
    if (int rc = check_pool(pool, table->n_pages, &p)) return rc;
    if (!used) return bad("null argument");
    if (!ws || !aligned(ws, 4) || ws_bytes < rai::kv_compact_workspace(t.n_pages)) return bad("workspace is too small");
    if (int rc = rai::kernel_status_word(&t.err)) return rc;
    return done(rai::kv_compact(t, p, used, ws, static_cast<cudaStream_t>(stream)));
  });
}

int rai_gpu_kv_copy_pages(const rai_page_pool* pool, const int32_t* src, const int32_t* dst, size_t n, void* stream) {
  return guarded([&] {
    rai::PagePool p;
    if (int rc = check_pool(pool, 0, &p)) return rc;
    if (n > (1u << 30)) return bad("a size is out of range");
    if (n && (!src || !dst)) return bad("null argument");
    if (!n) return (int)RAI_OK;
    uint32_t* err = nullptr;
    if (int rc = rai::kernel_status_word(&err)) return rc;
    return done(rai::kv_copy(p, src, dst, nullptr, (int)n, err, static_cast<cudaStream_t>(stream)));
  });
}

size_t rai_gpu_beam_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t keep) {
  if (!batch || !beams || !vocab || batch > 65535 || beams > (uint32_t)rai::kMaxBeams || keep > (uint32_t)rai::kMaxKeep ||
      vocab > (1u << 30))
    return 0;
  return rai::beam_workspace((int)batch, (int)beams, (int)vocab, (int)keep);
}

int rai_gpu_beam_select(const rai_beam_select* a, void* stream) {
  return guarded([&] {
    if (!a || !a->logits || !a->scores || !a->cand_score || !a->cand_beam || !a->cand_token || !a->score || !a->parent ||
        !a->token)
      return bad("null argument");
    if (a->dtype > RAI_BF16) return unsupported("dtype");
    if (!a->batch || !a->beams || !a->vocab) return bad("a size is zero");
    if (a->beams > (uint32_t)rai::kMaxBeams || a->keep > (uint32_t)rai::kMaxKeep) return unsupported("beams up to 32, keep up to 64");
    if (a->keep < a->beams) return bad("keep: at least beams");
    if ((uint64_t)a->batch * a->beams > 65535 || (uint64_t)a->beams * a->vocab > (uint64_t)INT_MAX - (1 << 20))
      return bad("batch * beams up to 65535, beams * vocab below 2^31");
    if (a->row_stride < a->vocab || !aligned(a->logits, size_of(a->dtype))) return bad("row_stride");
    if (a->eos < -1) return bad("eos");
    rai::BeamArgs o;
    if (a->history) {
      if (!a->hist_len || !a->out_history || !a->out_len) return bad("null argument");
      if (!a->hist_cap || a->hist_stride < a->hist_cap || a->out_hist_stride < a->hist_cap) return bad("history strides");
      const uint64_t rows = (uint64_t)a->batch * a->beams;
      if (overlap(a->history, ((rows - 1) * a->hist_stride + a->hist_cap) * 4, a->out_history,
                  ((rows - 1) * a->out_hist_stride + a->hist_cap) * 4) ||
          overlap(a->hist_len, rows * 4, a->out_len, rows * 4))
        return bad("the new histories need their own memory");
      o.history = a->history, o.hist_len = a->hist_len, o.out_history = a->out_history, o.out_len = a->out_len;
      o.hist_stride = a->hist_stride, o.out_stride = a->out_hist_stride, o.hist_cap = (int)a->hist_cap;
      if (a->hist_cap > (1u << 30)) return bad("history strides");
    }
    o.logits = a->logits, o.row = a->row_stride, o.scores = a->scores;
    o.cand_score = a->cand_score, o.cand_beam = a->cand_beam, o.cand_token = a->cand_token;
    o.score = a->score, o.parent = a->parent, o.token = a->token;
    o.batch = (int)a->batch, o.beams = (int)a->beams, o.vocab = (int)a->vocab, o.keep = (int)a->keep;
    o.eos = a->eos, o.dtype = (int)a->dtype;
    if (!a->workspace || !aligned(a->workspace, 8) || a->workspace_bytes < rai::beam_workspace(o.batch, o.beams, o.vocab, o.keep))
      return bad("workspace is too small or not on an 8-byte boundary");
    o.ws = a->workspace;
    if (int rc = rai::kernel_status_word(&o.err)) return rc;
    return done(rai::beam_select(o, static_cast<cudaStream_t>(stream)));
  });
}

}  // extern "C"
