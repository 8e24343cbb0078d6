// The torch side of rai_b200.paged and rai_b200.beams: checks tensors, takes
// their addresses and strides, makes outputs and workspaces on the current
// stream and calls the C ABI (include/rai_gpu.h). In C++ because a decoding
// step makes several of these calls a layer, and the same in Python took two
// to three times as long as the kernels.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/rai_gpu.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

[[noreturn]] void bad(const std::string& what) { throw py::value_error(what); }
void need(bool ok, const char* what) {
  if (!ok) bad(what);
}

// Raises rai_b200.RaiError for a status other than RAI_OK.
void check(int rc) {
  if (rc != RAI_OK) py::module_::import("rai_b200.native").attr("check")(rc);
}

uint32_t dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return RAI_F32;
    case at::kHalf: return RAI_F16;
    case at::kBFloat16: return RAI_BF16;
    default: bad(std::string(name) + ": float32, float16 or bfloat16");
  }
}

// The CUDA device that all tensors are on.
template <typename... T>
c10::DeviceIndex device_of(const Tensor& first, const T&... rest) {
  need(first.is_cuda() && ((rest.is_cuda() && rest.get_device() == first.get_device()) && ...),
       "every tensor has to be on one CUDA device");
  return (c10::DeviceIndex)first.get_device();
}
void on_device(const OptTensor& t, c10::DeviceIndex dev) {
  if (t) need(t->is_cuda() && t->get_device() == dev, "every tensor has to be on one CUDA device");
}

// The device made current for a call, and its current torch stream.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(c10::DeviceIndex dev) : guard(dev), stream(c10::cuda::getCurrentCUDAStream(dev).stream()) {}
};

int32_t* ints(const Tensor& t, int64_t n, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
    bad(std::string(name) + ": a contiguous int32 vector of " + std::to_string(n) + " that fits the other arguments");
  return t.data_ptr<int32_t>();
}

struct Cells {
  int32_t* at;
  int64_t row, width;
};
Cells cells(const Tensor& t, int64_t rows, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != rows || (t.size(1) > 1 && t.stride(1) != 1))
    bad(std::string(name) + ": an int32 table of " + std::to_string(rows) + " rows, its last dimension contiguous");
  // A one-row table may have any row stride.
  return {t.data_ptr<int32_t>(), rows > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)), t.size(1)};
}

void no_gradient(const Tensor& t, const char* name) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    bad(std::string(name) + ": this operator has no gradient; call it under torch.no_grad()");
}
// A call writes t in place: a graph that has saved it has to notice.
// (Inference tensors count no versions.)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Pages are read, and by most calls written: neither with a gradient.
void no_gradient(const Tensor& k, const Tensor& v) {
  no_gradient(k, "k_pages");
  no_gradient(v, "v_pages");
}
void rows3(const Tensor& t, int64_t heads, int64_t dim, const char* name) {
  if (t.dim() != 3 || t.size(2) != dim || (heads >= 0 && t.size(1) != heads))
    bad(std::string(name) + ": [rows, heads, head_dim] that fits the pages");
  if (dim > 1 && t.stride(2) != 1) bad(std::string(name) + ": head_dim has to be contiguous");
  no_gradient(t, name);
}

uint32_t u32(int64_t v, const char* name) {
  if (v < 0 || v > (int64_t)UINT32_MAX) bad(std::string(name) + " is out of range");
  return (uint32_t)v;
}

rai_paged_chunk chunk_of(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& kv_len, const Tensor& q_start,
                         int64_t rows, int64_t max_rows) {
  need(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
       "k_pages, v_pages: two tensors [pages, kv_heads, page_size, head_dim] of one shape and type");
  need(k.size(3) <= 1 || (k.stride(3) == 1 && v.stride(3) == 1), "k_pages, v_pages: head_dim has to be contiguous");
  need(kv_len.dim() == 1, "kv_len: a vector");
  const int64_t n = kv_len.size(0);
  const Cells t = cells(table, n, "page_table");
  rai_paged_chunk c = {};
  c.k = k.data_ptr(), c.v = v.data_ptr();
  c.k_page = k.stride(0), c.k_head = k.stride(1), c.k_slot = k.stride(2);
  c.v_page = v.stride(0), c.v_head = v.stride(1), c.v_slot = v.stride(2);
  c.table = t.at, c.table_stride = t.row, c.max_pages = u32(t.width, "page_table");
  c.kv_len = ints(kv_len, n, "kv_len"), c.q_start = ints(q_start, n + 1, "q_start");
  c.n_seqs = u32(n, "sequences"), c.n_pages = u32(k.size(0), "pages"), c.n_kv_heads = u32(k.size(1), "kv_heads");
  c.page_size = u32(k.size(2), "page_size"), c.head_dim = u32(k.size(3), "head_dim");
  c.rows = u32(rows, "rows"), c.max_rows = u32(max_rows, "max_rows");
  c.dtype = dtype_of(k, "k_pages");
  return c;
}

Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& kv_len, const Tensor& q_start,
                 int64_t max_rows, std::optional<double> scale, double softcap, int64_t window, const OptTensor& out_in,
                 const OptTensor& lse, const OptTensor& ws_in) {
  need(k.dim() == 4, "k_pages, v_pages: two tensors [pages, kv_heads, page_size, head_dim] of one shape and type");
  const int64_t hd = k.size(3);
  dtype_of(k, "k_pages");
  no_gradient(k, v);
  rows3(q, -1, hd, "q");
  need(q.scalar_type() == k.scalar_type(), "q: the type of the pages");
  const int64_t rows = q.size(0), heads = q.size(1);
  const c10::DeviceIndex dev = device_of(q, k, v, table, kv_len, q_start);
  on_device(out_in, dev);
  on_device(lse, dev);
  on_device(ws_in, dev);
  if (lse) no_gradient(*lse, "lse");
  if (out_in) {
    rows3(*out_in, heads, hd, "out");
    need(out_in->size(0) == rows && out_in->scalar_type() == q.scalar_type(), "out: shape and type of q");
  }
  if (lse)
    need(lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == rows && lse->size(1) == heads && lse->is_contiguous(),
         "lse: contiguous float32 [rows, heads]");
  need(max_rows >= 0, "max_rows");
  On on(dev);
  Tensor out = out_in ? *out_in : at::empty({rows, heads, hd}, q.options());
  if (rows == 0 || kv_len.numel() == 0 || max_rows == 0) return out;
  rai_paged_attention a = {};
  a.chunk = chunk_of(k, v, table, kv_len, q_start, rows, std::min(max_rows, rows));
  a.q = q.data_ptr(), a.out = out.data_ptr(), a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.q_row = q.stride(0), a.q_head = q.stride(1), a.out_row = out.stride(0), a.out_head = out.stride(1);
  a.n_heads = u32(heads, "heads"), a.window = u32(window, "window");
  a.scale = scale ? (float)*scale : 1.f / std::sqrt((float)hd);
  a.softcap = (float)softcap;
  Tensor ws;
  if (ws_in) {
    need(ws_in->is_contiguous(), "workspace: contiguous");
    ws = *ws_in;
  } else if (const size_t n = rai_gpu_paged_attention_workspace_bytes(&a)) {
    ws = bytes(n, q);
  }
  if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.nbytes();
  check(rai_gpu_paged_attention(&a, on.stream));
  if (out_in) written(*out_in);
  if (lse) written(*lse);
  return out;
}

int64_t attention_workspace_bytes(const Tensor& q, const Tensor& k, const Tensor& table, int64_t max_rows) {
  need(q.dim() == 3 && k.dim() == 4 && table.dim() == 2 && q.is_cuda(), "q, k_pages, page_table as for attention");
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)q.get_device());
  rai_paged_attention a = {};
  a.chunk.dtype = dtype_of(k, "k_pages");
  a.chunk.head_dim = u32(k.size(3), "head_dim"), a.chunk.n_kv_heads = u32(k.size(1), "kv_heads");
  a.chunk.max_rows = u32(std::min(max_rows, q.size(0)), "max_rows"), a.chunk.max_pages = u32(table.size(1), "page_table");
  a.chunk.page_size = u32(k.size(2), "page_size"), a.chunk.n_seqs = u32(table.size(0), "sequences");
  a.n_heads = u32(q.size(1), "heads");
  return (int64_t)rai_gpu_paged_attention_workspace_bytes(&a);
}

Tensor rope_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                   const Tensor& table, const Tensor& kv_len, const Tensor& q_start, const Tensor& inv_freq, bool interleaved,
                   double mscale, const OptTensor& out_in) {
  need(k_pages.dim() == 4, "k_pages, v_pages: two tensors [pages, kv_heads, page_size, head_dim] of one shape and type");
  const int64_t hd = k_pages.size(3), nkv = k_pages.size(1);
  dtype_of(k_pages, "k_pages");
  no_gradient(k_pages, v_pages);
  no_gradient(inv_freq, "inv_freq");
  rows3(q, -1, hd, "q");
  rows3(k, nkv, hd, "k");
  rows3(v, nkv, hd, "v");
  const int64_t rows = q.size(0), heads = q.size(1);
  need(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.size(0) == rows && v.size(0) == rows,
       "q, k, v: one type and one number of rows");
  need(inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1 && inv_freq.is_contiguous(), "inv_freq: a contiguous float32 vector");
  const c10::DeviceIndex dev = device_of(q, k, v, k_pages, v_pages, table, kv_len, q_start, inv_freq);
  on_device(out_in, dev);
  if (out_in) {
    rows3(*out_in, heads, hd, "q_out");
    need(out_in->size(0) == rows && out_in->scalar_type() == k_pages.scalar_type(), "q_out: q's shape in the pages' type");
  }
  On on(dev);
  Tensor out = out_in ? *out_in : at::empty({rows, heads, hd}, k_pages.options());
  if (rows == 0 || kv_len.numel() == 0) return out;
  rai_rope_append a = {};
  a.chunk = chunk_of(k_pages, v_pages, table, kv_len, q_start, rows, rows);
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr(), a.q_out = out.data_ptr();
  a.inv_freq = inv_freq.data_ptr<float>();
  a.q_row = q.stride(0), a.q_head = q.stride(1), a.k_row = k.stride(0), a.k_head = k.stride(1);
  a.v_row = v.stride(0), a.v_head = v.stride(1), a.out_row = out.stride(0), a.out_head = out.stride(1);
  a.n_heads = u32(heads, "heads"), a.rot_dim = u32(2 * inv_freq.size(0), "inv_freq");
  a.interleaved = interleaved, a.in_dtype = dtype_of(q, "q"), a.mscale = (float)mscale;
  check(rai_gpu_rope_append(&a, on.stream));
  written(k_pages), written(v_pages);
  if (out_in) written(*out_in);
  return out;
}

rai_page_table table_of(const Tensor& table, const Tensor& lens, const Tensor& refs, int64_t page_size) {
  need(lens.dim() == 1 && refs.dim() == 1, "lens, refs: vectors");
  const int64_t n = lens.size(0);
  const Cells t = cells(table, n, "page_table");
  rai_page_table r = {};
  r.table = t.at, r.table_stride = t.row, r.max_pages = u32(t.width, "page_table");
  r.lens = ints(lens, n, "lens"), r.refs = ints(refs, refs.size(0), "refs");
  r.n_seqs = u32(n, "sequences"), r.n_pages = u32(refs.size(0), "refs"), r.page_size = u32(page_size, "page_size");
  return r;
}

// K and V pages of every layer, [layers, pages, kv_heads, page_size,
// head_dim] or one layer's four dimensions, a page being one dense block;
// also the page size.
std::pair<rai_page_pool, int64_t> pool_of(const Tensor& k, const Tensor& v) {
  dtype_of(k, "k");
  const int64_t d = k.dim();
  need((d == 4 || d == 5) && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(),
       "k, v: two tensors [layers, pages, kv_heads, page_size, head_dim] of one shape and type");
  const int64_t e = (int64_t)k.element_size(), layers = d == 5 ? k.size(0) : 1, pages = k.size(d - 4);
  const int64_t n = k.size(d - 3) * k.size(d - 2) * k.size(d - 1);
  for (const Tensor* t : {&k, &v}) {
    // A page's block may order its heads and slots either way.
    std::pair<int64_t, int64_t> dims[3];
    for (int i = 0; i < 3; ++i) dims[i] = {t->stride(d - 3 + i), t->size(d - 3 + i)};
    std::sort(dims, dims + 3);
    int64_t want = 1;
    for (const auto& [stride, size] : dims) {
      if (size <= 1) continue;
      need(stride == want, "k, v: every page has to be one contiguous block");
      want *= size;
    }
  }
  rai_page_pool p = {};
  p.k = k.data_ptr(), p.v = v.data_ptr();
  // The stride of a single page or layer means nothing.
  p.k_layer = layers > 1 ? k.stride(0) * e : 0, p.v_layer = layers > 1 ? v.stride(0) * e : 0;
  p.k_page = pages > 1 ? k.stride(d - 4) * e : n * e, p.v_page = pages > 1 ? v.stride(d - 4) * e : n * e;
  p.page_bytes = n * e, p.n_layers = u32(layers, "layers"), p.n_pages = u32(pages, "pages");
  return {p, k.size(d - 2)};
}

std::tuple<Tensor, Tensor> kv_fork(const Tensor& table, const Tensor& lens, const Tensor& refs, const Tensor& parents, int64_t page_size,
                                const OptTensor& table_in, const OptTensor& lens_in) {
  need(parents.dim() == 1 && parents.size(0) > 0 && lens.numel() > 0 && table.dim() == 2, "fork: no sequences");
  // The number of children is the outputs': one for each parent named.
  need(!lens_in || (lens_in->dim() == 1 && lens_in->size(0) == parents.size(0)), "out_lens: as many as parents");
  need(!table_in || (table_in->dim() == 2 && table_in->size(0) == parents.size(0)), "out_table: as many rows as parents");
  const c10::DeviceIndex dev = device_of(table, lens, refs, parents);
  on_device(table_in, dev);
  on_device(lens_in, dev);
  On on(dev);
  const int64_t n = parents.size(0);
  Tensor out = table_in ? *table_in : at::empty({n, table.size(1)}, table.options());
  Tensor out_lens = lens_in ? *lens_in : at::empty({n}, lens.options());
  const rai_page_table a = table_of(table, lens, refs, page_size), b = table_of(out, out_lens, refs, page_size);
  check(rai_gpu_kv_fork(&a, &b, ints(parents, n, "parents"), on.stream));
  written(refs);
  if (table_in) written(*table_in);
  if (lens_in) written(*lens_in);
  return {out, out_lens};
}

Tensor kv_resize(const Tensor& table, const Tensor& lens, const Tensor& refs, const Tensor& k, const Tensor& v, int64_t delta,
              const OptTensor& new_lens, const OptTensor& ws_in) {
  no_gradient(k, v);
  const c10::DeviceIndex dev = device_of(table, lens, refs, k, v);
  on_device(new_lens, dev);
  on_device(ws_in, dev);
  const auto [pool, page] = pool_of(k, v);
  const rai_page_table t = table_of(table, lens, refs, page);
  need(delta >= INT32_MIN && delta <= INT32_MAX, "delta is out of range");
  On on(dev);
  Tensor status = at::empty({1}, lens.options());
  if (ws_in) need(ws_in->is_contiguous(), "workspace: contiguous");
  Tensor ws = ws_in ? *ws_in : bytes(rai_gpu_kv_resize_workspace_bytes(t.n_seqs), lens);
  check(rai_gpu_kv_resize(&t, &pool, new_lens ? ints(*new_lens, t.n_seqs, "new_lens") : nullptr, (int32_t)delta,
                          status.data_ptr<int32_t>(), ws.data_ptr(), ws.nbytes(), on.stream));
  for (const Tensor* x : {&table, &lens, &refs, &k, &v}) written(*x);
  return status;
}

Tensor kv_compact(const Tensor& table, const Tensor& lens, const Tensor& refs, const Tensor& k, const Tensor& v, const OptTensor& ws_in) {
  no_gradient(k, v);
  const c10::DeviceIndex dev = device_of(table, lens, refs, k, v);
  on_device(ws_in, dev);
  const auto [pool, page] = pool_of(k, v);
  const rai_page_table t = table_of(table, lens, refs, page);
  On on(dev);
  Tensor used = at::empty({1}, refs.options());
  if (ws_in) need(ws_in->is_contiguous(), "workspace: contiguous");
  Tensor ws = ws_in ? *ws_in : bytes(rai_gpu_kv_compact_workspace_bytes(t.n_pages), refs);
  check(rai_gpu_kv_compact(&t, &pool, used.data_ptr<int32_t>(), ws.data_ptr(), ws.nbytes(), on.stream));
  for (const Tensor* x : {&table, &refs, &k, &v}) written(*x);
  return used;
}

void copy_pages(const Tensor& k, const Tensor& v, const Tensor& src, const Tensor& dst) {
  no_gradient(k, v);
  const c10::DeviceIndex dev = device_of(k, v, src, dst);
  const auto [pool, page] = pool_of(k, v);
  need(src.dim() == 1, "src: a vector");
  On on(dev);
  check(rai_gpu_kv_copy_pages(&pool, ints(src, src.size(0), "src"), ints(dst, src.size(0), "dst"), (size_t)src.size(0), on.stream));
  written(k), written(v);
}

py::tuple beam_select(const Tensor& logits, const Tensor& scores, std::optional<int64_t> keep_in, int64_t eos, const OptTensor& history,
                 const OptTensor& hist_len, const OptTensor& ws_in) {
  const uint32_t dtype = dtype_of(logits, "logits");
  need(logits.dim() == 3, "logits: [batch, beams, vocab]");
  const int64_t b = logits.size(0), n = logits.size(1), v = logits.size(2), keep = keep_in ? *keep_in : 2 * n;
  need(b > 0 && n > 0 && v > 0, "logits: a size is zero");
  need(keep >= n && keep <= 64, "keep: from beams to 64");  // before outputs of that size are made
  need(v == 1 || logits.stride(2) == 1, "logits: vocab has to be contiguous");
  const int64_t row = n > 1 ? logits.stride(1) : b > 1 ? logits.stride(0) : v;
  need(n == 1 || b == 1 || logits.stride(0) == n * row, "logits: rows have to be evenly spaced");
  need(scores.scalar_type() == at::kFloat && scores.dim() == 2 && scores.size(0) == b && scores.size(1) == n && scores.is_contiguous(),
       "scores: contiguous float32 [batch, beams]");
  no_gradient(logits, "logits");
  no_gradient(scores, "scores");
  const c10::DeviceIndex dev = device_of(logits, scores);
  on_device(history, dev);
  on_device(hist_len, dev);
  on_device(ws_in, dev);
  need(!history || hist_len, "hist_len: needed with history");
  On on(dev);
  const auto f32 = scores.options(), i32 = scores.options().dtype(at::kInt);
  Tensor cs = at::empty({b, keep}, f32), sc = at::empty({b, n}, f32);
  Tensor cb = at::empty({b, keep}, i32), ct = at::empty({b, keep}, i32), pa = at::empty({b, n}, i32), tk = at::empty({b, n}, i32);
  rai_beam_select a = {};
  a.logits = logits.data_ptr(), a.scores = scores.data_ptr<float>(), a.row_stride = row;
  a.cand_score = cs.data_ptr<float>(), a.cand_beam = cb.data_ptr<int32_t>(), a.cand_token = ct.data_ptr<int32_t>();
  a.score = sc.data_ptr<float>(), a.parent = pa.data_ptr<int32_t>(), a.token = tk.data_ptr<int32_t>();
  Tensor out_h, out_n;
  if (history) {
    const Cells h = cells(*history, b * n, "history");
    out_h = at::empty({b * n, h.width}, i32), out_n = at::empty({b * n}, i32);
    a.history = h.at, a.hist_stride = h.row, a.hist_cap = u32(h.width, "history");
    a.hist_len = ints(*hist_len, b * n, "hist_len");
    a.out_history = out_h.data_ptr<int32_t>(), a.out_len = out_n.data_ptr<int32_t>(), a.out_hist_stride = h.width;
  }
  a.batch = u32(b, "batch"), a.beams = u32(n, "beams"), a.vocab = u32(v, "vocab"), a.keep = u32(keep, "keep");
  need(eos >= INT32_MIN && eos <= INT32_MAX, "eos is out of range");
  a.eos = (int32_t)eos, a.dtype = dtype;
  if (ws_in) need(ws_in->is_contiguous(), "workspace: contiguous");
  Tensor ws = ws_in ? *ws_in : bytes(rai_gpu_beam_workspace_bytes(a.batch, a.beams, a.vocab, a.keep), scores);
  a.workspace = ws.data_ptr(), a.workspace_bytes = ws.nbytes();
  check(rai_gpu_beam_select(&a, on.stream));
  return py::make_tuple(cs, cb, ct, sc, pa, tk, history ? py::cast(out_h) : py::none(), history ? py::cast(out_n) : py::none());
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("attention", &attention);
  m.def("attention_workspace_bytes", &attention_workspace_bytes);
  m.def("rope_append", &rope_append);
  m.def("fork", &kv_fork);
  m.def("resize", &kv_resize);
  m.def("compact", &kv_compact);
  m.def("copy_pages", &copy_pages);
  m.def("select", &beam_select);
}
