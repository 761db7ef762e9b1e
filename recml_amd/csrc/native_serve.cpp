// Native host side of the serving operators (include/hstu_serve.h): a call of recml_amd.kv_write, kv_read, cached_attention or
// token_log_probs goes through ONE function here to the kernels, and, with gradients, one graph node.
//
// A step of serving is a handful of small kernels, so its host work is what it costs: filling the structs field by field from Python
// took 25 us of a call whose kernels take 10.  What a function here does not take as it is (a conversion, a copy, an error to
// report) comes back as None, and the Python side (recml_amd/hstu_cache_ops.py, hstu_scores.py), which knows every form and every
// message, runs.

#include "native_common.h"

#include <algorithm>
#include <limits>
#include <memory>
#include <mutex>
#include <unordered_set>
#include <utility>
#include <vector>

#include "hstu_serve.h"

namespace {

// What the Python side raises for these: arguments that are refused are a ValueError.
void serve_check(int rc, const char* what) {
  TORCH_CHECK_VALUE(rc != HSTU_SERVE_ERR_NULL && rc != HSTU_SERVE_ERR_SHAPE, what, " rejected the arguments (", rc, "): ", hstu_serve_last_error());
  TORCH_CHECK(rc == HSTU_SERVE_OK, what, " failed (", rc, "): ", hstu_serve_last_error());
}

constexpr int64_t MOST = std::numeric_limits<int32_t>::max();

bool head_dim(int64_t d) {
  for (const int64_t known : {8, 16, 24, 32, 48, 64, 96, 128, 192, 256})
    if (d == known) return true;
  return false;
}

// The tensors of a KVPages and what the kernels need to know of them; false: they are not what KVPages checks for.
struct Pages {
  Tensor t[4];                  // k, k_scales, v, v_scales
  int64_t d = 0, bits = 0;
};

bool fill_pages(const Pages& p, HstuKvPages* g) {
  const Tensor& k = p.t[0];
  if (!k.defined() || !k.is_cuda() || !head_dim(p.d)) return false;
  const auto dev = k.device();
  for (const Tensor& t : p.t)
    if (!t.defined() || !plain(t, dev, at::kByte) || t.dim() != 4 || !aligned(t)) return false;
  const int64_t n = k.size(0), H = k.size(1), size = k.size(2), width = k.size(3), blocks = (p.d + 31) / 32;
  if (8 * width != p.bits * p.d || (p.bits != 4 && p.bits != 8) || size < 32 || size % 32 || size > 1 << 20 || H < 1 || n > MOST || H > MOST) return false;
  if (p.t[2].sizes() != k.sizes()) return false;
  for (int i : {1, 3})
    if (p.t[i].size(0) != n || p.t[i].size(1) != H || p.t[i].size(2) != blocks || p.t[i].size(3) != size) return false;
  g->k_codes = p.t[0].data_ptr(); g->k_scales = p.t[1].data_ptr(); g->v_codes = p.t[2].data_ptr(); g->v_scales = p.t[3].data_ptr();
  g->n_pages = (int32_t)n; g->H = (int32_t)H; g->page_size = (int32_t)size; g->d = (int32_t)p.d; g->bits = (int32_t)p.bits;
  return true;
}

bool pages_arg(PyObject* o, Pages* p) {
  static PyObject* const names[5] = {PyUnicode_InternFromString("k"), PyUnicode_InternFromString("k_scales"), PyUnicode_InternFromString("v"),
                                     PyUnicode_InternFromString("v_scales"), PyUnicode_InternFromString("head_dim")};
  for (int i = 0; i < 5; ++i) {
    PyObject* const a = PyObject_GetAttr(o, names[i]);
    if (!a) { PyErr_Clear(); return false; }
    const bool ok = i < 4 ? THPVariable_Check(a) : long_arg(a, &p->d);
    if (ok && i < 4) p->t[i] = THPVariable_Unpack(a);
    Py_DECREF(a);
    if (!ok) return false;
  }
  if (p->t[0].dim() != 4 || p->d < 1) return false;
  p->bits = 8 * p->t[0].size(3) / p->d;
  return true;
}

// The page table and the batch's size.
bool table_arg(PyObject* o, c10::Device dev, Tensor* keep, HstuKvPages* g) {
  if (!tensor_arg(o, keep) || !keep->defined() || !plain(*keep, dev, at::kInt) || keep->dim() != 2 || keep->size(0) > MOST || keep->size(1) > MOST) return false;
  g->page_table = keep->const_data_ptr<int32_t>();
  g->B = (int32_t)keep->size(0);
  g->table_pages = (int32_t)keep->size(1);
  return true;
}

bool ints_arg(PyObject* o, c10::Device dev, int64_t n, Tensor* keep) {
  return tensor_arg(o, keep) && keep->defined() && plain(*keep, dev, at::kInt) && keep->dim() == 1 && keep->size(0) == n;
}

// Whether every entry has memory of its own, as far as strides of zero tell.
bool apart(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return false;
  return true;
}

struct RowStrides { int64_t b, t, h; };

// New events' rows, [B, n, H, d] or packed [T, H, d]: whether the kernels take them as they are.
bool rows_ready(const Tensor& x, c10::Device dev, const HstuKvPages& g, bool packed, RowStrides* s) {
  if (!on(x, dev) || x.dim() != (packed ? 3 : 4) || !aligned(x)) return false;
  const int64_t unit = x.scalar_type() == at::kFloat ? 4 : 8, at = packed ? 0 : 1;
  if (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16) return false;
  if (x.size(at + 1) != g.H || x.size(at + 2) != g.d || (!packed && x.size(0) != g.B) || x.size(at) > MOST) return false;
  if (x.stride(at + 2) != 1) return false;
  auto stride = [&](int64_t i) { return x.size(i) == 1 ? (int64_t)0 : x.stride(i); };
  *s = RowStrides{packed ? 0 : stride(0), stride(at), stride(at + 1)};
  return s->b % unit == 0 && s->t % unit == 0 && s->h % unit == 0;
}

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? HSTU_SERVE_FP32 : HSTU_SERVE_BF16; }

template <typename A>
void head(A* a) {
  memset(a, 0, sizeof(*a));
  a->struct_size = sizeof(*a);
  a->version = HSTU_SERVE_ABI_VERSION;
}

// check_pages(k, k_scales, v, v_scales, head_dim, bits): whether they are pages.
PyObject* check_pages(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 6) {
    PyErr_SetString(PyExc_TypeError, "check_pages takes 6 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Pages p;
    HstuKvPages g;
    for (int i = 0; i < 4; ++i)
      if (!THPVariable_Check(a[i])) Py_RETURN_FALSE;
      else p.t[i] = THPVariable_Unpack(a[i]);
    if (!long_arg(a[4], &p.d) || !long_arg(a[5], &p.bits)) Py_RETURN_FALSE;
    return PyBool_FromLong(fill_pages(p, &g));
  });
}

void fill_rows(HstuKvRowsArgs* a, const Tensor& starts, const Tensor& offsets, int64_t per_seq, int64_t total, const Tensor& k, const Tensor& v,
               const RowStrides& ks, const RowStrides& vs) {
  a->starts = starts.const_data_ptr<int32_t>();
  a->offsets = offsets.defined() ? offsets.const_data_ptr<int32_t>() : nullptr;
  a->total_rows = total; a->rows_per_seq = (int32_t)per_seq; a->dtype = dtype_of(k);
  a->k = const_cast<void*>(k.const_data_ptr()); a->v = const_cast<void*>(v.const_data_ptr());
  a->k_stride_b = ks.b; a->k_stride_t = ks.t; a->k_stride_h = ks.h;
  a->v_stride_b = vs.b; a->v_stride_t = vs.t; a->v_stride_h = vs.h;
}

// kv_write(pages, k, v, page_table, starts, offsets, max_new) -> True, or None
PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 7) {
    PyErr_SetString(PyExc_TypeError, "kv_write takes 7 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Pages pages;
    Tensor k, v, table, starts, offsets;
    HstuKvRowsArgs args;
    head(&args);
    if (!pages_arg(a[0], &pages) || !fill_pages(pages, &args.pages)) Py_RETURN_NONE;
    const auto dev = pages.t[0].device();
    int64_t max_new = 0;
    RowStrides ks, vs;
    if (!tensor_arg(a[1], &k) || !tensor_arg(a[2], &v) || !k.defined() || !v.defined() || !table_arg(a[3], dev, &table, &args.pages) ||
        !ints_arg(a[4], dev, args.pages.B, &starts)) Py_RETURN_NONE;
    const bool packed = a[5] != Py_None;
    if (packed && (!ints_arg(a[5], dev, (int64_t)args.pages.B + 1, &offsets) || !long_arg(a[6], &max_new) || max_new < 0 || max_new > 1 << 30)) Py_RETURN_NONE;
    if (!packed && a[6] != Py_None) Py_RETURN_NONE;
    if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || !rows_ready(k, dev, args.pages, packed, &ks) || !rows_ready(v, dev, args.pages, packed, &vs) ||
        wants_grad({&k, &v}) || dual({&k, &v})) Py_RETURN_NONE;
    fill_rows(&args, starts, offsets, packed ? max_new : k.size(1), packed ? k.size(0) : 0, k, v, ks, vs);
    without_lock(k, [&] {
      serve_check(hstu_kv_write(&args, stream_of(pages.t[0])), "hstu_kv_write");
      return true;
    });
    Py_RETURN_TRUE;
  });
}

// kv_read(pages, page_table, starts, count, offsets, max_new, total, fp32) -> (k, v), or None
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 8) {
    PyErr_SetString(PyExc_TypeError, "kv_read takes 8 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Pages pages;
    Tensor table, starts, offsets, k, v;
    HstuKvRowsArgs args;
    head(&args);
    if (!pages_arg(a[0], &pages) || !fill_pages(pages, &args.pages)) Py_RETURN_NONE;
    const auto dev = pages.t[0].device();
    if (!table_arg(a[1], dev, &table, &args.pages) || !ints_arg(a[2], dev, args.pages.B, &starts)) Py_RETURN_NONE;
    const bool packed = a[4] != Py_None;
    int64_t n = 0, total = 0;
    if (packed) {
      if (a[3] != Py_None || !ints_arg(a[4], dev, (int64_t)args.pages.B + 1, &offsets) || !long_arg(a[5], &n) || !long_arg(a[6], &total)) Py_RETURN_NONE;
    } else if (!long_arg(a[3], &n) || a[5] != Py_None || a[6] != Py_None) {
      Py_RETURN_NONE;
    }
    if (n < 0 || n > 1 << 30 || total < 0 || total > MOST) Py_RETURN_NONE;
    const auto type = a[7] == Py_True ? at::kFloat : at::kBFloat16;
    without_lock(pages.t[0], [&] {
      const int64_t B = args.pages.B, H = args.pages.H, d = args.pages.d;
      const auto how = pages.t[0].options().dtype(type);
      const std::vector<int64_t> shape = packed ? std::vector<int64_t>{total, H, d} : std::vector<int64_t>{B, n, H, d};
      k = at::empty(shape, how);
      v = at::empty(shape, how);
      const RowStrides s{packed ? 0 : n * H * d, H * d, d};
      fill_rows(&args, starts, offsets, n, total, k, v, s, s);
      serve_check(hstu_kv_read(&args, stream_of(k)), "hstu_kv_read");
      return true;
    });
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
  });
}

// cached_attention(q, pages, page_table, lengths, max_len, offsets, max_new, n, alpha, pos_bias, timestamps, ts_bias, ts_bucket_size, out)
// -> Tensor, or None
PyObject* cached_attention(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 14) {
    PyErr_SetString(PyExc_TypeError, "cached_attention takes 14 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Pages pages;
    Tensor q, table_, lengths, offsets, pos, ts, ts_tab, out;
    HstuCachedAttnArgs args;
    head(&args);
    if (!pages_arg(a[1], &pages) || !fill_pages(pages, &args.pages)) Py_RETURN_NONE;
    const auto dev = pages.t[0].device();
    int64_t max_len, max_new = 0, heads, width;
    double n = 0.0, alpha, bucket;
    RowStrides qs, os;
    if (!tensor_arg(a[0], &q) || !q.defined() || !table_arg(a[2], dev, &table_, &args.pages) || !ints_arg(a[3], dev, args.pages.B, &lengths) ||
        !long_arg(a[4], &max_len) || max_len < 1 || max_len > 1 << 30) Py_RETURN_NONE;
    const bool packed = a[5] != Py_None;
    if (packed && (!ints_arg(a[5], dev, (int64_t)args.pages.B + 1, &offsets) || !long_arg(a[6], &max_new))) Py_RETURN_NONE;
    if (!packed && a[6] != Py_None) Py_RETURN_NONE;
    if ((a[7] != Py_None && (!float_arg(a[7], &n) || !(n > 0.0))) || !float_arg(a[8], &alpha) || !float_arg(a[12], &bucket)) Py_RETURN_NONE;
    if (!tensor_arg(a[9], &pos) || !tensor_arg(a[10], &ts) || !tensor_arg(a[11], &ts_tab) || !tensor_arg(a[13], &out)) Py_RETURN_NONE;
    if (!rows_ready(q, dev, args.pages, packed, &qs) || wants_grad({&q, &pos, &ts_tab, &out}) || dual({&q, &pos, &ts_tab})) Py_RETURN_NONE;
    if (!packed) max_new = q.size(1);
    if (max_new < 0 || max_new > 1 << 30) Py_RETURN_NONE;
    args.lengths = lengths.const_data_ptr<int32_t>();
    args.offsets = packed ? offsets.const_data_ptr<int32_t>() : nullptr;
    args.total_rows = packed ? q.size(0) : 0; args.rows_per_seq = (int32_t)max_new; args.dtype = dtype_of(q);
    args.max_len = (int32_t)max_len; args.alpha = (float)alpha; args.inv_n = (float)(1.0 / (n > 0.0 ? n : (double)max_len));
    if (pos.defined()) {
      if (!table(pos, dev, args.pages.H, &heads, &width) || width != 2 * max_len - 1) Py_RETURN_NONE;
      args.pos_tab = pos.const_data_ptr<float>();
      args.pos_heads = (int32_t)heads;
    }
    if (ts.defined() != ts_tab.defined()) Py_RETURN_NONE;
    if (ts.defined()) {
      if (!table(ts_tab, dev, args.pages.H, &heads, &width) || width < 1 || width > 129 || !plain(ts, dev, at::kLong) || ts.dim() != 2 ||
          ts.size(0) != args.pages.B || ts.size(1) != max_len || !(bucket > 0.0)) Py_RETURN_NONE;
      args.timestamps = ts.const_data_ptr<int64_t>();
      args.ts_tab = ts_tab.const_data_ptr<float>();
      args.ts_heads = (int32_t)heads; args.ts_buckets = (int32_t)width - 1; args.ts_bucket_size = (float)bucket;
    }
    if (out.defined() && (out.scalar_type() != q.scalar_type() || out.sizes() != q.sizes() || !apart(out) || !rows_ready(out, dev, args.pages, packed, &os))) Py_RETURN_NONE;
    without_lock(q, [&] {
      if (!out.defined()) {
        out = at::empty(q.sizes(), q.options().requires_grad(false));
        rows_ready(out, dev, args.pages, packed, &os);
      }
      args.q = q.const_data_ptr(); args.out = out.data_ptr();
      args.q_stride_b = qs.b; args.q_stride_t = qs.t; args.q_stride_h = qs.h;
      args.o_stride_b = os.b; args.o_stride_t = os.t; args.o_stride_h = os.h;
      Tensor scratch;
      if (const size_t need = hstu_cached_attn_workspace_bytes(&args)) {
        scratch = at::empty({(int64_t)need}, q.options().dtype(at::kByte).requires_grad(false));
        args.workspace = scratch.data_ptr();
        args.workspace_bytes = need;
      }
      serve_check(hstu_cached_attn(&args, stream_of(q)), "hstu_cached_attn");
      return true;
    });
    return THPVariable_Wrap(std::move(out));
  });
}

// ---------------------------------------------------------------------------
// log probabilities
// ---------------------------------------------------------------------------

// Rows of logits as the kernels read them: [rows, vocab] with one row stride.
bool logits_rows(const Tensor& x, int64_t* rows, int64_t* stride) {
  if (!x.is_cuda() || (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16) || x.dim() < 1) return false;
  const int64_t V = x.size(-1);
  if (V < 1 || V > 1 << 30 || (x.stride(-1) != 1 && V > 1)) return false;
  *rows = x.numel() / V;
  if (x.dim() == 2) { *stride = x.size(0) > 1 ? x.stride(0) : 0; return true; }
  *stride = V;
  return x.is_contiguous();
}

void fill_scores(HstuLogProbsArgs* a, const Tensor& x, int64_t rows, int64_t stride, const Tensor& tokens, int64_t per_row, int64_t top) {
  head(a);
  a->logits = x.const_data_ptr();
  a->rows = rows; a->stride = stride;
  a->vocab = (int32_t)x.size(-1); a->dtype = dtype_of(x); a->count = (int32_t)per_row; a->top = (int32_t)top;
  a->tokens = tokens.defined() ? tokens.const_data_ptr<int64_t>() : nullptr;
}

struct LogProbsBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable x, tokens, stats, top_tokens;
  int64_t per_row = 0, top = 0;
  bool asked[3] = {false, false, false};      // log_probs, entropy, top_log_probs: the outputs there are, in this order

  std::string name() const override { return "HstuLogProbsBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* s : {&x, &tokens, &stats, &top_tokens}) s->reset_data();
  }

  // The same gradient in torch's own steps, for derivatives of it.
  static Tensor plain_gradient(const Tensor& logits, const Tensor& ids, int64_t per_row, const Tensor& first, int64_t top, const Tensor (&g)[3]) {
    const int64_t V = logits.size(-1), rows = logits.numel() / V;
    const Tensor lp = at::log_softmax(logits.reshape({rows, V}).to(at::kFloat), -1), p = lp.exp();
    Tensor own = at::zeros_like(lp), total = at::zeros({rows, 1}, lp.options());
    if (g[0].defined()) {
      const Tensor id = ids.reshape({rows, per_row}), gi = g[0].reshape({rows, per_row}).masked_fill(id < 0, 0.0).masked_fill(id >= V, NAN);
      own = own.scatter_add(1, id.clamp(0, V - 1), gi);
      total = total + gi.sum(-1, true);
    }
    if (g[2].defined()) {
      const Tensor gi = g[2].reshape({rows, top});
      own = own.scatter_add(1, first.reshape({rows, top}), gi);
      total = total + gi.sum(-1, true);
    }
    if (g[1].defined()) {
      const Tensor there = at::where(p == 0, at::zeros_like(lp), lp), h = -(p * there).sum(-1, true);
      total = total + g[1].reshape({rows, 1}) * (there + h);
    }
    return (own - p * total).to(logits.scalar_type()).view(logits.sizes());
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    torch::autograd::variable_list r(1);
    Tensor g[3];
    size_t at = 0;
    for (int i = 0; i < 3; ++i)
      if (asked[i]) { if (at < grads.size()) g[i] = grads[at]; ++at; }
    if ((!g[0].defined() && !g[1].defined() && !g[2].defined()) || !task_should_compute_output(0)) return r;
    const Tensor logits = x.unpack();
    const Tensor ids = per_row > 0 ? tokens.unpack() : Tensor(), first = top > 0 ? top_tokens.unpack() : Tensor();
    const c10::DeviceGuard guard(logits.device());
    if (at::GradMode::is_enabled()) {
      r[0] = plain_gradient(logits, ids, per_row, first, top, g);
      return r;
    }
    const at::NoGradGuard no_grad;
    int64_t rows, stride;
    TORCH_CHECK(logits_rows(logits, &rows, &stride), "the saved logits do not fit the call");
    const Tensor st = stats.unpack();
    HstuLogProbsArgs a;
    fill_scores(&a, logits, rows, stride, ids, per_row, top);
    for (Tensor& t : g)
      if (t.defined()) t = t.to(at::kFloat).contiguous();
    const Tensor d = at::empty(logits.sizes(), logits.options().requires_grad(false));
    a.stats = const_cast<float*>(st.const_data_ptr<float>());
    a.top_tokens = first.defined() ? const_cast<int64_t*>(first.const_data_ptr<int64_t>()) : nullptr;
    a.g_tokens = g[0].defined() ? g[0].const_data_ptr<float>() : nullptr;
    a.g_entropy = g[1].defined() ? g[1].const_data_ptr<float>() : nullptr;
    a.g_top = g[2].defined() ? g[2].const_data_ptr<float>() : nullptr;
    a.d_logits = d.data_ptr();
    a.d_stride = logits.size(-1);
    serve_check(hstu_log_probs_bwd(&a, stream_of(logits)), "hstu_log_probs_bwd");
    r[0] = d;
    return r;
  }
};

// Gives `f` every accumulator of a leaf that a backward pass from x would reach.  (A leaf's own is there for as long as
// somebody holds it, and may be made for this walk: the edge is held until the end.)
template <typename F>
void each_accumulator(const Tensor& x, F&& f) {
  const torch::autograd::Edge root = torch::autograd::impl::gradient_edge(x);
  std::vector<torch::autograd::Node*> todo{root.function.get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!todo.empty()) {
    torch::autograd::Node* const node = todo.back();
    todo.pop_back();
    if (!node || !seen.insert(node).second) continue;
    for (const auto& e : node->next_edges()) todo.push_back(e.function.get());
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node)) f(node);
  }
}

// A backward pass into a graph waits for the streams of the leaves' accumulators.  Those that an eager graph of the same leaves made, and
// keeps alive, belong to a stream that is not captured: the wait fails on the engine's thread and takes the process with it.
void refuse_mixed_graphs(const Tensor& x) {
  if (!capturing(stream_of(x))) return;
  const c10::Stream here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).unwrap();
  each_accumulator(x, [&](torch::autograd::Node* node) {
    const auto stream = node->stream();
    if (!stream || *stream == here) return;
    // (the default stream may not be asked while another is captured)
    void* const other = (void*)c10::hip::HIPStreamMasqueradingAsCUDA(*stream).stream();
    TORCH_CHECK_VALUE(other && capturing(other),
                      "token_log_probs is captured with a gradient while an eager graph of the same leaves lives: let go of its outputs first");
  });
}

// accumulators(tensor) -> how many leaves' accumulators a backward pass from it reaches
PyObject* accumulators(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 1 || !THPVariable_Check(a[0])) {
    PyErr_SetString(PyExc_TypeError, "accumulators takes a tensor");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const Tensor x = THPVariable_Unpack(a[0]);
    int64_t n = 0;
    if (x.requires_grad()) each_accumulator(x, [&](torch::autograd::Node*) { ++n; });
    return PyLong_FromLongLong(n);
  });
}

// token_log_probs(logits, tokens, top, entropy) -> (log_probs, entropy, top_log_probs, top_tokens), each a tensor or None; or None
PyObject* token_log_probs(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 4) {
    PyErr_SetString(PyExc_TypeError, "token_log_probs takes 4 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Tensor x, tokens;
    int64_t top, rows, stride;
    if (!tensor_arg(a[0], &x) || !x.defined()) Py_RETURN_NONE;
    if (x.is_cuda() && wants_grad({&x})) refuse_mixed_graphs(x);
    if (!tensor_arg(a[1], &tokens) || !long_arg(a[2], &top) || !logits_rows(x, &rows, &stride)) Py_RETURN_NONE;
    if (a[3] != Py_True && a[3] != Py_False) Py_RETURN_NONE;
    const bool entropy = a[3] == Py_True;
    const int64_t V = x.size(-1);
    if (top < 0 || top > std::min<int64_t>(V, 256) || rows < 1 || dual({&x})) Py_RETURN_NONE;
    if (!tokens.defined() && !entropy && top == 0) Py_RETURN_NONE;
    int64_t per_row = 0;
    if (tokens.defined()) {
      if (!plain(tokens, x.device(), at::kLong) || tokens.numel() < 1) Py_RETURN_NONE;
      const int64_t lead = x.dim() - 1;
      if (tokens.dim() != lead && tokens.dim() != lead + 1) Py_RETURN_NONE;
      for (int64_t i = 0; i < lead; ++i)
        if (tokens.size(i) != x.size(i)) Py_RETURN_NONE;
      per_row = tokens.dim() == lead ? 1 : tokens.size(lead);
      if (per_row > 1 << 30) Py_RETURN_NONE;
    }
    const bool graph = wants_grad({&x});
    Tensor lp, ent, stats, tl, ti;
    without_lock(x, [&] {
      const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
      std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
      if (per_row) lp = at::empty(tokens.sizes(), f32);
      if (entropy) ent = at::empty(shape, f32);
      if (graph) stats = at::empty({rows, 3}, f32);
      if (top) {
        shape.push_back(top);
        tl = at::empty(shape, f32);
        ti = at::empty(shape, f32.dtype(at::kLong));
      }
      HstuLogProbsArgs args;
      fill_scores(&args, x, rows, stride, tokens, per_row, top);
      if (lp.defined()) args.log_probs = lp.data_ptr<float>();
      if (entropy) args.entropy = ent.data_ptr<float>();
      if (graph) args.stats = stats.data_ptr<float>();
      if (top) { args.top_log_probs = tl.data_ptr<float>(); args.top_tokens = ti.data_ptr<int64_t>(); }
      Tensor scratch;
      if (const size_t need = hstu_log_probs_workspace_bytes(&args)) {
        scratch = at::empty({(int64_t)need}, f32.dtype(at::kByte));
        args.workspace = scratch.data_ptr();
        args.workspace_bytes = need;
      }
      serve_check(hstu_log_probs_fwd(&args, stream_of(x)), "hstu_log_probs_fwd");
      return true;
    });
    if (graph) {
      auto node = std::shared_ptr<LogProbsBackward>(new LogProbsBackward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(x));
      node->x = keep(x);
      node->stats = keep(stats);
      if (per_row) node->tokens = keep(tokens);
      if (top) node->top_tokens = keep(ti);
      node->per_row = per_row;
      node->top = top;
      const Tensor* outs[3] = {&lp, &ent, &tl};
      for (int i = 0; i < 3; ++i)
        if ((node->asked[i] = outs[i]->defined())) torch::autograd::set_history(*outs[i], node);
    }
    auto wrap = [](Tensor& t) -> PyObject* {
      if (t.defined()) return THPVariable_Wrap(std::move(t));
      Py_RETURN_NONE;
    };
    return Py_BuildValue("(NNNN)", wrap(lp), wrap(ent), wrap(tl), wrap(ti));
  });
}

PyMethodDef methods[] = {
#define HSTU_FAST(name, doc) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, doc}
    HSTU_FAST(check_pages, "Whether tensors are the pages of a cache."),
    HSTU_FAST(kv_write, "New events' keys and values into the pages."),
    HSTU_FAST(kv_read, "The keys and values that pages stand for."),
    HSTU_FAST(cached_attention, "The attention of new events over a cache."),
    HSTU_FAST(token_log_probs, "Log probabilities of tokens (differentiable)."),
    HSTU_FAST(accumulators, "How many leaves a backward pass from a tensor reaches."),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native_serve", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native_serve(void) { return PyModule_Create(&module); }
