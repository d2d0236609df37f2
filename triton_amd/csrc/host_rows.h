// The row operators' half of the native host path (included by host_path.cpp): layer norm, token log probabilities and distillation from
// top logits, with their autograd nodes.
//
// What bounds it: a training step's call makes an autograd node, whose backward pass runs on a thread of its own.  With nodes written in
// Python that thread and the caller's pass the interpreter's lock to and fro: some 100 us a call of forward and backward where the kernels
// take 10.  These nodes need the lock for the stream's address only.
#pragma once
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <unordered_set>
#include <vector>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool row_dtype(const Tensor& t) {
  return t.scalar_type() == ScalarType::Float || t.scalar_type() == ScalarType::BFloat16 || t.scalar_type() == ScalarType::Half;
}
bool index_type(const Tensor& t) { return t.scalar_type() == ScalarType::Long || t.scalar_type() == ScalarType::Int; }
// A dual tensor's tangent is dropped by whoever reads its data: such calls are left to the Python path, which refuses them.
bool dual(const Tensor& t) { return t._fw_grad(0).defined(); }
bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
bool on_device_of(const Tensor& t, const Tensor& x) { return t.is_cuda() && t.get_device() == x.get_device(); }
// Whether a backward pass from t runs a node on the default stream: the accumulation of a leaf's gradient, for the sake of a graph of this
// process that still lives, or an operation in front of t.  A backward pass that is captured would make the default stream wait for the
// capture, which ends the process.
bool on_default_stream(torch::autograd::Node* node) {
  const auto stream = node->stream();
  return stream && stream->id() == 0;
}
bool kept_by_default_stream(const Tensor& t) {
  if (!t.requires_grad()) return false;
  if (!t.grad_fn()) {
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    return node && on_default_stream(node.get());
  }
  std::vector<torch::autograd::Node*> todo = {t.grad_fn().get()};
  std::unordered_set<torch::autograd::Node*> seen = {todo[0]};
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    if (on_default_stream(node)) return true;
    for (const auto& edge : node->next_edges())
      if (edge.function && seen.insert(edge.function.get()).second) todo.push_back(edge.function.get());
  }
  return false;
}
// Whether the current stream, `stream`, is being captured (the default stream never is).  The callers leave captured calls with such leaves
// to the Python path, which refuses them; outside a capture the default stream may well wait, and the nodes of this file are 50 to 70 us a
// call faster than Python's.
bool captured(void* stream) {
  if (!stream) return false;
  Ref r(PyObject_CallNoArgs(B.capturing));
  if (!r) throw PyError();
  return PyObject_IsTrue(r) != 0;
}
float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int32_t code_of(const Tensor& t) { return t.defined() ? dtype_code(t.scalar_type()) : TK_F32; }

// ---- on the thread of a backward pass: the tensor's device made current, its stream, and the call ----------------------------------
template <class F>
void backward_call(const Tensor& t, F&& f) {
  c10::OptionalDeviceGuard guard(t.device());
  void* stream = nullptr;
  {
    const PyGILState_STATE gil = PyGILState_Ensure();
    bool known = false;
    try {
      if (auto s = stream_of(t)) stream = *s, known = true;
    } catch (const PyError&) {
      PyErr_Clear();
    }
    PyGILState_Release(gil);
    TORCH_CHECK(known, "the stream of a backward pass is not known");
  }
  const int32_t status = f(stream);
  TORCH_CHECK(status == TK_OK, B.last_error());
}

// A saved tensor as the kernels take it.  Hooks on saved tensors (offloading, compression, recomputation) may give back another layout,
// which is copied; another shape or device, or a type that its place does not take, is an error before anything reads it.
enum class Kind { ROWS, INDEX, STATS };
Tensor unpacked(const Tensor& t, at::IntArrayRef sizes, const Tensor& like, Kind kind) {
  const bool type = t.defined() && (kind == Kind::ROWS ? row_dtype(t) : kind == Kind::INDEX ? index_type(t) : t.scalar_type() == ScalarType::Float);
  TORCH_CHECK(type && t.sizes() == sizes && t.device() == like.device(), "a tensor saved by the forward pass came back with another shape, type or device");
  return kind == Kind::STATS || t.dim() != 2 || t.stride(1) != 1 ? t.contiguous() : t;
}

// Gradients that are themselves to be differentiated (create_graph) raise an error when they are.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>("the row operators are differentiable once", (int64_t)grads.size());
  return (*node)(std::move(grads));
}

// ---- layer norm ---------------------------------------------------------------------------------------------------------------------

struct LayerNormRows {  // the rows of a tensor whose last dimension is dense
  int64_t M, C, stride;
  explicit LayerNormRows(const Tensor& t) : M(t.numel() / t.size(-1)), C(t.size(-1)), stride(t.dim() == 2 ? t.stride(0) : C) {}
};
bool dense_rows(const Tensor& t) { return t.is_contiguous() || (t.dim() == 2 && t.stride(1) == 1); }

variable_list layer_norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, void* stream, bool with_stats) {
  const LayerNormRows r(x);
  Tensor y = empty(x.sizes(), x.scalar_type(), x), stats;
  if (with_stats) stats = empty({2, r.M}, ScalarType::Float, x);
  float* mean = floats(stats);
  launch([&] {
    return B.layer_norm(x.data_ptr(), dtype_code(x.scalar_type()), r.M, r.C, r.stride, data(w), code_of(w), data(b), code_of(b), (float)eps, y.data_ptr(), r.C,
                        mean, mean ? mean + r.M : nullptr, stream);
  });
  return {y, stats};
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps, int64_t stream) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    variable_list out = layer_norm_forward(x, w, b, eps, reinterpret_cast<void*>(stream), true);
    ctx->save_for_backward({x, w, b, out[1]});
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor x = unpacked(saved[0], grads[0].sizes(), grads[0], Kind::ROWS);
    const int64_t cols = x.size(-1);
    const Tensor w = saved[1].defined() ? unpacked(saved[1], {cols}, x, Kind::ROWS) : saved[1], b = saved[2].defined() ? unpacked(saved[2], {cols}, x, Kind::ROWS) : saved[2];
    const Tensor stats = unpacked(saved[3], {2, x.numel() / cols}, x, Kind::STATS);
    // (the numbers of the inputs count the tensors that there are)
    const bool need_x = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(1),
               need_b = b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1);
    const Tensor g0 = grads[0].to(x.scalar_type()), dy = dense_rows(g0) ? g0 : g0.contiguous();
    const LayerNormRows r(x), g(dy);
    Tensor dx, dw, db;
    backward_call(x, [&](void* stream) {
      Tensor ws;
      if (need_x) dx = empty(x.sizes(), x.scalar_type(), x);
      if (need_w) dw = empty({r.C}, w.scalar_type(), x);
      if (need_b) db = empty({r.C}, b.scalar_type(), x);
      if (need_w || need_b) ws = empty({B.layer_norm_workspace(r.M, r.C)}, ScalarType::Byte, x);
      return B.layer_norm_backward(dy.data_ptr(), g.stride, x.data_ptr(), dtype_code(x.scalar_type()), r.M, r.C, r.stride, data(w), code_of(w), floats(stats),
                                   floats(stats) + r.M, data(dx), r.C, data(dw), data(db), code_of(b), data(ws), stream);
    });
    return once({dx, dw, db, Tensor(), Tensor()});
  }
};

// (x, weight, bias, eps)
PyObject* run_layer_norm(PyObject* const* v) {
  const Tensor* x = tensor_of(v[0]);
  const Tensor *w = tensor_of(v[1]), *b = tensor_of(v[2]);
  const double eps = PyFloat_AsDouble(v[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (!x || !x->is_cuda() || x->dim() < 1 || x->numel() == 0 || !row_dtype(*x) || !dense_rows(*x) || dual(*x) || !(eps >= 0. && eps <= 3e38)) return none();
  for (auto [t, o] : {std::pair(w, v[1]), std::pair(b, v[2])}) {
    if (!t && !is_none(o)) return none();
    if (t && (!on_device_of(*t, *x) || !row_dtype(*t) || t->dim() != 1 || t->size(0) != x->size(-1) || !t->is_contiguous() || dual(*t))) return none();
  }
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*x);
  if (!stream) return none();
  const Tensor no, &wt = w ? *w : no, &bt = b ? *b : no;
  if (wants_grad(*x) || (w && wants_grad(*w)) || (b && wants_grad(*b))) {
    if (captured(*stream) && (kept_by_default_stream(*x) || (w && kept_by_default_stream(*w)) || (b && kept_by_default_stream(*b)))) return none();
    return THPVariable_Wrap(LayerNormNode::apply(*x, w ? std::optional<Tensor>(*w) : std::nullopt, b ? std::optional<Tensor>(*b) : std::nullopt, eps,
                                                 reinterpret_cast<int64_t>(*stream)));
  }
  return THPVariable_Wrap(layer_norm_forward(*x, wt, bt, eps, *stream, false)[0]);
}

// ---- rows over a vocabulary -----------------------------------------------------------------------------------------------------------

bool plain_logits(const Tensor* z, double temperature) {
  return z && z->is_cuda() && z->dim() == 2 && z->numel() != 0 && z->stride(1) == 1 && row_dtype(*z) && temperature >= 1.2e-38 && temperature <= 3e38
         && z->size(0) <= 0x7FFFFFFF && z->size(1) <= 1 << 30 && !dual(*z);
}
tk_vocab_desc vocab_desc(const Tensor& z, double temperature) {
  tk_vocab_desc d = {};
  d.logits = z.data_ptr(), d.logits_dtype = dtype_code(z.scalar_type()), d.logits_stride_m = z.stride(0);
  d.n_rows = (int32_t)z.size(0), d.vocab = (int32_t)z.size(1), d.temperature = (float)temperature;
  return d;
}
Tensor vocab_workspace(const tk_vocab_desc& d, const Tensor& like) {
  const int64_t n = B.vocab_workspace(d.n_rows, d.vocab, d.k);
  return n ? empty({n}, ScalarType::Byte, like) : Tensor();
}
// A gradient of a row's output, and the number of elements between rows
const float* row_gradient(const Tensor& g, int64_t* stride) {
  *stride = g.defined() && g.size(0) > 1 ? g.stride(0) : 0;
  return floats(g);
}

// logprobs, entropy, stats, and with k top_logprobs and top_indx
std::array<Tensor, 5> logprobs_forward(const Tensor& z, const Tensor& tokens, int64_t k, double temperature, void* stream, bool with_stats) {
  const int64_t T = z.size(0);
  std::array<Tensor, 5> o = {empty({T}, ScalarType::Float, z), empty({T}, ScalarType::Float, z)};
  if (with_stats) o[2] = empty({2, T}, ScalarType::Float, z);
  if (k) o[3] = empty({T, k}, ScalarType::Float, z), o[4] = empty({T, k}, ScalarType::Int, z);
  tk_vocab_desc d = vocab_desc(z, temperature);
  d.tokens = tokens.data_ptr(), d.tokens_i64 = tokens.scalar_type() == ScalarType::Long;
  d.logprobs = floats(o[0]), d.entropy = floats(o[1]), d.stats = floats(o[2]);
  d.k = (int32_t)k, d.top_logprobs = floats(o[3]), d.top_indx = static_cast<int32_t*>(data(o[4]));
  const Tensor ws = vocab_workspace(d, z);
  d.workspace = data(ws);
  launch([&] { return B.token_logprobs(&d, stream); });
  return o;
}

struct LogprobsNode : torch::autograd::Function<LogprobsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& tokens, int64_t k, double temperature, int64_t stream) {
    auto o = logprobs_forward(z, tokens, k, temperature, reinterpret_cast<void*>(stream), true);
    ctx->save_for_backward({z, tokens, o[1], o[2]});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["vocab"] = z.size(1);
    ctx->set_materialize_grads(false);
    if (!k) return {o[0], o[1]};
    ctx->mark_non_differentiable({o[3], o[4]});
    return {o[0], o[1], o[3], o[4]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    Tensor dz;
    if (grads[0].defined() || grads[1].defined()) {
      const Tensor& g = grads[0].defined() ? grads[0] : grads[1];
      const int64_t T = g.size(0);
      const Tensor z = unpacked(saved[0], {T, ctx->saved_data["vocab"].toInt()}, g, Kind::ROWS), tokens = unpacked(saved[1], {T}, g, Kind::INDEX);
      const Tensor entropy = unpacked(saved[2], {T}, g, Kind::STATS), stats = unpacked(saved[3], {2, T}, g, Kind::STATS);
      backward_call(z, [&](void* stream) {
        dz = empty(z.sizes(), z.scalar_type(), z);
        tk_vocab_desc d = vocab_desc(z, ctx->saved_data["temperature"].toDouble());
        d.tokens = tokens.data_ptr(), d.tokens_i64 = tokens.scalar_type() == ScalarType::Long;
        d.entropy = floats(entropy), d.stats = floats(stats);
        d.d_logprobs = row_gradient(grads[0], &d.d_logprobs_stride), d.d_entropy = row_gradient(grads[1], &d.d_entropy_stride);
        d.d_logits = dz.data_ptr(), d.d_logits_stride_m = dz.size(1);
        return B.token_logprobs_backward(&d, stream);
      });
    }
    return once({dz, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// (logits, tokens, k, temperature): the four fields of TokenLogprobs
PyObject* run_token_logprobs(PyObject* const* v) {
  const Tensor *z = tensor_of(v[0]), *tokens = tensor_of(v[1]);
  const int64_t k = PyLong_AsLongLong(v[2]);
  const double temperature = PyFloat_AsDouble(v[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (!plain_logits(z, temperature) || k < 0 || k > z->size(1) || k > TK_VOCAB_MAX_TOP || (k && z->size(1) > TK_VOCAB_MAX_TOP_COLUMNS)) return none();
  if (!tokens || !on_device_of(*tokens, *z) || !index_type(*tokens) || tokens->dim() != 1 || tokens->size(0) != z->size(0) || !tokens->is_contiguous())
    return none();
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*z);
  if (!stream) return none();
  variable_list o;
  if (wants_grad(*z)) {
    if (captured(*stream) && kept_by_default_stream(*z)) return none();
    o = LogprobsNode::apply(*z, *tokens, k, temperature, reinterpret_cast<int64_t>(*stream));
  } else {
    auto f = logprobs_forward(*z, *tokens, k, temperature, *stream, false);
    o = {f[0], f[1], f[3], f[4]};
  }
  Ref lp(THPVariable_Wrap(o[0])), h(THPVariable_Wrap(o[1]));
  Ref top(k ? THPVariable_Wrap(o[2]) : none()), indx(k ? THPVariable_Wrap(o[3]) : none());
  if (!lp.p || !h.p || !top.p || !indx.p) throw PyError();
  return PyTuple_Pack(4, lp.p, h.p, top.p, indx.p);
}

void set_teacher(tk_vocab_desc& d, const Tensor& q, const Tensor& at) {
  d.teacher_logits = q.data_ptr(), d.teacher_dtype = dtype_code(q.scalar_type()), d.teacher_stride_m = q.stride(0);
  d.teacher_indx = at.data_ptr(), d.teacher_indx_i64 = at.scalar_type() == ScalarType::Long, d.teacher_indx_stride_m = at.stride(0);
  d.n_teacher = (int32_t)q.size(1);
}

// loss, and the statistics of the student's and the teacher's rows
std::array<Tensor, 2> distill_forward(const Tensor& z, const Tensor& q, const Tensor& at, double temperature, void* stream, bool with_stats) {
  const int64_t T = z.size(0);
  std::array<Tensor, 2> o = {empty({T}, ScalarType::Float, z)};
  tk_vocab_desc d = vocab_desc(z, temperature);
  set_teacher(d, q, at);
  d.loss = floats(o[0]);
  if (with_stats) {
    o[1] = empty({4, T}, ScalarType::Float, z);
    d.stats = floats(o[1]), d.teacher_stats = d.stats + 2 * T;
  }
  const Tensor ws = vocab_workspace(d, z);
  d.workspace = data(ws);
  launch([&] { return B.distill_topk(&d, stream); });
  return o;
}

struct DistillNode : torch::autograd::Function<DistillNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& q, const Tensor& at, double temperature, int64_t stream) {
    auto o = distill_forward(z, q, at, temperature, reinterpret_cast<void*>(stream), true);
    ctx->save_for_backward({z, q, at, o[1]});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["vocab"] = z.size(1);
    ctx->saved_data["entries"] = q.size(1);
    return o[0];
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const int64_t T = grads[0].size(0), K = ctx->saved_data["entries"].toInt();
    const Tensor z = unpacked(saved[0], {T, ctx->saved_data["vocab"].toInt()}, grads[0], Kind::ROWS), q = unpacked(saved[1], {T, K}, z, Kind::ROWS);
    const Tensor at = unpacked(saved[2], {T, K}, z, Kind::INDEX), stats = unpacked(saved[3], {4, T}, z, Kind::STATS);
    Tensor dz;
    backward_call(z, [&](void* stream) {
      dz = empty(z.sizes(), z.scalar_type(), z);
      tk_vocab_desc d = vocab_desc(z, ctx->saved_data["temperature"].toDouble());
      set_teacher(d, q, at);
      d.stats = floats(stats), d.teacher_stats = d.stats + 2 * z.size(0);
      d.d_loss = row_gradient(grads[0], &d.d_loss_stride);
      d.d_logits = dz.data_ptr(), d.d_logits_stride_m = dz.size(1);
      return B.distill_topk_backward(&d, stream);
    });
    return once({dz, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// (logits, teacher logits, teacher indices, temperature)
PyObject* run_distill_topk(PyObject* const* v) {
  const Tensor *z = tensor_of(v[0]), *q = tensor_of(v[1]), *at = tensor_of(v[2]);
  const double temperature = PyFloat_AsDouble(v[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (!plain_logits(z, temperature) || !q || !at) return none();
  if (!on_device_of(*q, *z) || !row_dtype(*q) || q->dim() != 2 || q->size(0) != z->size(0) || q->size(1) < 1 || q->size(1) > TK_VOCAB_MAX_TEACHER
      || q->stride(1) != 1 || wants_grad(*q) || dual(*q))
    return none();
  if (!on_device_of(*at, *z) || !index_type(*at) || at->sizes() != q->sizes() || at->stride(1) != 1) return none();
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*z);
  if (!stream) return none();
  if (wants_grad(*z)) {
    if (captured(*stream) && kept_by_default_stream(*z)) return none();
    return THPVariable_Wrap(DistillNode::apply(*z, *q, *at, temperature, reinterpret_cast<int64_t>(*stream)));
  }
  return THPVariable_Wrap(distill_forward(*z, *q, *at, temperature, *stream, false)[0]);
}

PyObject* run_kept_by_default_stream(PyObject* const* v) {
  const Tensor* t = tensor_of(v[0]);
  return PyBool_FromLong(t && kept_by_default_stream(*t));
}

}  // namespace
