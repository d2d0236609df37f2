// The native host path of e4m3 in blocks of 128 (included by host_path.cpp): the quantiser and its inverse, the ragged product, the linear layer and swiglu with
// their autograd nodes.  Calls of another form than these functions name are left to fp8_blocks.py, which checks, copies and refuses.
//
// What bounds it: in Python a product took 15 us, the quantiser with its inverse 30, a step of swiglu 113 and one of the linear layer 220, at sizes whose kernels take
// 2 to 30.
#pragma once
#include <ATen/SavedTensorHooks.h>

namespace {

constexpr int64_t kFp8 = 128, kFp8Rows = 64, kFp8Most = 0x7FFFFF00;  // a block; the row blocks of the schedule that the product's kernels go by; the most of a size
int64_t fp8_blocks(int64_t n) { return (n + kFp8 - 1) / kFp8; }
int64_t fp8_pitch(int64_t n) { return (n + 15) / 16 * 16; }
bool is_e4m3(const Tensor& t) { return t.scalar_type() == ScalarType::Float8_e4m3fn; }
bool plain_scales(const Tensor* s, const Tensor& like, at::IntArrayRef sizes) {
  return s && on_device_of(*s, like) && s->scalar_type() == ScalarType::Float && s->sizes() == sizes && !wants_grad(*s) && !dual(*s);
}

// [.., R, C] e4m3 whose rows begin at sixteen-byte boundaries
Tensor fp8_values(int64_t R, int64_t C, const Tensor& like) { return empty_strided({R, C}, {fp8_pitch(C), 1}, ScalarType::Float8_e4m3fn, like); }
Tensor fp8_values(int64_t E, int64_t R, int64_t C, const Tensor& like) {
  return empty_strided({E, R, C}, {R * fp8_pitch(C), fp8_pitch(C), 1}, ScalarType::Float8_e4m3fn, like);
}
uint8_t* bytes(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

// Rows of x (2-D, dense columns) in 8 bits: a status, and the results
struct Fp8Rows {
  Tensor v, s;
  int32_t make(const Tensor& x, void* stream) {
    const int64_t R = x.size(0), C = x.size(1);
    v = fp8_values(R, C, x), s = empty({R, fp8_blocks(C)}, ScalarType::Float, x);
    return B.fp8_downcast(x.data_ptr(), dtype_code(x.scalar_type()), 1, R, C, 0, x.stride(0), 1, bytes(v), 0, v.stride(0), nullptr, 0, 0, floats(s), 0, s.size(1), 1, stream);
  }
};

// ---- the quantiser and its inverse: 2-D, blocks of a row or of 128 x 128 -------------------------------------------------------------------------------
// (x, block rows)
PyObject* run_fp8_downcast(PyObject* const* v) {
  const Tensor* x = tensor_of(v[0]);
  const long block = PyLong_Check(v[1]) ? PyLong_AsLong(v[1]) : -1;
  if (!x || !x->is_cuda() || x->dim() != 2 || x->numel() == 0 || x->stride(1) != 1 || !row_dtype(*x) || wants_grad(*x) || dual(*x) || (block != 1 && block != kFp8)) return none();
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*x);
  if (!stream) return none();
  const int64_t R = x->size(0), C = x->size(1);
  Tensor q = fp8_values(R, C, *x), s = empty({(R + block - 1) / block, fp8_blocks(C)}, ScalarType::Float, *x);
  launch([&] {
    return B.fp8_downcast(x->data_ptr(), dtype_code(x->scalar_type()), 1, R, C, 0, x->stride(0), (int32_t)block, bytes(q), 0, q.stride(0), nullptr, 0, 0, floats(s), 0, s.size(1), 1,
                          *stream);
  });
  Ref qo(THPVariable_Wrap(std::move(q))), so(THPVariable_Wrap(std::move(s)));
  if (!qo.p || !so.p) throw PyError();
  return PyTuple_Pack(2, qo.p, so.p);
}

// (values, scales, dtype, block rows)
PyObject* run_fp8_upcast(PyObject* const* v) {
  const Tensor *q = tensor_of(v[0]), *s = tensor_of(v[1]);
  const long block = PyLong_Check(v[3]) ? PyLong_AsLong(v[3]) : -1;
  if (!q || !q->is_cuda() || q->dim() != 2 || q->numel() == 0 || q->stride(1) != 1 || !is_e4m3(*q) || wants_grad(*q) || !THPDtype_Check(v[2]) || (block != 1 && block != kFp8)) return none();
  const ScalarType out = reinterpret_cast<THPDtype*>(v[2])->scalar_type;
  const int64_t R = q->size(0), C = q->size(1);
  if ((out != ScalarType::Float && out != ScalarType::BFloat16 && out != ScalarType::Half) || !plain_scales(s, *q, {(R + block - 1) / block, fp8_blocks(C)})) return none();
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*q);
  if (!stream) return none();
  Tensor y = empty({R, C}, out, *q);
  launch([&] {
    return B.fp8_upcast(bytes(*q), 1, R, C, 0, q->stride(0), (int32_t)block, floats(*s), 0, s->stride(0), s->stride(1), y.data_ptr(), dtype_code(out), 0, C, *stream);
  });
  return THPVariable_Wrap(std::move(y));
}

// ---- the ragged product ----------------------------------------------------------------------------------------------------------------------------------

struct Fp8Lines {  // weights [E, K, N] as the product reads them: lines along K
  const uint8_t* w;
  int64_t e, n;
  const float* s;
  int64_t s_e, s_k, s_n;
};
struct Fp8Slices {  // a ragged call's metadata (undefined: one slice)
  Tensor sizes, offs, schedule;
};
tk_fp8_gemm_desc fp8_desc(const Tensor& a, const Tensor& s, const Fp8Lines& w, int64_t E, int64_t M, int64_t N, const Fp8Slices& md, Tensor& y) {
  tk_fp8_gemm_desc d = {};
  d.x = bytes(a), d.x_stride_m = a.stride(0), d.x_rows = a.size(0);
  d.x_scale = floats(s), d.xs_stride_m = s.stride(0), d.xs_stride_k = s.stride(1);
  d.w = w.w, d.w_stride_e = w.e, d.w_stride_n = w.n;
  d.w_scale = w.s, d.ws_stride_e = w.s_e, d.ws_stride_k = w.s_k, d.ws_stride_n = w.s_n;
  d.n_slices = (int32_t)E, d.M = (int32_t)M, d.N = (int32_t)N, d.K = (int32_t)a.size(1);
  if (md.sizes.defined()) {
    d.slice_sizes = static_cast<int32_t*>(data(md.sizes)), d.slice_offs = static_cast<int32_t*>(data(md.offs));
    d.block_schedule = static_cast<int32_t*>(data(md.schedule)) + 2 * md.schedule.stride(0);  // (block sizes 16, 32, 64, ..)
    d.grid_m = (int32_t)std::min(n_blocks(E, M, kFp8Rows), md.schedule.size(1));
  }
  d.y = y.data_ptr(), d.y_dtype = dtype_code(y.scalar_type()), d.y_stride_m = y.size(1);
  return d;
}
bool read_slices(PyObject* o, const Tensor& like, int64_t E, Fp8Slices* md) {
  if (is_none(o)) return E == 1;
  Metadata m;
  if (!m.read(o) || m.sizes->size(0) != E || !on_device_of(*m.sizes, like) || m.schedule->size(0) < 3 || m.offs->size(0) <= E) return false;
  md->sizes = *m.sizes, md->offs = *m.offs, md->schedule = *m.schedule;
  return true;
}
bool lines_aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) | (uint64_t)t.stride(0)) % 16 == 0; }

// (a, a scale, w, w scale, bias, metadata, gather, scatter, gammas, activation, output type)
PyObject* run_fp8_matmul(PyObject* const* v) {
  const Tensor *a = tensor_of(v[0]), *as = tensor_of(v[1]), *w = tensor_of(v[2]), *ws = tensor_of(v[3]), *gather, *scatter, *bias = nullptr, *gammas = nullptr;
  if (!a || !a->is_cuda() || a->dim() != 2 || !is_e4m3(*a) || wants_grad(*a) || a->stride(1) != 1 || a->numel() == 0 || !plain_scales(as, *a, {a->size(0), fp8_blocks(a->size(1))})) return none();
  if (!w || !on_device_of(*w, *a) || w->dim() != 3 || !is_e4m3(*w) || wants_grad(*w) || w->stride(1) != 1 || w->size(1) != a->size(1) || w->numel() == 0) return none();
  const int64_t E = w->size(0), K = w->size(1), N = w->size(2);
  if (!plain_scales(ws, *a, {E, fp8_blocks(K), fp8_blocks(N)})) return none();
  Activation act;
  Fp8Slices md;
  if (!plain_index(v[6], &gather) || !plain_index(v[7], &scatter) || !act.read(v[9]) || !THPDtype_Check(v[10]) || !read_slices(v[5], *a, E, &md)) return none();
  for (const Tensor* i : {gather, scatter})
    if (i && !on_device_of(*i, *a)) return none();
  const ScalarType out = reinterpret_cast<THPDtype*>(v[10])->scalar_type;
  if ((out != ScalarType::Float && out != ScalarType::BFloat16 && out != ScalarType::Half) || (act.swiglu && N % 2)) return none();
  const int64_t M = gather ? gather->size(0) : a->size(0);
  if (!is_none(v[4])) {
    bias = tensor_of(v[4]);
    if (!bias || !on_device_of(*bias, *a) || bias->dim() != 2 || bias->size(0) != E || bias->size(1) != N || bias->stride(1) != 1 || !f32_or_bf16(*bias) || wants_grad(*bias) || dual(*bias))
      return none();
  }
  if (!is_none(v[8])) {
    gammas = tensor_of(v[8]);
    if (!gammas || !on_device_of(*gammas, *a) || gammas->dim() != 1 || gammas->size(0) != M || !gammas->is_contiguous() || !f32_or_bf16(*gammas) || wants_grad(*gammas) || dual(*gammas)) return none();
  }
  if (M == 0 || M > kFp8Most || K > kFp8Most || N > kFp8Most || (scatter && (scatter->size(0) == 0 || scatter->size(0) > kFp8Most))) return none();
  // (many rows of lines that begin anywhere are copied first; the kernel for fp32 results takes any)
  if (out != ScalarType::Float && M > E * 256 && ((reinterpret_cast<uintptr_t>(w->data_ptr()) | (uint64_t)w->stride(0) | (uint64_t)w->stride(2)) % 16 || !lines_aligned(*a))) return none();
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*a);
  if (!stream) return none();
  Tensor y = empty({scatter ? scatter->size(0) : M, act.swiglu ? N / 2 : N}, out, *a);
  tk_fp8_gemm_desc d = fp8_desc(*a, *as, {bytes(*w), w->stride(0), w->stride(2), floats(*ws), ws->stride(0), ws->stride(1), ws->stride(2)}, E, M, N, md, y);
  if (bias) d.bias = bias->data_ptr(), d.bias_dtype = dtype_code(bias->scalar_type()), d.bias_stride_e = bias->stride(0);
  if (gather) d.gather_indx = static_cast<int32_t*>(gather->data_ptr());
  if (scatter) d.scatter_indx = static_cast<int32_t*>(scatter->data_ptr()), d.scatter_len = (int32_t)scatter->size(0);
  if (gammas) d.gammas = gammas->data_ptr(), d.gammas_dtype = dtype_code(gammas->scalar_type());
  if (act.swiglu) d.activation = TK_ACT_SWIGLU, d.act_alpha = (float)act.alpha, d.act_limit = (float)act.limit, d.act_has_limit = act.has_limit;
  launch([&] { return B.fp8_gemm(&d, *stream); });
  return THPVariable_Wrap(std::move(y));
}

// ---- the linear layer ------------------------------------------------------------------------------------------------------------------------------------

struct LinearFp8 {
  Tensor x, w;  // [T, K]; [E, K, N] or [K, N], dense along N or (turned) along K
  Fp8Slices md;
  bool turned = false;
  int64_t E, K, N;
  Fp8Rows x8;
  Tensor k_first, n_first, scales, y;  // the weights in 8 bits: lines along K [E, N, K], along N [E, K, N]; scales in the blocks' order in memory
  Fp8Lines forward_lines() const {
    const int64_t r = scales.size(1), c = scales.size(2);
    return {bytes(k_first), N * fp8_pitch(K), fp8_pitch(K), floats(scales), r * c, turned ? 1 : c, turned ? c : 1};
  }
  int32_t forward(void* stream) {
    if (const int32_t rc = x8.make(x, stream)) return rc;
    k_first = fp8_values(E, N, K, x), n_first = fp8_values(E, K, N, x);
    const int64_t R = turned ? N : K, C = turned ? K : N, w_e = w.dim() == 3 ? w.stride(0) : 0;
    scales = empty({E, fp8_blocks(R), fp8_blocks(C)}, ScalarType::Float, x);
    const Tensor &same = turned ? k_first : n_first, &other = turned ? n_first : k_first;
    if (const int32_t rc = B.fp8_downcast(w.data_ptr(), dtype_code(w.scalar_type()), E, R, C, w_e, w.stride(turned ? -1 : -2), kFp8, bytes(same), same.stride(0), same.stride(1),
                                          bytes(other), other.stride(0), other.stride(1), floats(scales), scales.stride(0), scales.stride(1), 1, stream))
      return rc;
    y = empty({x.size(0), N}, x.scalar_type(), x);
    tk_fp8_gemm_desc d = fp8_desc(x8.v, x8.s, forward_lines(), E, x.size(0), N, md, y);
    d.zero_rest = d.pow2_scales = 1;
    return B.fp8_gemm(&d, stream);
  }
};

// A saved tensor of the forward pass, or what a hook on saved tensors gives for it
Tensor fp8_saved(const Tensor& t, at::IntArrayRef sizes, ScalarType type, const Tensor& like) {
  TORCH_CHECK(t.defined() && t.scalar_type() == type && t.sizes() == sizes && t.device() == like.device(), "a tensor saved by the forward pass came back with another shape, type or device: not as the forward pass saved it");
  return type == ScalarType::Float8_e4m3fn && t.stride(-1) == 1 ? t : t.contiguous();
}

struct LinearFp8Node : torch::autograd::Function<LinearFp8Node> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& sizes, const std::optional<Tensor>& offs, const std::optional<Tensor>& schedule,
                        bool turned, int64_t stream) {
    LinearFp8 f;
    f.x = x, f.w = w, f.turned = turned;
    f.E = w.dim() == 3 ? w.size(0) : 1, f.K = w.size(-2), f.N = w.size(-1);
    if (sizes) f.md = {*sizes, *offs, *schedule};
    launch([&] { return f.forward(reinterpret_cast<void*>(stream)); });
    ctx->save_for_backward({f.x8.v, f.x8.s, f.n_first, f.scales, f.md.sizes, f.md.offs, f.md.schedule});
    // (what hooks give back for the scales need not be the quantiser's: the backward pass takes those as any)
    const bool hooked = !at::SavedTensorDefaultHooks::get_tls_state().stack.empty();
    ctx->saved_data["dims"] = std::vector<int64_t>{f.E, f.K, f.N, w.dim(), (int64_t)w.scalar_type(), turned ? 1 : 0, hooked ? 0 : 1};
    return f.y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const auto dims = ctx->saved_data["dims"].toIntVector();
    const int64_t E = dims[0], K = dims[1], N = dims[2], T = grads[0].size(0);
    const bool turned = dims[5] != 0;
    const int32_t pow2 = (int32_t)dims[6];
    const Tensor dy = grads[0].stride(1) == 1 ? grads[0] : grads[0].contiguous();
    const Tensor x8 = fp8_saved(saved[0], {T, K}, ScalarType::Float8_e4m3fn, dy), xs = fp8_saved(saved[1], {T, fp8_blocks(K)}, ScalarType::Float, dy);
    const Tensor wn = fp8_saved(saved[2], {E, K, N}, ScalarType::Float8_e4m3fn, dy);
    const Tensor ws = fp8_saved(saved[3], {E, fp8_blocks(turned ? N : K), fp8_blocks(turned ? K : N)}, ScalarType::Float, dy);
    Fp8Slices md;
    if (saved[4].defined()) {
      md.sizes = fp8_saved(saved[4], {E}, ScalarType::Int, dy);
      TORCH_CHECK(saved[5].defined() && saved[6].defined() && saved[5].scalar_type() == ScalarType::Int && saved[6].scalar_type() == ScalarType::Int && saved[5].dim() == 1 && saved[6].dim() == 2 &&
                      saved[5].size(0) > E && saved[6].size(0) >= 3 && saved[5].device() == dy.device() && saved[6].device() == dy.device(),
                  "the metadata of the forward pass came back with another shape, type or device: not as the forward pass saved it");
      md.offs = saved[5].contiguous(), md.schedule = saved[6].size(1) == 0 || saved[6].stride(1) == 1 ? saved[6] : saved[6].contiguous();
    }
    Tensor dx, dw;
    backward_call(dy, [&](void* stream) -> int32_t {
      if (ctx->needs_input_grad(0)) {
        Fp8Rows d8;
        if (const int32_t rc = d8.make(dy, stream)) return rc;
        dx = empty({T, K}, dy.scalar_type(), dy);
        const int64_t r = ws.size(1), c = ws.size(2);
        tk_fp8_gemm_desc d = fp8_desc(d8.v, d8.s, {bytes(wn), wn.stride(0), wn.stride(1), floats(ws), r * c, turned ? c : 1, turned ? 1 : c}, E, T, K, md, dx);
        d.zero_rest = 1, d.pow2_scales = pow2;
        if (const int32_t rc = B.fp8_gemm(&d, stream)) return rc;
      }
      if (ctx->needs_input_grad(1)) {
        Tensor g = dy;
        if (reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 || g.stride(0) % 8 || g.stride(0) < N) {  // (lines of their own at sixteen-byte boundaries: a copy costs less than the kernel for any)
          g = empty_strided({T, N}, {(N + 7) / 8 * 8, 1}, dy.scalar_type(), dy);
          g.copy_(dy);
        }
        const auto wt = (ScalarType)dims[4];
        dw = dims[3] == 3 ? empty({E, K, N}, wt, dy) : empty({K, N}, wt, dy);
        tk_fp8_wgrad_desc d = {};
        d.x = bytes(x8), d.x_stride_t = x8.stride(0), d.x_scale = floats(xs), d.xs_stride_t = xs.size(1), d.xs_stride_k = 1;
        d.dy = g.data_ptr(), d.dy_dtype = dtype_code(g.scalar_type()), d.dy_stride_t = g.stride(0);
        if (md.sizes.defined()) d.slice_sizes = static_cast<int32_t*>(data(md.sizes)), d.slice_offs = static_cast<int32_t*>(data(md.offs));
        d.n_slices = (int32_t)E, d.T = (int32_t)T, d.K = (int32_t)K, d.N = (int32_t)N;
        d.y = dw.data_ptr(), d.y_dtype = dtype_code(wt), d.y_stride_e = K * N, d.y_stride_k = N;
        d.pow2_scales = pow2;
        const int64_t n = B.fp8_wgrad_workspace(d.T, d.K, d.N, d.n_slices);
        const Tensor ws2 = n > 0 ? empty({n}, ScalarType::Byte, dy) : Tensor();
        d.workspace = data(ws2);
        if (const int32_t rc = B.fp8_wgrad(&d, stream)) return rc;
      }
      return TK_OK;
    });
    return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// (x, w, metadata)
PyObject* run_fp8_linear(PyObject* const* v) {
  const Tensor *x = tensor_of(v[0]), *w = tensor_of(v[1]);
  if (!x || !x->is_cuda() || x->dim() != 2 || x->stride(1) != 1 || x->numel() == 0 || (x->scalar_type() != ScalarType::BFloat16 && x->scalar_type() != ScalarType::Half) || dual(*x)) return none();
  if (!w || !on_device_of(*w, *x) || (w->dim() != 2 && w->dim() != 3) || w->numel() == 0 || !row_dtype(*w) || w->size(-2) != x->size(1) || dual(*w)) return none();
  const bool turned = w->stride(-1) != 1;
  if (turned && w->stride(-2) != 1) return none();
  LinearFp8 f;
  f.E = w->dim() == 3 ? w->size(0) : 1, f.K = w->size(-2), f.N = w->size(-1);
  if (x->size(0) > kFp8Most || f.K > kFp8Most || f.N > kFp8Most || !read_slices(v[2], *x, f.E, &f.md) || dispatcher_heard()) return none();
  auto stream = stream_of(*x);
  if (!stream) return none();
  if (wants_grad(*x) || wants_grad(*w)) {
    if (captured(*stream) && (kept_by_default_stream(*x) || kept_by_default_stream(*w))) return none();
    std::optional<Tensor> sizes, offs, schedule;
    if (f.md.sizes.defined()) sizes = f.md.sizes, offs = f.md.offs, schedule = f.md.schedule;
    return THPVariable_Wrap(LinearFp8Node::apply(*x, *w, sizes, offs, schedule, turned, reinterpret_cast<int64_t>(*stream)));
  }
  f.x = *x, f.w = *w, f.turned = turned;
  launch([&] { return f.forward(*stream); });
  return THPVariable_Wrap(std::move(f.y));
}

// ---- swiglu ----------------------------------------------------------------------------------------------------------------------------------------------

struct SwigluFp8 {
  Tensor h, v, s;
  int32_t forward(const Tensor& a, double alpha, std::optional<double> limit, bool keep, void* stream) {
    const LayerNormRows r(a);  // (rows of dense columns)
    c10::SmallVector<int64_t, 5> sizes(a.sizes());
    sizes.back() /= 2;
    h = empty(sizes, a.scalar_type(), a);
    if (keep) v = fp8_values(r.M, r.C, a), s = empty({r.M, fp8_blocks(r.C)}, ScalarType::Float, a);
    return B.swiglu_fp8(a.data_ptr(), dtype_code(a.scalar_type()), r.M, r.C / 2, r.stride, h.data_ptr(), r.C / 2, keep ? bytes(v) : nullptr, fp8_pitch(r.C), floats(s), fp8_blocks(r.C), 1,
                        (float)alpha, (float)limit.value_or(0.), limit.has_value(), stream);
  }
};

struct SwigluFp8Node : torch::autograd::Function<SwigluFp8Node> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, double alpha, double limit, bool limited, int64_t stream) {
    SwigluFp8 f;
    launch([&] { return f.forward(a, alpha, limited ? std::optional<double>(limit) : std::nullopt, true, reinterpret_cast<void*>(stream)); });
    ctx->save_for_backward({f.v, f.s});
    ctx->saved_data["alpha"] = alpha, ctx->saved_data["limit"] = limit, ctx->saved_data["limited"] = limited;
    ctx->saved_data["sizes"] = a.sizes().vec();
    return f.h;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t C = sizes.back();
    int64_t M = 1;
    for (size_t i = 0; i + 1 < sizes.size(); ++i) M *= sizes[i];
    const Tensor dh = dense_rows(grads[0]) ? grads[0] : grads[0].contiguous();
    const Tensor v = fp8_saved(saved[0], {M, C}, ScalarType::Float8_e4m3fn, dh), s = fp8_saved(saved[1], {M, fp8_blocks(C)}, ScalarType::Float, dh);
    Tensor da;
    backward_call(dh, [&](void* stream) {
      da = empty(sizes, dh.scalar_type(), dh);
      const LayerNormRows r(dh);
      return B.swiglu_fp8_backward(dh.data_ptr(), dtype_code(dh.scalar_type()), M, C / 2, r.stride, bytes(v), v.stride(0), floats(s), s.size(1), 1, da.data_ptr(), C,
                                   (float)ctx->saved_data["alpha"].toDouble(), (float)ctx->saved_data["limit"].toDouble(), ctx->saved_data["limited"].toBool(), stream);
    });
    return once({da, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// (a, alpha, limit)
PyObject* run_fp8_swiglu(PyObject* const* v) {
  const Tensor* a = tensor_of(v[0]);
  const double alpha = PyFloat_AsDouble(v[1]), limit = is_none(v[2]) ? 0. : PyFloat_AsDouble(v[2]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (!a || !a->is_cuda() || a->dim() < 1 || a->numel() == 0 || a->size(-1) % 2 || !row_dtype(*a) || !dense_rows(*a) || dual(*a) || !(limit >= 0.)) return none();
  if (dispatcher_heard()) return none();
  auto stream = stream_of(*a);
  if (!stream) return none();
  const bool limited = !is_none(v[2]);
  if (wants_grad(*a)) {
    if (captured(*stream) && kept_by_default_stream(*a)) return none();
    return THPVariable_Wrap(SwigluFp8Node::apply(*a, alpha, limit, limited, reinterpret_cast<int64_t>(*stream)));
  }
  SwigluFp8 f;
  launch([&] { return f.forward(*a, alpha, limited ? std::optional<double>(limit) : std::nullopt, false, *stream); });
  return THPVariable_Wrap(std::move(f.h));
}

}  // namespace
