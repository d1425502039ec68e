// activations_binding.cpp -- the host side of the 8-bit activation checkpoint
// operators as a torch extension: argument checks, allocation and the autograd
// nodes, around the C-ABI of libsandmuon_b200.so.
//
// A training step calls these operators once or twice per layer and pass, often
// on tensors whose kernels take a few microseconds; with the checks and the
// autograd nodes in Python a call took 10 to 50 microseconds of host time.
// The library is opened by path (bind), so that another build of it can be
// named at run time as for the ctypes binding.
#include <ATen/autocast_mode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <mutex>

#include "sandmuon_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&sm_last_error) last_error = nullptr;
  decltype(&sm_stats_workspace_bytes) stats_workspace_bytes = nullptr;
  decltype(&sm_stats_accumulate) stats_accumulate = nullptr;
  decltype(&sm_activation_sums_workspace_bytes) sums_workspace_bytes = nullptr;
  decltype(&sm_activation_pack) pack = nullptr;
  decltype(&sm_activation_unpack) unpack = nullptr;
  decltype(&sm_gelu_forward) gelu_forward = nullptr;
  decltype(&sm_gelu_backward) gelu_backward = nullptr;
  decltype(&sm_weight_gradient_workspace_bytes) weight_gradient_workspace_bytes = nullptr;
  decltype(&sm_weight_gradient) weight_gradient = nullptr;
};
Api api;

template <typename F>
void resolve(void* lib, const char* name, F& fn) {
  fn = reinterpret_cast<F>(dlsym(lib, name));
  TORCH_CHECK(fn != nullptr, "sandmuon_b200: the library has no ", name);
}

void bind(const std::string& path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib != nullptr, "sandmuon_b200: cannot open ", path, ": ", dlerror());
  resolve(lib, "sm_last_error", api.last_error);
  resolve(lib, "sm_stats_workspace_bytes", api.stats_workspace_bytes);
  resolve(lib, "sm_stats_accumulate", api.stats_accumulate);
  resolve(lib, "sm_activation_sums_workspace_bytes", api.sums_workspace_bytes);
  resolve(lib, "sm_activation_pack", api.pack);
  resolve(lib, "sm_activation_unpack", api.unpack);
  resolve(lib, "sm_gelu_forward", api.gelu_forward);
  resolve(lib, "sm_gelu_backward", api.gelu_backward);
  resolve(lib, "sm_weight_gradient_workspace_bytes", api.weight_gradient_workspace_bytes);
  resolve(lib, "sm_weight_gradient", api.weight_gradient);
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == SM_OK, "sandmuon_b200 ", what, " failed (status ", rc, "): ", api.last_error());
}

bool is_code(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

int code_of(at::ScalarType t, const char* what) {
  TORCH_CHECK_TYPE(is_code(t), what, " must be float32, bfloat16 or float16; got ", t);
  return t == at::kFloat ? SM_DTYPE_F32 : t == at::kBFloat16 ? SM_DTYPE_BF16 : SM_DTYPE_F16;
}

void on_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "sandmuon_b200 runs on CUDA (sm_100) tensors only; got a tensor on ", t.device());
}

// The operators have no rule for forward-mode derivatives; their kernels would
// drop a tangent without a word.
void no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(),
                              "sandmuon_b200.activations has no forward-mode derivatives");
}

// A trace (torch.jit.trace, make_fx) records the torch operators that run: the
// allocation of an output, and not the kernel that fills it.
void no_trace() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !(Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY)),
              "functions of sandmuon_b200.activations cannot be traced");
}

std::string text(const Tensor& t) {
  std::string s = "[";
  for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
  return s + "]";
}

// [..., columns] as [rows, columns] whose memory holds the values (that of a
// negative view, such as the imaginary part of a conjugate, does not).
Tensor flat(const Tensor& given, const char* what) {
  TORCH_CHECK_VALUE(given.dim() > 0, what, " has at least one dimension");
  const Tensor t = given.is_neg() ? given.resolve_neg() : given;
  if (t.dim() == 2) return t;
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  return t.reshape({rows, t.size(-1)});
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

Tensor new_values(const Tensor& like, int64_t rows, int64_t cols) {
  return at::empty({rows, SM_ACTIVATION_LD(cols)}, like.options().dtype(at::kChar));
}
Tensor new_codes(const Tensor& like, int64_t rows, int64_t cols) {
  return at::empty({rows, SM_ACTIVATION_LDE(cols)}, like.options().dtype(at::kByte));
}

// A workspace of one call: captured graphs and streams never share it.
struct Workspace {
  Tensor bytes;
  size_t n;
  Workspace(const Tensor& like, size_t size) : n(size) {
    if (n > 0) bytes = at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
  }
  void* ptr() const { return n > 0 ? bytes.data_ptr() : nullptr; }
};

void* ptr(const optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

// Gradients that are computed while autograd records (a backward pass with
// create_graph, or a call of a backward operator).  Those that depend on
// something with a gradient -- the cotangent, or a tensor of the forward pass --
// are usable, and an error once something differentiates through them; the
// others are constants.
variable_list once(variable_list grads, const std::vector<bool>& depends) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list aliases;
  for (size_t i = 0; i < grads.size(); ++i) {
    if (!grads[i].defined() || !depends[i]) continue;
    Tensor a = grads[i].detach();
    a.set_requires_grad(true);
    aliases.push_back(a);
  }
  if (aliases.empty()) return grads;
  torch::autograd::DelayedError error(
      "trying to differentiate twice a function of sandmuon_b200.activations, which can be differentiated once",
      static_cast<int64_t>(aliases.size()));
  const variable_list marked = error.apply(std::move(aliases));
  size_t next = 0;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined() && depends[i]) grads[i] = marked[next++];
  return grads;
}

using Packed = std::tuple<Tensor, Tensor, optional<Tensor>>;

Packed pack_rows(const Tensor& x, bool stats) {
  const int code = code_of(x.scalar_type(), "an activation");
  on_gpu(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), cols = x.size(1);
  Tensor values = new_values(x, rows, cols), codes = new_codes(x, rows, cols);
  optional<Tensor> sums;
  if (stats) sums = at::empty({2, cols}, x.options().dtype(at::kFloat));
  const Workspace ws(x, stats ? api.sums_workspace_bytes(rows, cols) : 0);
  check(api.pack(x.data_ptr(), code, rows, cols, x.stride(0), x.stride(1), values.data_ptr<int8_t>(),
                 codes.data_ptr<uint8_t>(), static_cast<float*>(ptr(sums)), ws.ptr(), ws.n, stream_of(x)),
        "sm_activation_pack");
  return {values, codes, sums};
}

Packed pack_values(const Tensor& x, bool stats) {
  no_trace();
  return pack_rows(flat(x.detach(), "an activation"), stats);
}

Tensor unpack(const Tensor& values, const Tensor& codes, at::IntArrayRef shape, at::ScalarType dtype) {
  no_trace();
  const int code = code_of(dtype, "the unpacked type");
  on_gpu(values);
  const c10::cuda::CUDAGuard guard(values.device());
  Tensor out = at::empty(shape, values.options().dtype(dtype));
  check(api.unpack(values.data_ptr<int8_t>(), codes.data_ptr<uint8_t>(), values.size(0), shape.back(), out.data_ptr(),
                   code, stream_of(values)),
        "sm_activation_unpack");
  return out;
}

Tensor weight_gradient_rows(const Tensor& delta, const Tensor& values, const Tensor& codes, int64_t d_in,
                            at::ScalarType dtype) {
  const int code = code_of(delta.scalar_type(), "a cotangent");
  const int out_code = code_of(dtype, "a weight gradient");
  on_gpu(delta);
  const c10::cuda::CUDAGuard guard(delta.device());
  const int64_t rows = delta.size(0), d_out = delta.size(1);
  Tensor out = at::empty({d_out, d_in}, delta.options().dtype(dtype));
  const Workspace ws(delta, api.weight_gradient_workspace_bytes(delta.data_ptr(), code, rows, d_out, delta.stride(0),
                                                                delta.stride(1), d_in));
  check(api.weight_gradient(delta.data_ptr(), code, rows, d_out, delta.stride(0), delta.stride(1),
                            values.data_ptr<int8_t>(), codes.data_ptr<uint8_t>(), d_in, out.data_ptr(), out_code,
                            ws.ptr(), ws.n, stream_of(delta)),
        "sm_weight_gradient");
  return out;
}

Tensor weight_gradient(const Tensor& delta, const Tensor& values, const Tensor& codes, int64_t d_in,
                       at::ScalarType dtype) {
  no_trace();
  no_tangent(delta);
  return once({weight_gradient_rows(flat(delta.detach(), "a cotangent"), values, codes, d_in, dtype)},
              {delta.requires_grad()})[0];
}

// [2, columns]: column sums of the squares and of the values, by the statistics
// kernels of the plain layers' hooks.
Tensor column_statistics(const Tensor& rows, const char* what) {
  const int code = rows.scalar_type() == at::kDouble ? SM_DTYPE_F64 : code_of(rows.scalar_type(), what);
  on_gpu(rows);
  const c10::cuda::CUDAGuard guard(rows.device());
  const int64_t n = rows.size(1);
  Tensor both = at::zeros({2, n}, rows.options().dtype(at::kFloat));
  float* sq = both.data_ptr<float>();
  const Workspace ws(rows, api.stats_workspace_bytes(rows.size(0), n));
  check(api.stats_accumulate(rows.data_ptr(), code, rows.size(0), n, rows.stride(0), rows.stride(1), sq, sq + n,
                             ws.ptr(), ws.n, stream_of(rows)),
        "sm_stats_accumulate");
  return both;
}

// delta.float().sum(0)
Tensor column_sums(const Tensor& rows) { return column_statistics(rows, "a cotangent").select(0, 1); }

struct GeluOut {
  Tensor y;
  optional<Tensor> in_values, in_codes, out_values, out_codes, sums;
};

// x: the rows of an activation of the given shape, which y takes.
GeluOut gelu_rows(const Tensor& x, at::IntArrayRef shape, int64_t form, bool keep_input, bool pack_output,
                  bool stats) {
  const int code = code_of(x.scalar_type(), "an activation");
  on_gpu(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), cols = x.size(1);
  GeluOut o;
  o.y = at::empty(shape, x.options());
  if (keep_input) o.in_values = new_values(x, rows, cols), o.in_codes = new_codes(x, rows, cols);
  if (pack_output) o.out_values = new_values(x, rows, cols), o.out_codes = new_codes(x, rows, cols);
  if (stats) o.sums = at::empty({2, cols}, x.options().dtype(at::kFloat));
  const Workspace ws(x, stats ? api.sums_workspace_bytes(rows, cols) : 0);
  check(api.gelu_forward(x.data_ptr(), code, rows, cols, x.stride(0), x.stride(1), static_cast<int>(form),
                         o.y.data_ptr(), static_cast<int8_t*>(ptr(o.in_values)), static_cast<uint8_t*>(ptr(o.in_codes)),
                         static_cast<int8_t*>(ptr(o.out_values)), static_cast<uint8_t*>(ptr(o.out_codes)),
                         static_cast<float*>(ptr(o.sums)), ws.ptr(), ws.n, stream_of(x)),
        "sm_gelu_forward");
  return o;
}

Tensor gelu_backward_rows(const Tensor& delta, const Tensor& values, const Tensor& codes, int64_t form) {
  const int code = code_of(delta.scalar_type(), "a cotangent");
  on_gpu(delta);
  const c10::cuda::CUDAGuard guard(delta.device());
  Tensor dx = at::empty({delta.size(0), delta.size(1)}, delta.options());
  check(api.gelu_backward(delta.data_ptr(), code, delta.size(0), delta.size(1), delta.stride(0), delta.stride(1),
                          values.data_ptr<int8_t>(), codes.data_ptr<uint8_t>(), static_cast<int>(form), dx.data_ptr(),
                          stream_of(delta)),
        "sm_gelu_backward");
  return dx;
}

Tensor as_shape(const Tensor& t, at::IntArrayRef shape) { return t.sizes() == shape ? t : t.view(shape); }

Tensor gelu_backward(const Tensor& delta, const Tensor& values, const Tensor& codes, int64_t form) {
  no_trace();
  no_tangent(delta);
  return once({as_shape(gelu_backward_rows(flat(delta.detach(), "a cotangent"), values, codes, form), delta.sizes())},
              {delta.requires_grad()})[0];
}

// Where 16-bit layers that share a checkpoint send their input gradients: a
// tensor of x's shape in FP32 (one element of memory, never read) whose gradient
// is x's.  Autograd adds what the layers return for it in FP32, and the sum is
// rounded to x's type once, by this node.
struct Widen : torch::autograd::Node {
  const at::ScalarType type;
  explicit Widen(const Tensor& x)
      : torch::autograd::Node({torch::autograd::impl::gradient_edge(x)}), type(x.scalar_type()) {}
  variable_list apply(variable_list&& grads) override {
    return {grads[0].defined() ? grads[0].to(type) : Tensor()};
  }
};

struct Linear : torch::autograd::Function<Linear> {
  // x: the input, or where `data` is given its wide stand-in
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                        const Tensor& values, const Tensor& codes, const optional<Tensor>& data) {
    const Tensor& input = data ? *data : x;
    const at::ScalarType dtype = input.scalar_type();
    const Tensor cast = weight.to(dtype);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({cast, values, codes});
    ctx->saved_data["weight"] = static_cast<int64_t>(weight.scalar_type());
    ctx->saved_data["bias"] = static_cast<int64_t>(bias ? bias->scalar_type() : at::kFloat);
    ctx->saved_data["shape"] = input.sizes();
    ctx->saved_data["x_grad"] = x.requires_grad();
    ctx->saved_data["wide"] = data.has_value();
    optional<Tensor> b;
    if (bias) b = bias->to(dtype);
    // a view would not let in-place operations (an activation, a residual) at it
    const Tensor y = at::linear(input, cast, b);
    return y.is_view() ? at::_unsafe_view(y, y.sizes()) : y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const bool delta_grad = grads[0].requires_grad();
    {
      const at::NoGradGuard no_grad;
      const variable_list saved = ctx->get_saved_variables();
      const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
      const Tensor rows = flat(grads[0], "a cotangent");
      if (ctx->needs_input_grad(0))
        out[0] = as_shape(ctx->saved_data["wide"].toBool() ? at::mm(rows, saved[0], at::kFloat) : at::mm(rows, saved[0]),
                          shape);
      if (ctx->needs_input_grad(1))
        out[1] = weight_gradient_rows(rows, saved[1], saved[2], shape.back(),
                                      static_cast<at::ScalarType>(ctx->saved_data["weight"].toInt()));
      if (ctx->needs_input_grad(2))
        out[2] = column_sums(rows).to(static_cast<at::ScalarType>(ctx->saved_data["bias"].toInt()));
    }
    // delta W (W has a gradient, or this node would not be), delta^T x^, sum delta
    return once(std::move(out),
                {true, delta_grad || ctx->saved_data["x_grad"].toBool(), delta_grad, false, false, false});
  }
};

at::ScalarType compute_type(const Tensor& x) {
  return at::autocast::is_autocast_enabled(at::kCUDA) ? at::autocast::get_autocast_dtype(at::kCUDA) : x.scalar_type();
}

// What the layers that are called with one checkpoint share: the stand-in of the
// x that they are called with, for as long as one of them holds it.
struct Shared {
  std::mutex mutex;
  std::weak_ptr<torch::autograd::Node> node;

  // The node's gradient goes where x's does (x is not, say, a copy of what it
  // was made for), and it runs on this stream: a backward pass that is captured
  // into a graph must not wait on a stream outside of it.
  static bool stands_for(torch::autograd::Node& node, const Tensor& x) {
    const optional<c10::Stream> stream = node.stream();
    return node.next_edge(0) == torch::autograd::impl::gradient_edge(x) && stream &&
           *stream == c10::cuda::getCurrentCUDAStream(x.device().index()).unwrap();
  }

  Tensor wide(const Tensor& x) {
    const Tensor t = at::empty({}, x.options().dtype(at::kFloat)).expand(x.sizes());
    const std::lock_guard<std::mutex> lock(mutex);
    if (const auto known = node.lock(); known && stands_for(*known, x)) {
      torch::autograd::impl::set_gradient_edge(t, {known, 0});
    } else {
      const std::shared_ptr<torch::autograd::Node> made(new Widen(x), torch::autograd::deleteNode);
      torch::autograd::set_history(t, made);
      node = made;
    }
    return t;
  }
};
using SharedRef = std::shared_ptr<Shared>;

// For an x whose layers would send it gradients.
SharedRef shared_by(const Tensor& x) {
  return at::GradMode::is_enabled() && x.requires_grad() ? std::make_shared<Shared>() : nullptr;
}

std::tuple<Packed, SharedRef> pack(const Tensor& x, bool stats) { return {pack_values(x, stats), shared_by(x)}; }

// and whether it is of float16 values.  The sums are always those of x itself:
// where it was rounded to float16 they take a read of their own.
std::tuple<Packed, bool> pack_input_values(const Tensor& x, bool stats) {
  const bool half = compute_type(x) == at::kHalf;
  const bool rounded = half && x.scalar_type() != at::kHalf;
  Packed p = pack_values(rounded ? x.detach().to(at::kHalf) : x, stats && !rounded);
  if (stats && rounded) std::get<2>(p) = column_statistics(flat(x.detach(), "an activation"), "an activation");
  return {std::move(p), half};
}

std::tuple<Packed, bool, SharedRef> pack_input(const Tensor& x, bool stats) {
  auto [p, half] = pack_input_values(x, stats);
  return {std::move(p), half, shared_by(x)};
}

// packed_cols, packed_half, shared: of the given checkpoint (values, codes), if any
Tensor linear(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, const optional<Tensor>& values,
              const optional<Tensor>& codes, int64_t packed_cols, bool packed_half, const SharedRef& shared) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() > 0 && x.size(-1) == weight.size(1), "linear: input ", text(x),
                    " does not fit weight ", text(weight));
  TORCH_CHECK_VALUE(!bias || (bias->dim() == 1 && bias->size(0) == weight.size(0)), "linear: bias ",
                    text(*bias), " does not fit weight ", text(weight));
  on_gpu(x);
  const at::ScalarType dtype = compute_type(x);
  TORCH_CHECK_TYPE(is_code(dtype) && is_code(weight.scalar_type()) && (!bias || is_code(bias->scalar_type())),
                   "linear computes in float32, bfloat16 or float16, with weight and bias of these types; got ", dtype,
                   " and a weight of ", weight.scalar_type());
  if (values) {
    TORCH_CHECK_VALUE(values->device() == x.device(), "input on ", x.device(), ", checkpoint on ", values->device());
    TORCH_CHECK_VALUE(packed_cols == x.size(-1) && values->size(0) * packed_cols == x.numel(),
                      "the checkpoint of a [", values->size(0), ", ", packed_cols,
                      "] activation does not fit an input ", text(x));
    TORCH_CHECK_TYPE(dtype != at::kHalf || packed_half, "a float16 layer needs a checkpoint of float16 values");
  }
  if (!(at::GradMode::is_enabled() && weight.requires_grad())) {
    // nothing reads a checkpoint, and torch's own layer keeps no x
    optional<Tensor> b;
    if (bias) b = bias->to(dtype);
    return at::linear(x.to(dtype), weight.to(dtype), b);
  }
  no_trace();
  no_tangent(x);
  no_tangent(weight);
  if (bias) no_tangent(*bias);
  if (!values) {
    const Packed p = std::get<0>(pack_input_values(x, false));
    return Linear::apply(x.to(dtype), weight, bias, std::get<0>(p), std::get<1>(p), optional<Tensor>());
  }
  if (shared && dtype != at::kFloat && x.requires_grad())
    return Linear::apply(shared->wide(x), weight, bias, *values, *codes, optional<Tensor>(x.detach().to(dtype)));
  return Linear::apply(x.to(dtype), weight, bias, *values, *codes, optional<Tensor>());
}

struct Gelu : torch::autograd::Function<Gelu> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, int64_t form, bool pack_output, bool stats) {
    GeluOut o = gelu_rows(flat(x, "an activation"), x.sizes(), form, true, pack_output, stats);
    // no zeros in place of the gradients that y's checkpoint and sums never have
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({*o.in_values, *o.in_codes});
    ctx->saved_data["form"] = form;
    variable_list out{o.y};
    if (pack_output) {
      variable_list plain{*o.out_values, *o.out_codes};
      if (stats) plain.push_back(*o.sums);
      ctx->mark_non_differentiable(plain);
      out.insert(out.end(), plain.begin(), plain.end());
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    {
      const at::NoGradGuard no_grad;
      const variable_list saved = ctx->get_saved_variables();
      const Tensor dx = gelu_backward_rows(flat(grads[0], "a cotangent"), saved[0], saved[1],
                                           ctx->saved_data["form"].toInt());
      out[0] = as_shape(dx, grads[0].sizes());
    }
    return once(std::move(out), {true, false, false, false});  // x has a gradient, or this node would not be
  }
};

// (y, (values, codes, sums) of y or None)
std::tuple<Tensor, optional<Packed>> gelu(const Tensor& x, int64_t form, bool pack_output, bool stats) {
  TORCH_CHECK_VALUE(x.dim() > 0, "an activation has at least one dimension");
  on_gpu(x);
  no_trace();
  no_tangent(x);
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    const variable_list out = Gelu::apply(x, form, pack_output, stats);
    if (!pack_output) return {out[0], std::nullopt};
    return {out[0], Packed(out[1], out[2], stats ? optional<Tensor>(out[3]) : std::nullopt)};
  }
  GeluOut o = gelu_rows(flat(x.detach(), "an activation"), x.sizes(), form, false, pack_output, stats);
  if (!pack_output) return {o.y, std::nullopt};
  return {o.y, Packed(*o.out_values, *o.out_codes, o.sums)};
}

}  // namespace

// Without Python's lock: an allocation or a launch may wait for the GPU, and
// other threads (the one that a collective waits for among them) run meanwhile.
using Unlocked = pybind11::call_guard<pybind11::gil_scoped_release>;

PYBIND11_MODULE(_activations, m) {
  pybind11::class_<Shared, SharedRef>(m, "Shared");
  m.def("bind", &bind);
  m.def("pack", &pack, Unlocked());
  m.def("pack_input", &pack_input, Unlocked());
  m.def(
      "unpack",
      [](const Tensor& values, const Tensor& codes, const std::vector<int64_t>& shape, at::ScalarType dtype) {
        return unpack(values, codes, shape, dtype);
      },
      Unlocked());
  m.def("weight_gradient", &weight_gradient, Unlocked());
  m.def("linear", &linear, Unlocked());
  m.def("gelu", &gelu, Unlocked());
  m.def("gelu_backward", &gelu_backward, Unlocked());
}
