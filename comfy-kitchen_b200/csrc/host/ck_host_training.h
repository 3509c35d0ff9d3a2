// The training operators' host half: layer norm and GELU with their autograd nodes, a linear layer's gradients.  A part of
// ck_host.cpp, whose helpers it uses and whose rule it follows: a call that is not plain is refused by None and made in Python.
//
// The nodes are C++ ones (forward, saved tensors, backward without the interpreter): a norm's step through Python functions took
// 180 us of host time, the kernels of 1003 x 769 about 20.

// A plain CUDA tensor on `device`, of any strides, that may belong to an autograd graph; null for anything else.
const Tensor* dense(PyObject* o, int device) {
  if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass) && Py_TYPE(o) != parameter_type) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  static const c10::DispatchKeySet usual = c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                           c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
                                           c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
  return usual.has_all(t.key_set()) && t.is_cuda() && t.get_device() == device ? &t : nullptr;
}

// Row r of a tensor (its last dimension is a row) starts at (r / inner) * outer_stride + (r % inner) * inner_stride elements.
struct Rows {
  Tensor t;  // the tensor, or a copy of it where its rows do not lie so, or not on `align` bytes
  int64_t rows, cols, inner, outer_stride, inner_stride;
};

Rows rows_in_levels(const Tensor& given, int64_t align) {
  Rows r = {given, 0, given.size(-1), 0, 0, 0};
  r.rows = given.numel() / r.cols;
  const int64_t size = given.element_size();
  const auto aligned = [&](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % align == 0; };
  if (!given.is_contiguous()) {
    int64_t sizes[3], strides[3];
    int levels = 0;
    bool fits = (r.cols == 1 || given.stride(-1) == 1) && aligned(given);
    for (int64_t d = 0; fits && d + 1 < given.dim(); ++d) {
      if (given.size(d) == 1) continue;
      if (levels > 0 && strides[levels - 1] == given.size(d) * given.stride(d)) {
        sizes[levels - 1] *= given.size(d);
        strides[levels - 1] = given.stride(d);
      } else {
        fits = levels < 2;
        sizes[levels] = given.size(d);
        strides[levels++] = given.stride(d);
      }
    }
    for (int l = 0; fits && l < levels; ++l) fits = strides[l] * size % align == 0;
    if (fits) {
      r.inner = levels > 0 ? sizes[levels - 1] : 1;
      r.inner_stride = levels > 0 ? strides[levels - 1] : r.cols;
      r.outer_stride = levels > 1 ? strides[0] : 0;
      return r;
    }
    r.t = given.contiguous();
  }
  if (!aligned(r.t)) r.t = r.t.clone(at::MemoryFormat::Contiguous);
  r.inner = r.rows;
  r.inner_stride = r.cols;
  return r;
}

[[noreturn]] void library_error(const char* what) { TORCH_CHECK(false, what, " failed: ", lib.last_error()); }

struct NormParams {
  Tensor weight, bias;  // undefined: none
  int code = 0;
  int64_t groups = 1, weight_stride = 0, bias_stride = 0;
};

// False: the Python wrapper's to refuse, or to copy.
bool norm_params(const Tensor& x, const Tensor* weight, const Tensor* bias, NormParams* p) {
  const Tensor* const some = weight != nullptr ? weight : bias;
  p->code = code_of(x.scalar_type());
  if (some == nullptr) return true;
  if (weight != nullptr && bias != nullptr && (weight->sizes() != bias->sizes() || weight->scalar_type() != bias->scalar_type())) return false;
  const int code = code_of(some->scalar_type());
  if (some->dim() < 1 || some->size(-1) != x.size(-1) || (code != p->code && code != 0)) return false;
  p->code = code;
  if (some->dim() > 1) {
    p->groups = some->size(0);
    if (x.dim() < 2 || x.size(0) != p->groups || some->numel() != p->groups * x.size(-1)) return false;
  }
  const auto take = [&](const Tensor* t, Tensor* to, int64_t* stride) {
    if (t == nullptr) return true;
    if (x.size(-1) > 1 && t->stride(-1) != 1) return false;
    *to = *t;
    *stride = t->dim() > 1 ? t->stride(0) : 0;
    return true;
  };
  return take(weight, &p->weight, &p->weight_stride) && take(bias, &p->bias, &p->bias_stride);  // (they may be one tensor)
}

const void* data_of(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* room_of(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

struct NormResult {
  Tensor y, mean, rstd, codes, scales;
};

bool norm_forward(const Tensor& x, const NormParams& p, double eps, double offset, bool stats, bool copy, const Call& c, NormResult* out) {
  const Rows r = rows_in_levels(x, copy ? 16 : 1);
  out->y = result(x.sizes(), x.scalar_type(), c.device);
  if (stats) {
    out->mean = result({r.rows}, ScalarType::Float, c.device);
    out->rstd = result({r.rows}, ScalarType::Float, c.device);
  }
  if (copy) {
    out->codes = result({r.rows, r.cols}, ScalarType::Float8_e4m3fn, c.device);
    out->scales = result({round_up(r.rows, 128), round_up(r.cols / 32, 4)}, ScalarType::Float8_e8m0fnu, c.device);
  }
  return lib.layer_norm_forward(r.t.const_data_ptr(), code_of(x.scalar_type()), r.rows, r.cols, r.inner, r.outer_stride, r.inner_stride, data_of(p.weight),
                                data_of(p.bias), p.code, p.groups, p.weight_stride, p.bias_stride, static_cast<float>(offset), static_cast<float>(eps),
                                out->y.mutable_data_ptr(), static_cast<float*>(room_of(out->mean)), static_cast<float*>(room_of(out->rstd)),
                                room_of(out->codes), room_of(out->scales), c.stream) == 0;
}

// Gradients of gradients raise when somebody asks for them, as with torch's once_differentiable.
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list asked;
  for (const Tensor& g : grads) {
    if (g.defined()) asked.push_back(g.detach().set_requires_grad(true));
  }
  const auto refuse = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable",
                                                                       static_cast<int64_t>(asked.size()));
  torch::autograd::variable_list marked = (*refuse)(std::move(asked));
  size_t i = 0;
  for (Tensor& g : grads) {
    if (g.defined()) g = marked[i++];
  }
  return grads;
}

// A gradient as it stands in memory: a view whose negation is pending (the imaginary part of a conjugate) or a symbolic zero is laid out.
Tensor materialized(const Tensor& grad) { return grad._is_zerotensor() ? at::zeros(grad.sizes(), grad.options()) : grad.resolve_neg(); }

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                        const NormParams& p, double eps, double offset, bool copy) {
    const Call c;
    NormResult r;
    if (!norm_forward(x, p, eps, offset, true, copy, c, &r)) library_error("layer_norm_forward");
    ctx->save_for_backward(copy ? torch::autograd::variable_list{r.mean, r.rstd, p.weight, r.codes, r.scales}
                                : torch::autograd::variable_list{r.mean, r.rstd, p.weight, x});
    const Tensor& some = p.weight.defined() ? p.weight : p.bias;
    auto& held = ctx->saved_data;
    held["offset"] = offset;
    held["groups"] = p.groups;
    held["code"] = static_cast<int64_t>(p.code);
    held["weight"] = p.weight.defined();
    held["bias"] = p.bias.defined();
    if (some.defined()) held["shape"] = some.sizes().vec();
    return r.y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    torch::autograd::variable_list out(7);
    if (!grads[0].defined()) return out;
    const Tensor grad = materialized(grads[0]);
    const c10::cuda::CUDAGuard on(grad.device());
    const Call c;
    const auto saved = ctx->get_saved_variables();
    const Tensor &mean = saved[0], &rstd = saved[1], &weight = saved[2];
    const bool copy = saved.size() == 5;
    auto& held = ctx->saved_data;
    const bool has_weight = held["weight"].toBool(), has_bias = held["bias"].toBool();
    const int code = static_cast<int>(held["code"].toInt());
    const int64_t groups = held["groups"].toInt();
    const bool want_weight = has_weight && ctx->needs_input_grad(1), want_bias = has_bias && ctx->needs_input_grad(1 + has_weight);
    const Rows dy = rows_in_levels(grad, copy ? 16 : 1);
    const Tensor dx = result(grad.sizes(), grad.scalar_type(), c.device);
    const ScalarType param = code == 0 ? ScalarType::Float : code == 1 ? ScalarType::Half : ScalarType::BFloat16;
    const std::vector<int64_t> shape = has_weight || has_bias ? held["shape"].toIntVector() : std::vector<int64_t>{};
    Tensor dweight, dbias;
    if (want_weight) dweight = result(shape, param, c.device);
    if (want_bias) dbias = result(shape, param, c.device);
    const Rows x = copy ? Rows{} : rows_in_levels(saved[3], 1);
    const int64_t need = want_weight || want_bias ? lib.layer_norm_backward_workspace_bytes(dy.rows, dy.cols, groups) : 0;
    Workspace ws(need);
    if (lib.layer_norm_backward(dy.t.const_data_ptr(), code_of(dx.scalar_type()), dy.rows, dy.cols, dy.inner, dy.outer_stride, dy.inner_stride,
                                copy ? nullptr : x.t.const_data_ptr(), x.inner, x.outer_stride, x.inner_stride, copy ? saved[3].const_data_ptr() : nullptr,
                                copy ? saved[4].const_data_ptr() : nullptr, static_cast<const float*>(mean.const_data_ptr()),
                                static_cast<const float*>(rstd.const_data_ptr()), data_of(weight), code, groups,
                                weight.defined() && weight.dim() > 1 ? weight.stride(0) : 0, static_cast<float>(held["offset"].toDouble()),
                                dx.mutable_data_ptr(), room_of(dweight), room_of(dbias), ws.ptr(), need, c.stream) != 0) {
      library_error("layer_norm_backward");
    }
    if (ctx->needs_input_grad(0)) out[0] = dx;
    out[1] = dweight;
    out[2] = dbias;
    return once(std::move(out));
  }
};

PyObject* layer_norm(PyObject*, Args a, Py_ssize_t n_args) {  // x, weight, bias, eps, weight_offset, checkpoint
  return or_none(a, n_args, 6, [&]() -> PyObject* {
    const Call c;
    const Tensor* x = dense(a[0], c.device);
    const Tensor* weight = a[1] == Py_None ? nullptr : dense(a[1], c.device);
    const Tensor* bias = a[2] == Py_None ? nullptr : dense(a[2], c.device);
    if (x == nullptr || (weight == nullptr && a[1] != Py_None) || (bias == nullptr && a[2] != Py_None) || !PyFloat_Check(a[3]) || !PyFloat_Check(a[4]) ||
        !PyBool_Check(a[5]) || x->dim() < 1 || x->numel() == 0 || code_of(x->scalar_type()) < 0) {
      return nullptr;
    }
    const bool copy = a[5] == Py_True;
    const double eps = PyFloat_AS_DOUBLE(a[3]), offset = PyFloat_AS_DOUBLE(a[4]);
    NormParams p;
    if ((copy && x->size(-1) % 32 != 0) || !norm_params(*x, weight, bias, &p)) return nullptr;
    const bool graph = c10::GradMode::is_enabled() && (x->requires_grad() || (weight != nullptr && weight->requires_grad()) ||
                                                       (bias != nullptr && bias->requires_grad()));
    if (!graph) {
      NormResult r;
      {
        const WithoutGil released;
        if (!norm_forward(*x, p, eps, offset, false, false, c, &r)) return nullptr;
      }
      return THPVariable_Wrap(std::move(r.y));
    }
    const auto maybe = [](const Tensor* t) { return t != nullptr ? std::optional<Tensor>(*t) : std::nullopt; };
    Tensor y;
    {
      const WithoutGil released;
      y = LayerNormNode::apply(*x, maybe(weight), maybe(bias), p, eps, offset, copy);
    }
    return THPVariable_Wrap(std::move(y));
  });
}

Tensor gelu_forward(const Tensor& x, const Call& c, Tensor* codes, Tensor* scales) {  // null: no copy
  const Tensor from = rows_in_levels(x, 32).t.contiguous();
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  Tensor y = result(x.sizes(), x.scalar_type(), c.device);
  if (codes != nullptr) {
    *codes = result({rows, cols}, ScalarType::Float8_e4m3fn, c.device);
    *scales = result({round_up(rows, 128), round_up(cols / 32, 4)}, ScalarType::Float8_e8m0fnu, c.device);
  }
  if (lib.gelu_mxfp8_forward(from.const_data_ptr(), code_of(x.scalar_type()), y.mutable_data_ptr(), codes != nullptr ? codes->mutable_data_ptr() : nullptr,
                             codes != nullptr ? scales->mutable_data_ptr() : nullptr, rows, cols, c.stream) != 0) {
    library_error("gelu_mxfp8_forward");
  }
  return y;
}

struct GeluNode : torch::autograd::Function<GeluNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x) {
    const Call c;
    Tensor codes, scales;
    Tensor y = gelu_forward(x, c, &codes, &scales);
    ctx->save_for_backward({codes, scales});
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    if (!grads[0].defined()) return {Tensor()};
    const c10::cuda::CUDAGuard on(grads[0].device());
    const Call c;
    const auto saved = ctx->get_saved_variables();
    const int64_t cols = grads[0].size(-1);
    Tensor dy = materialized(grads[0]).contiguous();
    if (reinterpret_cast<uintptr_t>(dy.const_data_ptr()) % 32 != 0) dy = dy.clone();
    const Tensor dx = result(dy.sizes(), dy.scalar_type(), c.device);
    if (lib.gelu_mxfp8_backward(dy.const_data_ptr(), code_of(dy.scalar_type()), saved[0].const_data_ptr(), saved[1].const_data_ptr(), dx.mutable_data_ptr(),
                                dy.numel() / cols, cols, c.stream) != 0) {
      library_error("gelu_mxfp8_backward");
    }
    return once({dx});
  }
};

PyObject* gelu_checkpointed(PyObject*, Args a, Py_ssize_t n_args) {  // x
  return or_none(a, n_args, 1, [&]() -> PyObject* {
    const Call c;
    const Tensor* x = dense(a[0], c.device);
    if (x == nullptr || x->dim() < 1 || x->numel() == 0 || x->size(-1) % 32 != 0 || code_of(x->scalar_type()) < 0) return nullptr;
    Tensor y;
    {
      const WithoutGil released;
      y = c10::GradMode::is_enabled() && x->requires_grad() ? GeluNode::apply(*x) : gelu_forward(*x, c, nullptr, nullptr);
    }
    return THPVariable_Wrap(std::move(y));
  });
}

// dy [M, N] of no autograd graph, an MXFP8 matrix [rows, K]; null codes: not plain.
struct GradOperands {
  const Tensor* dy = nullptr;
  const Tensor* codes = nullptr;
  const Tensor* scales = nullptr;
  ScalarType type = ScalarType::Undefined;
  bool fit(Args a, const Call& c, bool rows_are_tokens) {
    dy = matrix(a[0], c.device);
    codes = matrix(a[1], c.device, ScalarType::Float8_e4m3fn);
    scales = matrix(a[2], c.device, ScalarType::Float8_e8m0fnu);
    if (dy == nullptr || codes == nullptr || scales == nullptr || code_of(dy->scalar_type()) < 0) return false;
    type = dy->scalar_type();
    return codes->size(0) == dy->size(rows_are_tokens ? 0 : 1) && codes->size(1) % 32 == 0 && dy->size(1) % 8 == 0 &&
           scales_fit(*scales, codes->size(0), codes->size(1) / 32) && reinterpret_cast<uintptr_t>(dy->const_data_ptr()) % 16 == 0 &&
           dtype_of(a[3], &type);
  }
};

PyObject* linear_weight_grad_mxfp8(PyObject*, Args a, Py_ssize_t n_args) {  // dy, x_codes, x_block_scales, out_dtype, bias_grad
  return or_none(a, n_args, 5, [&]() -> PyObject* {
    const Call c;
    GradOperands g;
    if (!g.fit(a, c, true) || !PyBool_Check(a[4])) return nullptr;
    const bool bias = a[4] == Py_True;
    const int64_t m = g.dy->size(0), n = g.dy->size(1), k = g.codes->size(1);
    const int code = code_of(g.dy->scalar_type());
    const int64_t need = lib.linear_grad_mxfp8_workspace_bytes(1, code, bias, m, n, k);
    if (need <= 0) return nullptr;
    Workspace ws(need);
    Tensor dweight = result({n, k}, g.type, c.device), dbias;
    if (bias) dbias = result({n}, g.type, c.device);
    if (!launched(lib.linear_weight_grad_mxfp8, g.dy->const_data_ptr(), code, g.codes->const_data_ptr(), g.scales->const_data_ptr(),
                  dweight.mutable_data_ptr(), code_of(g.type), room_of(dbias), m, n, k, ws.ptr(), need, c.stream)) {
      return nullptr;
    }
    PyObject* t = PyTuple_New(2);
    if (t == nullptr) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(dweight)));
    if (!bias) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(t, 1, bias ? THPVariable_Wrap(std::move(dbias)) : Py_None);
    return t;
  });
}

PyObject* linear_input_grad_mxfp8(PyObject*, Args a, Py_ssize_t n_args) {  // dy, w_codes, w_block_scales, out_dtype
  return or_none(a, n_args, 4, [&]() -> PyObject* {
    const Call c;
    GradOperands g;
    if (!g.fit(a, c, false)) return nullptr;
    const int64_t m = g.dy->size(0), n = g.dy->size(1), k = g.codes->size(1);
    const int code = code_of(g.dy->scalar_type());
    const int64_t need = lib.linear_grad_mxfp8_workspace_bytes(0, code, 0, m, n, k);
    if (need <= 0) return nullptr;
    Workspace ws(need);
    Tensor dx = result({m, k}, g.type, c.device);
    if (!launched(lib.linear_input_grad_mxfp8, g.dy->const_data_ptr(), code, g.codes->const_data_ptr(), g.scales->const_data_ptr(), dx.mutable_data_ptr(),
                  code_of(g.type), m, n, k, ws.ptr(), need, c.stream)) {
      return nullptr;
    }
    return THPVariable_Wrap(std::move(dx));
  });
}
