// The host half of RMS norm (with its autograd node), clipping by the gradients' norm and the products with experts' weights.  A part of
// ck_host.cpp, whose helpers and those of ck_host_training.h it uses and whose rule it follows: a call that is not plain is refused
// by None and made in Python.  (1003 x 769 through Python functions took 170 us of host time forward and backward, 300 gradients 530.)

// A weight [cols] of x's type or fp32, and a residual like x.
bool rms_operands(const Tensor& x, const Tensor* weight, const Tensor* residual, int* code) {
  *code = code_of(x.scalar_type());
  if (weight != nullptr) {
    const int of_weight = code_of(weight->scalar_type());
    if (weight->dim() != 1 || weight->size(0) != x.size(-1) || !weight->is_contiguous() || (of_weight != *code && of_weight != 0)) return false;
    *code = of_weight;
  }
  return residual == nullptr || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type());
}

struct RmsResult {
  Tensor y, h, rstd, codes, scales;
};

bool rms_forward(const Tensor& x, const Tensor& weight, const Tensor& residual, int code, double eps, double offset, bool stats, bool codes, const Call& c,
                 RmsResult* out) {
  const int64_t align = codes ? 32 : 1;
  const Rows r = rows_in_levels(x, align);
  Rows add = {Tensor(), 0, 0, 0, 0, 0};
  if (residual.defined()) add = rows_in_levels(residual, align);
  if (codes) {
    out->codes = result({r.rows, r.cols}, ScalarType::Float8_e4m3fn, c.device);
    out->scales = result({round_up(r.rows, 128), round_up(r.cols / 32, 4)}, ScalarType::Float8_e8m0fnu, c.device);
  } else {
    out->y = result(x.sizes(), x.scalar_type(), c.device);
  }
  if (residual.defined()) out->h = result(x.sizes(), x.scalar_type(), c.device);
  if (stats) out->rstd = result({r.rows}, ScalarType::Float, c.device);
  return lib.rms_norm_forward(r.t.const_data_ptr(), code_of(x.scalar_type()), r.rows, r.cols, r.inner, r.outer_stride, r.inner_stride, data_of(add.t),
                              add.inner, add.outer_stride, add.inner_stride, data_of(weight), code, static_cast<float>(offset), static_cast<float>(eps),
                              room_of(out->y), room_of(out->h), static_cast<float*>(room_of(out->rstd)), room_of(out->codes), room_of(out->scales),
                              c.stream) == 0;
}

struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                                                const std::optional<Tensor>& residual, int64_t code, double eps, double offset) {
    const Call c;
    RmsResult r;
    const Tensor none, &w = weight ? *weight : none, &add = residual ? *residual : none;
    if (!rms_forward(x, w, add, static_cast<int>(code), eps, offset, true, false, c, &r)) library_error("rms_norm_forward");
    ctx->save_for_backward({residual ? r.h : x, r.rstd, w});
    ctx->set_materialize_grads(false);
    auto& held = ctx->saved_data;
    held["offset"] = offset;
    held["code"] = code;
    held["weight"] = weight.has_value();
    held["residual"] = residual.has_value();
    if (residual) return {r.y, r.h};
    return {r.y};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    torch::autograd::variable_list out(6);
    auto& held = ctx->saved_data;
    const bool has_weight = held["weight"].toBool(), has_residual = held["residual"].toBool();
    const bool want_x = ctx->needs_input_grad(0), want_weight = has_weight && ctx->needs_input_grad(1);
    const bool want_residual = has_residual && ctx->needs_input_grad(1 + has_weight);
    const bool of_y = grads[0].defined(), of_h = has_residual && grads[1].defined();
    if (!of_y) {
      if (of_h && want_x) out[0] = grads[1];
      if (of_h && want_residual) out[2] = grads[1];
      return once(std::move(out));
    }
    const Tensor dy = materialized(grads[0]), dh = of_h ? materialized(grads[1]) : Tensor();
    const c10::cuda::CUDAGuard on(dy.device());
    const Call c;
    const auto saved = ctx->get_saved_variables();
    const Rows d = rows_in_levels(dy, 1), h = rows_in_levels(saved[0], 1);
    Rows more = {Tensor(), 0, 0, 0, 0, 0};
    if (of_h) more = rows_in_levels(dh, 1);
    const Tensor& weight = saved[2];
    const int code = static_cast<int>(held["code"].toInt()), type = code_of(dy.scalar_type());
    const Tensor dx = result(dy.sizes(), dy.scalar_type(), c.device);
    Tensor dweight;
    if (want_weight) dweight = result({d.cols}, weight.scalar_type(), c.device);
    const int64_t need = want_weight ? lib.rms_norm_backward_workspace_bytes(type, d.rows, d.cols) : 0;
    Workspace ws(need);
    if (lib.rms_norm_backward(d.t.const_data_ptr(), type, d.rows, d.cols, d.inner, d.outer_stride, d.inner_stride, h.t.const_data_ptr(), h.inner,
                              h.outer_stride, h.inner_stride, data_of(more.t), more.inner, more.outer_stride, more.inner_stride,
                              static_cast<const float*>(saved[1].const_data_ptr()), data_of(weight), code, static_cast<float>(held["offset"].toDouble()),
                              dx.mutable_data_ptr(), room_of(dweight), ws.ptr(), need, c.stream) != 0) {
      library_error("rms_norm_backward");
    }
    if (want_x) out[0] = dx;
    out[1] = dweight;
    if (want_residual) out[2] = dx;
    return once(std::move(out));
  }
};

struct RmsCall {
  const Tensor *x, *weight = nullptr, *residual = nullptr;
  int code = 0;
  double eps = 0, offset = 0;
  bool graph = false;
  bool fit(Args a, const Call& c) {  // x, weight, residual, eps, weight_offset
    x = dense(a[0], c.device);
    weight = a[1] == Py_None ? nullptr : dense(a[1], c.device);
    residual = a[2] == Py_None ? nullptr : dense(a[2], c.device);
    if (x == nullptr || (weight == nullptr && a[1] != Py_None) || (residual == nullptr && a[2] != Py_None) || !PyFloat_Check(a[3]) || !PyFloat_Check(a[4]) ||
        x->dim() < 1 || x->numel() == 0 || code_of(x->scalar_type()) < 0 || !rms_operands(*x, weight, residual, &code)) {
      return false;
    }
    eps = PyFloat_AS_DOUBLE(a[3]);
    offset = PyFloat_AS_DOUBLE(a[4]);
    graph = c10::GradMode::is_enabled() &&
            (x->requires_grad() || (weight != nullptr && weight->requires_grad()) || (residual != nullptr && residual->requires_grad()));
    return true;
  }
};

Tensor or_undefined(const Tensor* t) { return t != nullptr ? *t : Tensor(); }

PyObject* rms_norm(PyObject*, Args a, Py_ssize_t n_args) {  // x, weight, residual, eps, weight_offset
  return or_none(a, n_args, 5, [&]() -> PyObject* {
    const Call c;
    RmsCall k;
    if (!k.fit(a, c)) return nullptr;
    RmsResult r;
    {
      const WithoutGil released;
      if (k.graph) {
        const auto maybe = [](const Tensor* t) { return t != nullptr ? std::optional<Tensor>(*t) : std::nullopt; };
        auto out = RmsNormNode::apply(*k.x, maybe(k.weight), maybe(k.residual), static_cast<int64_t>(k.code), k.eps, k.offset);
        r.y = std::move(out[0]);
        if (k.residual != nullptr) r.h = std::move(out[1]);
      } else if (!rms_forward(*k.x, or_undefined(k.weight), or_undefined(k.residual), k.code, k.eps, k.offset, false, false, c, &r)) {
        return nullptr;
      }
    }
    if (k.residual == nullptr) return THPVariable_Wrap(std::move(r.y));
    return pair(std::move(r.y), std::move(r.h));
  });
}

PyObject* rms_norm_mxfp8(PyObject*, Args a, Py_ssize_t n_args) {  // x, weight, residual, eps, weight_offset
  return or_none(a, n_args, 5, [&]() -> PyObject* {
    const Call c;
    RmsCall k;
    if (!k.fit(a, c) || k.graph || k.x->size(-1) % 32 != 0 ||
        (k.weight != nullptr && reinterpret_cast<uintptr_t>(k.weight->const_data_ptr()) % 16 != 0)) {
      return nullptr;
    }
    RmsResult r;
    {
      const WithoutGil released;
      if (!rms_forward(*k.x, or_undefined(k.weight), or_undefined(k.residual), k.code, k.eps, k.offset, false, true, c, &r)) return nullptr;
    }
    if (k.residual == nullptr) return pair(std::move(r.codes), std::move(r.scales));
    PyObject* t = PyTuple_New(3);
    if (t == nullptr) return nullptr;
    PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(r.codes)));
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(r.scales)));
    PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(r.h)));
    return t;
  });
}

// ---- gradients' norm ---------------------------------------------------------------------------
// The gradients of a list of parameters; max_norm as the C ABI has it.
PyObject* clip_grad_norm(PyObject*, Args a, Py_ssize_t n_args) {  // [parameters], max_norm
  try {
    if (n_args != 2 || !PyList_CheckExact(a[0]) || !PyFloat_Check(a[1]) || !quiet()) Py_RETURN_NONE;
    const Call c;
    const Py_ssize_t n = PyList_GET_SIZE(a[0]);
    std::vector<Tensor> grads;  // held while the GIL is released
    std::vector<void*> data;
    std::vector<int64_t> counts;
    std::vector<int> types;
    grads.reserve(n);
    data.reserve(n);
    counts.reserve(n);
    types.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(a[0], i);
      if (Py_TYPE(o) != reinterpret_cast<PyTypeObject*>(THPVariableClass) && Py_TYPE(o) != parameter_type) Py_RETURN_NONE;
      const Tensor& g = THPVariable_Unpack(o).grad();
      if (!g.defined()) continue;
      static const c10::DispatchKeySet usual = c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
                                               c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) | c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
      if (!usual.has_all(g.key_set()) || !g.is_cuda() || g.get_device() != c.device || !g.is_contiguous() || g.is_inference() || g.requires_grad() ||
          code_of(g.scalar_type()) < 0) {
        Py_RETURN_NONE;
      }
      grads.push_back(g);
      data.push_back(g.mutable_data_ptr());
      counts.push_back(g.numel());
      types.push_back(code_of(g.scalar_type()));
    }
    if (grads.empty()) Py_RETURN_NONE;
    const int64_t count = static_cast<int64_t>(grads.size()), need = lib.clip_grad_norm_workspace_bytes(count);
    Workspace ws(need);
    Tensor norm = result({}, ScalarType::Float, c.device);
    if (!launched(lib.clip_grad_norm, data.data(), counts.data(), types.data(), count, static_cast<float>(PyFloat_AS_DOUBLE(a[1])),
                  static_cast<float*>(norm.mutable_data_ptr()), ws.ptr(), need, c.stream)) {
      Py_RETURN_NONE;
    }
    for (const Tensor& g : grads) g.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(std::move(norm));
  } catch (const std::exception&) {
  }
  Py_RETURN_NONE;
}

// ---- experts -----------------------------------------------------------------------------------
// Weights [E, N, K] with their scales, and the groups' ends.
struct Experts {
  const Tensor *codes = nullptr, *scales = nullptr, *offsets = nullptr;
  int64_t count = 0, n = 0, k = 0;
  bool fit(PyObject* w, PyObject* s, PyObject* ends, const Call& c) {
    codes = plain(w, c.device);
    scales = plain(s, c.device);
    offsets = plain(ends, c.device);
    if (codes == nullptr || scales == nullptr || offsets == nullptr || codes->scalar_type() != ScalarType::Float8_e4m3fn || codes->dim() != 3 ||
        scales->scalar_type() != ScalarType::Float8_e8m0fnu || scales->dim() != 3 || offsets->scalar_type() != ScalarType::Int || offsets->dim() != 1) {
      return false;
    }
    count = codes->size(0);
    n = codes->size(1);
    k = codes->size(2);
    return count > 0 && n > 0 && k > 0 && n % 8 == 0 && k % 32 == 0 && offsets->size(0) == count && scales->size(0) == count &&
           scales->size(1) == round_up(n, 128) && scales->size(2) == round_up(k / 32, 4);
  }
  const int* ends() const { return static_cast<const int*>(offsets->const_data_ptr()); }
  bool bias_of(PyObject* o, const Call& c, Bias* b) const {
    if (o == Py_None) return true;
    const Tensor* t = plain(o, c.device);
    if (t == nullptr || t->dim() != 2 || t->size(0) != count || t->size(1) != n || code_of(t->scalar_type()) < 0) return false;
    b->ptr = t->const_data_ptr();
    b->code = code_of(t->scalar_type());
    return true;
  }
};
bool on_boundary(const Tensor* t, int64_t align) { return reinterpret_cast<uintptr_t>(t->const_data_ptr()) % align == 0; }

PyObject* grouped_mm_mxfp8(PyObject*, Args a, Py_ssize_t n_args) {  // a, b, block_scale_a, block_scale_b, offsets, bias, out_dtype
  return or_none(a, n_args, 7, [&]() -> PyObject* {
    const Call c;
    Experts e;
    Bias bias;
    ScalarType type = ScalarType::BFloat16;
    const Tensor* x = matrix(a[0], c.device, ScalarType::Float8_e4m3fn);
    const Tensor* sx = matrix(a[2], c.device, ScalarType::Float8_e8m0fnu);
    if (x == nullptr || sx == nullptr || !e.fit(a[1], a[3], a[4], c) || x->size(1) != e.k || !scales_fit(*sx, x->size(0), e.k / 32) ||
        !e.bias_of(a[5], c, &bias) || !dtype_of(a[6], &type)) {
      return nullptr;
    }
    const int64_t m = x->size(0), need = lib.grouped_mm_mxfp8_workspace_bytes(0, m, e.k, e.count);
    if (need <= 0) return nullptr;
    Workspace ws(need);
    Tensor out = result({m, e.n}, type, c.device);
    if (!launched(lib.grouped_mm_mxfp8, x->const_data_ptr(), e.codes->const_data_ptr(), sx->const_data_ptr(), e.scales->const_data_ptr(), e.ends(),
                  bias.ptr, bias.code, out.mutable_data_ptr(), code_of(type), m, e.n, e.k, e.count, ws.ptr(), need, c.stream)) {
      return nullptr;
    }
    return THPVariable_Wrap(std::move(out));
  });
}

PyObject* grouped_linear_mxfp8(PyObject*, Args a, Py_ssize_t n_args) {  // x, w_codes, w_block_scales, offsets, bias
  return or_none(a, n_args, 5, [&]() -> PyObject* {
    const Call c;
    Experts e;
    Bias bias;
    const Tensor* x = matrix(a[0], c.device);
    if (x == nullptr || code_of(x->scalar_type()) < 0 || !on_boundary(x, 16) || !e.fit(a[1], a[2], a[3], c) || x->size(1) != e.k || !e.bias_of(a[4], c, &bias)) {
      return nullptr;
    }
    const int64_t m = x->size(0), need = lib.grouped_mm_mxfp8_workspace_bytes(1, m, e.k, e.count);
    if (need <= 0) return nullptr;
    Workspace ws(need);
    const int code = code_of(x->scalar_type());
    Tensor out = result({m, e.n}, x->scalar_type(), c.device);
    if (!launched(lib.grouped_linear_mxfp8, x->const_data_ptr(), code, e.codes->const_data_ptr(), e.scales->const_data_ptr(), e.ends(), bias.ptr, bias.code,
                  out.mutable_data_ptr(), code, m, e.n, e.k, e.count, ws.ptr(), need, c.stream)) {
      return nullptr;
    }
    return THPVariable_Wrap(std::move(out));
  });
}

PyObject* grouped_input_grad_mxfp8(PyObject*, Args a, Py_ssize_t n_args) {  // dy, w_codes, w_block_scales, offsets, out_dtype
  return or_none(a, n_args, 5, [&]() -> PyObject* {
    const Call c;
    Experts e;
    const Tensor* dy = matrix(a[0], c.device);
    if (dy == nullptr || code_of(dy->scalar_type()) < 0 || !on_boundary(dy, 16) || !e.fit(a[1], a[2], a[3], c) || dy->size(1) != e.n ||
        !on_boundary(e.codes, 32)) {
      return nullptr;
    }
    ScalarType type = dy->scalar_type();
    if (!dtype_of(a[4], &type)) return nullptr;
    const int code = code_of(dy->scalar_type());
    const int64_t m = dy->size(0), need = lib.grouped_input_grad_mxfp8_workspace_bytes(code, m, e.n, e.k, e.count);
    if (need <= 0) return nullptr;
    Workspace ws(need);
    Tensor dx = result({m, e.k}, type, c.device);
    if (!launched(lib.grouped_input_grad_mxfp8, dy->const_data_ptr(), code, e.codes->const_data_ptr(), e.scales->const_data_ptr(), e.ends(),
                  dx.mutable_data_ptr(), code_of(type), m, e.n, e.k, e.count, ws.ptr(), need, c.stream)) {
      return nullptr;
    }
    return THPVariable_Wrap(std::move(dx));
  });
}
