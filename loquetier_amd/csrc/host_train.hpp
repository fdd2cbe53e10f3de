// The native host side of the operators around a fine-tuning step (part of host_path.cpp): the residual's addition with its norm, the
// loss over the vocabulary, the update of many tensors.  As there, a call that is not plain goes back to Python untouched.

// What a backward hands out when a graph of it is made (create_graph): tensors that hang on its inputs and refuse to be differentiated.
struct LastGradients : public Function<LastGradients> {
  static variable_list forward(AutogradContext* ctx, at::TensorList gradients, at::TensorList, const std::string& name) {
    ctx->saved_data["name"] = name;
    variable_list out;
    for (const Tensor& t : gradients) out.push_back(t.variable_data());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list) {
    TORCH_CHECK(false, "the gradients of ", ctx->saved_data["name"].toStringRef(), " cannot be differentiated");
  }
};
void last_gradients(std::initializer_list<Tensor*> made, variable_list of, const char* name) {
  if (!at::GradMode::is_enabled()) return;
  variable_list out, from;
  for (Tensor* t : made)
    if (t->defined()) out.push_back(*t);
  for (const Tensor& t : of)
    if (t.defined()) from.push_back(t);
  const variable_list hang = LastGradients::apply(at::TensorList(out), at::TensorList(from), std::string(name));
  size_t n = 0;
  for (Tensor* t : made)
    if (t->defined()) *t = hang[n++];
}

// ---- add_rms_norm ----
struct AddRmsNorm : public Function<AddRmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& w, double eps) {
    Tensor rms = at::empty({x.size(0), 1}, x.options().dtype(at::kFloat)), out = at::empty_like(x), h = at::empty_like(x);
    check(lib.add_rms_fwd(out.data_ptr(), (float*)rms.data_ptr(), h.data_ptr(), x.data_ptr(), residual.data_ptr(), w.data_ptr(),
                          nullptr, nullptr, 0, (int)x.size(0), (int)x.size(1), (float)eps, dtype_code(x), stream(x)),
          "add_rms_norm");
    ctx->save_for_backward({h, w, rms});
    ctx->set_materialize_grads(false);
    return {out, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {grads[1], grads[1], Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const Tensor &h = s[0], &w = s[1], &rms = s[2];
    const Tensor g = grads[0].contiguous(), gh = grads[1].defined() ? grads[1].contiguous() : Tensor();
    check_input(h, "h"), check_input(w, "w"), check_input(rms, "rms"), check_input(g, "grad_output");
    TORCH_CHECK(g.sizes() == h.sizes() && (!gh.defined() || gh.sizes() == h.sizes()), "grad_output and grad_residual must match h");
    TORCH_CHECK(w.dim() == 1 && w.size(0) == h.size(1), "w and dw must have one entry per column of h");
    TORCH_CHECK(rms.scalar_type() == at::kFloat && rms.numel() == h.size(0), "rms must be float32 with one entry per row");
    TORCH_CHECK(half(h) && g.scalar_type() == h.scalar_type() && w.scalar_type() == h.scalar_type() &&
                    (!gh.defined() || gh.scalar_type() == h.scalar_type()), "the gradients, h and w must share one dtype");
    TORCH_CHECK(g.device() == h.device() && w.device() == h.device() && rms.device() == h.device() &&
                    (!gh.defined() || gh.device() == h.device()), "the gradients, h, w and rms must share one device");
    const int rows = (int)h.size(0), cols = (int)h.size(1);
    Tensor dh = at::empty_like(h), dw = at::empty_like(w);
    size_t need = 0;
    check(lib.rms_bwd_size(rows, cols, &need), "smlm_rms_norm_bwd_workspace_size");
    const Tensor mem = bytes(need, h);
    check(lib.add_rms_bwd(dh.data_ptr(), dw.data_ptr(), g.data_ptr(), gh.defined() ? gh.data_ptr() : nullptr, h.data_ptr(), w.data_ptr(),
                          (const float*)rms.data_ptr(), mem.data_ptr(), need, rows, cols, dtype_code(h), stream(h)),
          "add_rms_norm_backward");
    last_gradients({&dh, &dw}, {grads[0], grads[1], h, w}, "add_rms_norm");
    return {dh, dh, dw, Tensor()};
  }
};

bool same(const Tensor& t, const Tensor& like) {
  return t.scalar_type() == like.scalar_type() && t.is_contiguous() && t.sizes() == like.sizes() && t.device() == like.device();
}
bool norm_rows(const Tensor& x, const Tensor& w) {
  return half(x) && x.dim() == 2 && x.is_contiguous() && is(w, x.scalar_type(), 1) && w.size(0) == x.size(1) && x.size(0) > 0 && x.size(0) <= INT32_MAX &&
         x.size(1) > 0 && x.size(1) <= INT32_MAX && x.size(1) % 8 == 0 && x.device() == w.device() && here(x);
}

// add_rms_norm(x, residual, w, eps) -> (output, sum), or None
PyObject* py_add_rms_norm(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  if (n < 3 || n > 4 || !plain_thread() || !plain(p[0]) || !plain(p[1]) || !plain(p[2])) Py_RETURN_NONE;
  const Tensor &x = THPVariable_Unpack(p[0]), &residual = THPVariable_Unpack(p[1]), &w = THPVariable_Unpack(p[2]);
  if (!norm_rows(x, w) || !same(residual, x)) Py_RETURN_NONE;
  double eps = 1e-6;
  if (n == 4) eps = PyFloat_AsDouble(p[3]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_raised();
  variable_list out;
  {
    NoGil no_gil;
    out = AddRmsNorm::apply(x, residual, w, eps);
  }
  THPObjectPtr a0(THPVariable_Wrap(std::move(out[0]))), a1(THPVariable_Wrap(std::move(out[1])));
  if (!a0 || !a1) throw python_raised();
  return PyTuple_Pack(2, a0.get(), a1.get());
  SMLM_PY_END
}

// add_rms(output, rms_output, residual_output, input, residual, weight, epsilon, output8, scale) -> whether it was done
PyObject* py_add_rms(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  if (n != 9 || !plain_thread() || !plain(p[3]) || !plain(p[5])) Py_RETURN_FALSE;
  bool ok = true;
  const Tensor *out = optional(p[0], &ok), *rms = optional(p[1], &ok), *h = optional(p[2], &ok), *residual = optional(p[4], &ok),
               *out8 = optional(p[7], &ok), *scale = optional(p[8], &ok);
  const Tensor &x = THPVariable_Unpack(p[3]), &w = THPVariable_Unpack(p[5]);
  if (!ok || !norm_rows(x, w) || (out && !same(*out, x)) || (h && (!residual || !same(*h, x))) || (residual && !same(*residual, x)) ||
      (!out && !out8 && !h) || !out8 != !scale)
    Py_RETURN_FALSE;
  const int64_t rows = x.size(0), cols = x.size(1);
  if (rms && !(is(*rms, at::kFloat, 2) && rms->size(0) == rows && rms->size(1) == 1 && rms->device() == x.device())) Py_RETURN_FALSE;
  int group = 0;
  if (out8) {
    if (!is(*out8, at::kFloat8_e4m3fn, 2) || out8->sizes() != x.sizes() || out8->device() != x.device() || !is(*scale, at::kFloat, 2) ||
        scale->size(0) != rows || scale->device() != x.device())
      Py_RETURN_FALSE;
    if (scale->size(1) != 1) {
      if (cols % 128 || scale->size(1) != cols / 128) Py_RETURN_FALSE;
      group = 128;
    }
  }
  const double eps = PyFloat_AsDouble(p[6]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_raised();
  int rc;
  {
    void* st = stream(x);
    NoGil no_gil;
    rc = lib.add_rms_fwd(out ? out->data_ptr() : nullptr, rms ? (float*)rms->data_ptr() : nullptr, h ? h->data_ptr() : nullptr, x.data_ptr(),
                         residual ? residual->data_ptr() : nullptr, w.data_ptr(), out8 ? out8->data_ptr() : nullptr,
                         scale ? (float*)scale->data_ptr() : nullptr, group, (int)rows, (int)cols, (float)eps, dtype_code(x), st);
  }
  check(rc, "add_rms_norm");
  Py_RETURN_TRUE;
  SMLM_PY_END
}

// ---- linear_cross_entropy ----
struct LinearCrossEntropy : public Function<LinearCrossEntropy> {
  // for_x: the gradient of x will be wanted, and not that of w
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& labels,
                        const std::optional<Tensor>& partition, bool for_x) {
    const int T = (int)x.size(0), H = (int)x.size(1), V = (int)w.size(0), P = partition ? (int)partition->size(0) - 1 : 0;
    const auto floats = x.options().dtype(at::kFloat).requires_grad(false);
    Tensor loss = at::empty({T}, floats), lse = at::empty({T}, floats), means, weight;
    if (partition) means = at::empty({P}, floats), weight = at::empty({P}, floats);
    size_t need = 0, keep = 0;
    Tensor kept;
    if (for_x) {
      check(lib.loss_size(T, H, V, 5, &keep), "smlm_vocab_loss_workspace_size");
      kept = bytes(keep, x);
    }
    check(lib.loss_size(T, H, V, keep ? 4 : 0, &need), "smlm_vocab_loss_workspace_size");
    const Tensor mem = bytes(need, x);
    check(lib.loss_fwd((float*)loss.data_ptr(), (float*)lse.data_ptr(), P ? (float*)means.data_ptr() : nullptr,
                       P ? (float*)weight.data_ptr() : nullptr, keep ? kept.data_ptr() : nullptr, keep, x.data_ptr(), w.data_ptr(), (const int64_t*)labels.data_ptr(),
                       partition ? (const int32_t*)partition->data_ptr() : nullptr, P, mem.data_ptr(), need, T, H, V, dtype_code(x), stream(x)),
          "linear_cross_entropy");
    ctx->save_for_backward({x, w, labels, loss, lse, partition ? *partition : Tensor(), weight, kept});
    ctx->saved_data["partitioned"] = (bool)partition;
    return partition ? means : loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), parted = ctx->saved_data["partitioned"].toBool();
    if (!want_x && !want_w) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &labels = s[2], &loss = s[3], &lse = s[4], &partition = s[5], &weight = s[6],
                 &kept = s[7];
    const Tensor g = grads[0].contiguous();
    check_input(x, "x"), check_input(w, "w"), check_input(labels, "labels"), check_input(lse, "lse"), check_input(loss, "loss");
    TORCH_CHECK(x.dim() == 2 && half(x) && w.dim() == 2 && w.scalar_type() == x.scalar_type() && w.size(1) == x.size(1) &&
                    x.device() == g.device() && w.device() == g.device(), "x and w must come back as they were saved");
    const int T = (int)x.size(0), H = (int)x.size(1), V = (int)w.size(0);
    TORCH_CHECK(is(labels, at::kLong, 1) && labels.size(0) == T && labels.device() == g.device() && is(lse, at::kFloat, 1) &&
                    lse.size(0) == T && lse.device() == g.device() && is(loss, at::kFloat, 1) && loss.size(0) == T &&
                    loss.device() == g.device(), "labels, loss and lse must come back as they were saved");
    TORCH_CHECK(partition.defined() == parted && weight.defined() == parted, "the partition must come back as it was saved");
    const int P = parted ? (int)partition.numel() - 1 : 0;
    if (parted)
      TORCH_CHECK(is(partition, at::kInt, 1) && is(weight, at::kFloat, 1) && weight.size(0) == P && partition.device() == g.device() &&
                      weight.device() == g.device(), "the partition must come back as it was saved");
    TORCH_CHECK(is(g, at::kFloat, 1) && g.size(0) == (parted ? P : T), "grad must have one entry for each loss");
    Tensor dx = want_x ? at::empty_like(x) : Tensor(), dw = want_w ? at::empty_like(w) : Tensor();
    if (P == 0 && parted) {
      if (want_x) dx.zero_();
      if (want_w) dw.zero_();
    } else if (kept.defined() && !want_w) {
      size_t need = 0;
      check(lib.loss_size(T, H, V, 5, &need), "smlm_vocab_loss_workspace_size");
      TORCH_CHECK(is(kept, at::kByte, 1) && (size_t)kept.numel() >= need && kept.device() == g.device(), "kept must come back as it was saved");
      check(lib.loss_bwd_kept(dx.data_ptr(), (const float*)g.data_ptr(), kept.data_ptr(), (size_t)kept.numel(), w.data_ptr(),
                              parted ? (const int32_t*)partition.data_ptr() : nullptr, parted ? (const float*)weight.data_ptr() : nullptr, P,
                              T, H, V, dtype_code(x), stream(x)),
            "linear_cross_entropy_backward");
    } else {
      size_t need = 0;
      check(lib.loss_size(T, H, V, (int)want_x + 2 * (int)want_w, &need), "smlm_vocab_loss_workspace_size");
      const Tensor mem = bytes(need, x);
      check(lib.loss_bwd(want_x ? dx.data_ptr() : nullptr, want_w ? dw.data_ptr() : nullptr, (const float*)g.data_ptr(),
                         (const float*)loss.data_ptr(), (const float*)lse.data_ptr(), x.data_ptr(), w.data_ptr(), (const int64_t*)labels.data_ptr(),
                         parted ? (const int32_t*)partition.data_ptr() : nullptr, parted ? (const float*)weight.data_ptr() : nullptr, P,
                         mem.data_ptr(), need, T, H, V, dtype_code(x), stream(x)),
            "linear_cross_entropy_backward");
    }
    last_gradients({&dx, &dw}, {grads[0], x, w}, "linear_cross_entropy");
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};

// linear_cross_entropy(x, w, labels, partition) -> losses, or None
PyObject* py_linear_cross_entropy(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  if (n < 3 || n > 4 || !plain_thread() || !plain(p[0]) || !plain(p[1]) || !plain(p[2])) Py_RETURN_NONE;
  bool ok = true;
  const Tensor* partition = n == 4 ? optional(p[3], &ok) : nullptr;
  const Tensor &x = THPVariable_Unpack(p[0]), &w = THPVariable_Unpack(p[1]), &labels = THPVariable_Unpack(p[2]);
  if (!ok || !half(x) || !is(x, x.scalar_type(), 2) || !is(w, x.scalar_type(), 2) || w.size(1) != x.size(1) || x.size(0) == 0 ||
      x.size(1) == 0 || x.size(1) % 8 != 0 || w.size(0) == 0 || !is(labels, at::kLong, 1) || labels.size(0) != x.size(0) ||
      x.size(0) > INT32_MAX || w.size(0) > INT32_MAX || x.size(1) > INT32_MAX || x.device() != w.device() ||
      x.device() != labels.device() || !here(x))
    Py_RETURN_NONE;
  if (partition && (!is(*partition, at::kInt, 1) || partition->size(0) < 1 || partition->device() != x.device())) Py_RETURN_NONE;
  Tensor o;
  {
    NoGil no_gil;
    const bool for_x = at::GradMode::is_enabled() && x.requires_grad() && !w.requires_grad();
    o = LinearCrossEntropy::apply(x, w, labels, partition ? std::optional<Tensor>(*partition) : std::nullopt, for_x);
  }
  return THPVariable_Wrap(std::move(o));
  SMLM_PY_END
}

// ---- adamw_step ----
// adamw_step(params, grads, exp_avg, exp_avg_sq, step, hyper, group, avg_scale, sq_scale, master, workspace) -> whether it was done
PyObject* py_adamw_step(PyObject*, PyObject* const* p, Py_ssize_t nargs) {
  SMLM_PY_TRY
  if (nargs != 11 || !plain_thread() || !PyList_CheckExact(p[0]) || !PyList_CheckExact(p[1])) Py_RETURN_FALSE;
  for (int i = 2; i < 7; ++i)
    if (!plain(p[i])) Py_RETURN_FALSE;
  bool ok = true;
  const Tensor *ms = optional(p[7], &ok), *vs = optional(p[8], &ok), *master = optional(p[9], &ok);
  const Tensor &m = THPVariable_Unpack(p[2]), &v = THPVariable_Unpack(p[3]), &step = THPVariable_Unpack(p[4]),
               &hyper = THPVariable_Unpack(p[5]), &group = THPVariable_Unpack(p[6]);
  const Py_ssize_t n = PyList_GET_SIZE(p[0]);
  const bool eight = m.scalar_type() == at::kFloat8_e4m3fn;
  const auto state = eight ? at::kFloat8_e4m3fn : at::kFloat;
  auto on = [&](const Tensor* t) { return !t || t->device() == m.device(); };
  if (!ok || n == 0 || n > INT32_MAX || PyList_GET_SIZE(p[1]) != n || !is(m, state, 1) || !is(v, state, 1) || !is(step, at::kInt, 1) ||
      !is(group, at::kInt, 1) || !is(hyper, at::kFloat, 2) || hyper.size(1) != 5 || step.size(0) != n || group.size(0) != n || !here(m) ||
      !on(&v) || !on(&step) || !on(&group) || !on(&hyper) || !on(ms) || !on(vs) || !on(master) || eight != (ms != nullptr) ||
      eight != (vs != nullptr) || (ms && !is(*ms, at::kFloat, 1)) || (vs && !is(*vs, at::kFloat, 1)) ||
      (master && !is(*master, at::kFloat, 1)))
    Py_RETURN_FALSE;
  std::vector<void*> where(n), full;
  std::vector<std::pair<uintptr_t, uintptr_t>> written;  // from, to
  std::vector<const void*> at_(n, nullptr);
  std::vector<int64_t> sizes(n);
  full.reserve(n), written.reserve(n);
  int64_t blocks = 0;
  at::ScalarType type{};
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *po = PyList_GET_ITEM(p[0], i), *go = PyList_GET_ITEM(p[1], i);
    if (!(THPVariable_CheckExact(po) || THPVariable_Check(po))) Py_RETURN_FALSE;  // (a Parameter is a tensor too)
    const Tensor& t = THPVariable_Unpack(po);
    if (i == 0) type = t.scalar_type();
    if (!t.defined() || t.scalar_type() != type || t.device() != m.device() || t.layout() != at::kStrided || !t.is_contiguous()) Py_RETURN_FALSE;
    if (t.key_set().has(c10::DispatchKey::Python)) Py_RETURN_FALSE;
    if (go != Py_None) {
      if (!plain(go)) Py_RETURN_FALSE;
      const Tensor& g = THPVariable_Unpack(go);
      if (g.scalar_type() != type || g.device() != m.device() || !g.is_contiguous() || g.sizes() != t.sizes()) Py_RETURN_FALSE;
      at_[i] = g.data_ptr();
    }
    where[i] = t.data_ptr(), sizes[i] = t.numel();
    if (sizes[i]) full.push_back(where[i]);
    if (sizes[i] && at_[i]) written.emplace_back((uintptr_t)where[i], (uintptr_t)where[i] + t.nbytes());
    blocks += (sizes[i] + 255) / 256;
  }
  const bool f32 = type == at::kFloat;
  if (!(f32 || type == at::kHalf || type == at::kBFloat16) || (f32 && master)) Py_RETURN_FALSE;
  if (m.size(0) != blocks * 256 || v.size(0) != blocks * 256 || (master && master->size(0) != blocks * 256) ||
      (ms && (ms->size(0) != blocks || vs->size(0) != blocks)))
    Py_RETURN_FALSE;
  std::sort(full.begin(), full.end());
  if (std::adjacent_find(full.begin(), full.end()) != full.end()) Py_RETURN_FALSE;
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i - 1].second > written[i].first) Py_RETURN_FALSE;
  size_t need = 0;
  check(lib.adamw_size((int)n, &need), "smlm_adamw_workspace_size");
  const Tensor mem = scratch(p[10], need, m);
  smlm_adamw a{};
  a.params = where.data(), a.grads = at_.data(), a.sizes = sizes.data(), a.step = (int32_t*)step.data_ptr();
  a.group = (const int32_t*)group.data_ptr(), a.hyper = (const float*)hyper.data_ptr(), a.exp_avg = m.data_ptr();
  a.exp_avg_sq = v.data_ptr(), a.avg_scale = ms ? (float*)ms->data_ptr() : nullptr, a.sq_scale = vs ? (float*)vs->data_ptr() : nullptr;
  a.master = master ? (float*)master->data_ptr() : nullptr, a.n_tensors = (int)n, a.n_groups = (int)hyper.size(0);
  a.state_bits = eight ? 8 : 32, a.dtype = f32 ? 2 : type == at::kHalf ? SMLM_DTYPE_F16 : SMLM_DTYPE_BF16;
  int rc;
  {
    void* st = stream(m);
    NoGil no_gil;
    rc = lib.adamw(&a, mem.data_ptr(), (size_t)mem.numel(), st);
  }
  check(rc, "adamw_step");
  for (Py_ssize_t i = 0; i < n; ++i)  // (autograd then knows that saved weights are no longer what they were)
    if (at_[i]) torch::autograd::impl::bump_version(THPVariable_Unpack(PyList_GET_ITEM(p[0], i)));
  Py_RETURN_TRUE;
  SMLM_PY_END
}
