// The host side of the operators between the projections (ops._kernels: qk_norm_rope, AttentionPlan, paged_attention, kv_extend,
// kv_free, kv_fork), included by host_path.cpp into its namespace.  The same rules: a call in its plain form is done, any other
// is handed back, nothing done, and the Python function of the name checks it and raises.
// us a call, host bound, in Python / so: rotation into a cache of 256 rows 24.6 / 6.9, plan and attention of two rows 24.7 / 10,
// forward and backward through autograd of 1021 rows 188 / 84 (36 of which are autograd's own hand-over), extend and free 35 / 18.

// [rows, heads, head_dim] as the kernels read it
bool heads(const Tensor& t, const Tensor& like) {
  if (t.dim() != 3 || t.scalar_type() != like.scalar_type() || t.device() != like.device()) return false;
  return (t.size(2) == 1 || t.stride(2) == 1) && (t.size(0) < 2 || t.stride(0) % 8 == 0) && (t.size(1) < 2 || t.stride(1) % 8 == 0) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
bool written(const Tensor& t) {  // (an expanded tensor's elements share their places)
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return false;
  return true;
}
smlm_heads view(const Tensor& t) {
  return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
}
bool weight(const Tensor* w, const Tensor& q) {
  return !w || (is(*w, q.scalar_type(), 1) && w->size(0) == q.size(2) && w->device() == q.device());
}
bool on(const Tensor& t, const Tensor& like, at::ScalarType type, int64_t dim) { return is(t, type, dim) && t.device() == like.device(); }

// what the forward and the backward have in common; false: not plain
bool rope_args(const Tensor& q, const Tensor& k, const Tensor* qw, const Tensor* kw, const Tensor& table, const Tensor& pos, double eps,
               smlm_qk_rope* a) {
  if (!half(q) || !here(q) || q.dim() != 3 || k.dim() != 3 || q.size(0) == 0 || q.size(1) == 0 || k.size(1) == 0 ||
      q.size(2) == 0 || q.size(2) % 16 != 0 || q.size(2) > 512 || k.size(0) != q.size(0) || k.size(2) != q.size(2) || !heads(q, q) ||
      !heads(k, q) || !weight(qw, q) || !weight(kw, q) || !on(table, q, at::kFloat, 2) || !on(pos, q, at::kInt, 1) ||
      pos.size(0) != q.size(0) || table.size(1) % 16 != 0 || table.size(1) == 0 || table.size(1) > q.size(2))
    return false;
  a->q = view(q), a->k = view(k);
  a->q_weight = qw ? qw->data_ptr() : nullptr;
  a->k_weight = kw ? kw->data_ptr() : nullptr;
  a->table = (const float*)table.data_ptr();
  a->positions = (const int32_t*)pos.data_ptr();
  a->rows = (int)q.size(0), a->q_heads = (int)q.size(1), a->kv_heads = (int)k.size(1), a->head_dim = (int)q.size(2);
  a->rot_dim = (int)table.size(1), a->table_rows = (int)table.size(0);
  a->dtype = dtype_code(q), a->eps = (float)eps;
  return true;
}
bool caches(const Tensor& k, const Tensor& v, const Tensor& q, int64_t kv_heads) {
  if (k.dim() != 4 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || k.device() != q.device() ||
      v.device() != q.device() || k.size(0) == 0 || k.size(1) != kv_heads || k.size(2) == 0 || k.size(3) != q.size(2) ||
      k.sizes() != v.sizes() || k.strides() != v.strides() || k.stride(3) != 1)
    return false;
  for (int i = 0; i < 3; ++i)
    if (k.size(i) > 1 && k.stride(i) % 8 != 0) return false;
  return true;
}
int64_t stride_of(const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; }

// Gradients that hang on `of` in a graph that is being made of a backward: to differentiate them is refused, as there is no kernel for it.
struct QkGradients : public Function<QkGradients> {
  static variable_list forward(AutogradContext*, at::TensorList gradients, at::TensorList of) {
    (void)of;
    variable_list out;
    for (const Tensor& t : gradients) out.push_back(t.variable_data());
    return out;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "the gradients of qk_norm_rope cannot be differentiated");
  }
};

struct QkNormRope : public Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const std::optional<Tensor>& q_weight,
                               const std::optional<Tensor>& k_weight, const Tensor& table, const Tensor& pos, double eps) {
    const Tensor qw = q_weight ? *q_weight : Tensor(), kw = k_weight ? *k_weight : Tensor();
    Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    smlm_qk_rope a{};
    TORCH_CHECK(rope_args(q, k, qw.defined() ? &qw : nullptr, kw.defined() ? &kw : nullptr, table, pos, eps, &a), "qk_norm_rope");
    a.q_out = view(qo), a.k_out = view(ko);
    check(lib.rope_fwd(&a, stream(q)), "qk_norm_rope");
    ctx->save_for_backward({qw.defined() ? q : Tensor(), kw.defined() ? k : Tensor(), qw, kw, table, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["norms"] = (int64_t)(qw.defined() ? 1 : 0) + (kw.defined() ? 2 : 0);
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const int64_t norms = ctx->saved_data["norms"].toInt();
    Tensor g[2], d[2], dw[2];
    for (int i = 0; i < 2; ++i) {
      const Tensor& t = grads[i];
      const bool fits = (t.size(2) == 1 || t.stride(2) == 1) && (t.size(0) < 2 || t.stride(0) % 8 == 0) &&
                        (t.size(1) < 2 || t.stride(1) % 8 == 0) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
      g[i] = fits ? t : t.clone(at::MemoryFormat::Contiguous);
      d[i] = at::empty(t.sizes(), t.options());
      TORCH_CHECK(s[2 + i].defined() == (norms >> i & 1) && s[i].defined() == s[2 + i].defined(), "the weights must come back as they were saved");
      if (!s[i].defined()) continue;
      TORCH_CHECK(s[i].sizes() == t.sizes() && s[i].scalar_type() == t.scalar_type(), i ? "k" : "q", " must come back as it was saved");
      dw[i] = at::empty_like(s[2 + i]);
    }
    smlm_qk_rope a{};
    TORCH_CHECK(rope_args(s[0].defined() ? s[0] : g[0], s[1].defined() ? s[1] : g[1], s[2].defined() ? &s[2] : nullptr,
                          s[3].defined() ? &s[3] : nullptr, s[4], s[5], ctx->saved_data["eps"].toDouble(), &a),
                "q, k, the weights, table and positions must come back as they were saved");
    Tensor mem;
    size_t need = 0;
    if (norms) {
      check(lib.rope_bwd_size(a.rows, a.q_heads, a.kv_heads, a.head_dim, &need), "smlm_qk_norm_rope_bwd_workspace_size");
      mem = bytes(need, g[0]);
    }
    const smlm_heads gq = view(g[0]), gk = view(g[1]), dq = view(d[0]), dk = view(d[1]);
    check(lib.rope_bwd(&a, &gq, &gk, &dq, &dk, dw[0].defined() ? dw[0].data_ptr() : nullptr,
                       dw[1].defined() ? dw[1].data_ptr() : nullptr, need ? mem.data_ptr() : nullptr, need, stream(g[0])),
          "qk_norm_rope_backward");
    if (at::GradMode::is_enabled()) {
      variable_list made, of;
      for (const Tensor& t : {d[0], d[1], dw[0], dw[1]})
        if (t.defined()) made.push_back(t);
      for (const Tensor& t : {grads[0], grads[1], s[0], s[1], s[2], s[3]})
        if (t.defined()) of.push_back(t);
      const variable_list out = QkGradients::apply(at::TensorList(made), at::TensorList(of));
      d[0] = out[0], d[1] = out[1];
      size_t n = 2;
      for (Tensor& t : dw)
        if (t.defined()) t = out[n++];
    }
    return {d[0], d[1], dw[0], dw[1], Tensor(), Tensor(), Tensor()};
  }
};

// qk_norm_rope(q, k, q_weight, k_weight, table, positions, eps) -> (q_out, k_out), or None
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  if (n < 6 || n > 7 || !plain_thread() || !plain(p[0]) || !plain(p[1]) || !plain(p[4]) || !plain(p[5])) Py_RETURN_NONE;
  bool ok = true;
  const Tensor *qw = optional(p[2], &ok), *kw = optional(p[3], &ok);
  double eps = 1e-6;
  if (n == 7) eps = PyFloat_AsDouble(p[6]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_raised();
  smlm_qk_rope a{};
  const Tensor &q = THPVariable_Unpack(p[0]), &k = THPVariable_Unpack(p[1]), &table = THPVariable_Unpack(p[4]),
               &pos = THPVariable_Unpack(p[5]);
  if (!ok || !rope_args(q, k, qw, kw, table, pos, eps, &a)) Py_RETURN_NONE;
  variable_list out;
  {
    NoGil no_gil;
    out = QkNormRope::apply(q, k, qw ? std::optional<Tensor>(*qw) : std::nullopt, kw ? std::optional<Tensor>(*kw) : std::nullopt, table,
                            pos, eps);
  }
  THPObjectPtr a0(THPVariable_Wrap(std::move(out[0]))), a1(THPVariable_Wrap(std::move(out[1])));
  if (!a0 || !a1) throw python_raised();
  return PyTuple_Pack(2, a0.get(), a1.get());
  SMLM_PY_END
}

// rope(q_out, k_out, q, k, table, positions, q_weight, k_weight, eps, v, k_cache, v_cache, slots) -> whether it was done
PyObject* py_rope(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  TORCH_CHECK(n == 13, "rope takes 13 arguments");
  if (!plain_thread() || !plain(p[0]) || !plain(p[2]) || !plain(p[3]) || !plain(p[4]) || !plain(p[5])) Py_RETURN_FALSE;
  bool ok = true;
  const Tensor *ko = optional(p[1], &ok), *qw = optional(p[6], &ok), *kw = optional(p[7], &ok), *v = optional(p[9], &ok),
               *kc = optional(p[10], &ok), *vc = optional(p[11], &ok), *slots = optional(p[12], &ok);
  const double eps = PyFloat_AsDouble(p[8]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_raised();
  const Tensor &qo = THPVariable_Unpack(p[0]), &q = THPVariable_Unpack(p[2]), &k = THPVariable_Unpack(p[3]);
  smlm_qk_rope a{};
  if (!ok || !rope_args(q, k, qw, kw, THPVariable_Unpack(p[4]), THPVariable_Unpack(p[5]), eps, &a) || !heads(qo, q) ||
      !written(qo) || qo.sizes() != q.sizes() || (ko && (!heads(*ko, q) || !written(*ko) || ko->sizes() != k.sizes())))
    Py_RETURN_FALSE;
  a.q_out = view(qo);
  if (ko) a.k_out = view(*ko);
  if (kc) {
    if (!vc || !v || !slots || !caches(*kc, *vc, q, k.size(1)) || !written(*kc) || !heads(*v, q) || v->sizes() != k.sizes() ||
        !on(*slots, q, at::kLong, 1) || slots->size(0) != q.size(0))
      Py_RETURN_FALSE;
    a.v = view(*v);
    a.k_cache = kc->data_ptr(), a.v_cache = vc->data_ptr();
    a.slots = (const int64_t*)slots->data_ptr();
    a.page_stride = stride_of(*kc, 0), a.head_stride = stride_of(*kc, 1), a.slot_stride = stride_of(*kc, 2);
    a.n_pages = (int)kc->size(0), a.page_size = (int)kc->size(2);
  } else if (vc || v || slots || !ko) {
    Py_RETURN_FALSE;
  }
  check(lib.rope_fwd(&a, stream(q)), "qk_norm_rope");
  Py_RETURN_TRUE;
  SMLM_PY_END
}

// attention_plan(q_indptr, kv_len, page_table, n_rows, q_heads, kv_heads, page_size, requests) -> the plan's buffer, or None
PyObject* py_attention_plan(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  TORCH_CHECK(n == 8, "attention_plan takes 8 arguments");
  bool ok = plain_thread() && plain(p[0]) && plain(p[1]) && plain(p[2]);
  const Tensor* req = optional(p[7], &ok);
  for (int i = 3; i < 7; ++i) ok = ok && PyLong_CheckExact(p[i]);
  if (!ok) Py_RETURN_NONE;
  const Tensor &indptr = THPVariable_Unpack(p[0]), &len = THPVariable_Unpack(p[1]), &table = THPVariable_Unpack(p[2]);
  const int64_t T = integer(p[3]), Hq = integer(p[4]), Hkv = integer(p[5]), P = integer(p[6]);
  const int64_t S = indptr.dim() == 1 ? indptr.size(0) - 1 : -1;
  if (S < 1 || !here(indptr) || !is(indptr, at::kInt, 1) || !on(len, indptr, at::kInt, 1) || !on(table, indptr, at::kInt, 2) ||
      len.size(0) != S || (req && (!on(*req, indptr, at::kInt, 1) || req->size(0) != S)) || (!req && table.size(0) < S) || Hq < 1 ||
      Hkv < 1 || Hq % Hkv != 0 || T < 0 || P < 1 || T > 0x7fffffff || Hq > 0x7fffffff || P > 0x7fffffff)
    Py_RETURN_NONE;
  size_t need = 0;
  check(lib.attn_plan_size((int)T, (int)S, (int)Hq, (int)Hkv, &need), "smlm_attn_plan_size");
  Tensor buf = bytes(need, indptr);
  check(lib.attn_plan(buf.data_ptr(), need, (const int32_t*)indptr.data_ptr(), (const int32_t*)len.data_ptr(),
                      req ? (const int32_t*)req->data_ptr() : nullptr, (int)T, (int)S, (int)table.size(0), (int)table.size(1), (int)P,
                      (int)Hq, (int)Hkv, stream(indptr)),
        "AttentionPlan");
  return THPVariable_Wrap(std::move(buf));
  SMLM_PY_END
}

// paged_attention(out, q, k_cache, v_cache, plan, scale, workspace) -> whether it was done
PyObject* py_paged_attention(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  TORCH_CHECK(n == 7, "paged_attention takes 7 arguments");
  for (int i = 0; i < 4; ++i)
    if (!plain(p[i])) Py_RETURN_FALSE;
  if (!plain_thread()) Py_RETURN_FALSE;
  const Tensor &out = THPVariable_Unpack(p[0]), &q = THPVariable_Unpack(p[1]), &kc = THPVariable_Unpack(p[2]),
               &vc = THPVariable_Unpack(p[3]);
  THPObjectPtr buf_o = attr(p[4], names.buf), table_o = attr(p[4], names.page_table);
  if (!plain(buf_o) || !plain(table_o)) Py_RETURN_FALSE;
  const int64_t T = integer(attr(p[4], names.T)), S = integer(attr(p[4], names.S)), Hq = integer(attr(p[4], names.q_heads)),
                Hkv = integer(attr(p[4], names.kv_heads)), P = integer(attr(p[4], names.page_size));
  const Tensor &buf = THPVariable_Unpack(buf_o.get()), &table = THPVariable_Unpack(table_o.get());
  if (!half(q) || !here(q) || q.dim() != 3 || !heads(q, q) || !heads(out, q) || !written(out) || out.sizes() != q.sizes() || q.size(0) != T ||
      q.size(1) != Hq || (q.size(2) != 64 && q.size(2) != 128) || T == 0 || !caches(kc, vc, q, Hkv) || kc.size(2) != P ||
      buf.device() != q.device() || !on(table, q, at::kInt, 2))
    Py_RETURN_FALSE;
  double scale = p[5] == Py_None ? 1.0 / std::sqrt((double)q.size(2)) : PyFloat_AsDouble(p[5]);
  if (scale == -1.0 && PyErr_Occurred()) throw python_raised();
  if (!(scale > 0.0) || !(scale < 1.0e38)) Py_RETURN_FALSE;
  const int D = (int)q.size(2), M = (int)table.size(1);
  size_t need = 0;
  check(lib.attn_size((int)T, (int)S, M, (int)P, (int)Hq, (int)Hkv, D, &need), "smlm_paged_attn_workspace_size");
  Tensor mem;
  if (need) mem = scratch(p[6], need, q);
  const smlm_heads o = view(out), qv = view(q);
  check(lib.attn(&o, &qv, kc.data_ptr(), vc.data_ptr(), stride_of(kc, 0), stride_of(kc, 1), stride_of(kc, 2),
                 (const int32_t*)table.data_ptr(), buf.data_ptr(), (size_t)buf.numel(), need ? mem.data_ptr() : nullptr,
                 need ? (size_t)mem.numel() : 0, (int)T, (int)S, (int)table.size(0), M, (int)kc.size(0), (int)P, (int)Hq, (int)Hkv, D,
                 dtype_code(q), (float)scale, stream(q)),
        "paged_attention");
  Py_RETURN_TRUE;
  SMLM_PY_END
}

// table [R, M], length [R] (or null), refs [N], and int32 lists of one length; status may be null
bool pages(const Tensor& table, const Tensor* length, const Tensor& refs, const Tensor* status, const Tensor& a, const Tensor& b) {
  return is(table, at::kInt, 2) && here(table) && (!length || (on(*length, table, at::kInt, 1) && length->size(0) == table.size(0))) &&
         on(refs, table, at::kInt, 1) && (!status || (on(*status, table, at::kInt, 1) && status->size(0) == 1)) &&
         on(a, table, at::kInt, 1) && on(b, table, at::kInt, 1) && a.size(0) == b.size(0) && a.size(0) < (1 << 20) &&
         table.size(0) < (1 << 24) && table.size(1) < (1 << 20) && refs.size(0) < (1 << 28);
}

// kv_extend(table, length, refs, requests, counts, n_rows, page_size, status, workspace, max_tokens = None) -> the step's four tables, or None
PyObject* py_kv_extend(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  TORCH_CHECK(n == 9 || n == 10, "kv_extend takes 9 or 10 arguments");
  const bool limit = n == 10 && p[9] != Py_None;
  bool ok = plain_thread() && PyLong_CheckExact(p[5]) && PyLong_CheckExact(p[6]) && (!limit || PyLong_CheckExact(p[9]));
  for (int i = 0; i < 5; ++i) ok = ok && plain(p[i]);
  const Tensor* status = optional(p[7], &ok);
  if (!ok) Py_RETURN_NONE;
  const Tensor &table = THPVariable_Unpack(p[0]), &length = THPVariable_Unpack(p[1]), &refs = THPVariable_Unpack(p[2]),
               &req = THPVariable_Unpack(p[3]), &counts = THPVariable_Unpack(p[4]);
  const int64_t rows = integer(p[5]), P = integer(p[6]), most = limit ? integer(p[9]) : 0x7fffffff;
  if (most < 0 || most > 0x7fffffff || !pages(table, &length, refs, status, req, counts) || rows < 0 || rows > (1 << 20) || P < 1 ||
      P > (1 << 30))
    Py_RETURN_NONE;
  const int R = (int)table.size(0), M = (int)table.size(1), N = (int)refs.size(0), S = (int)req.size(0);
  const auto ints = table.options();
  Tensor indptr = at::empty({S + 1}, ints), len = at::empty({S}, ints), pos = at::empty({rows}, ints),
         slots = at::empty({rows}, ints.dtype(at::kLong));
  size_t need = 0;
  check(lib.kv_size(R, N, S, &need), "smlm_kv_workspace_size");
  const Tensor mem = scratch(p[8], need, table);
  auto i32 = [](const Tensor& t) { return (int32_t*)t.data_ptr(); };
  check(lib.kv_extend(i32(table), i32(length), i32(refs), i32(req), i32(counts), i32(indptr), i32(len), i32(pos),
                      (int64_t*)slots.data_ptr(), mem.data_ptr(), (size_t)mem.numel(), R, M, N, S, (int)rows, (int)P, (int)most,
                      status ? i32(*status) : nullptr, stream(table)),
        "kv_extend");
  THPObjectPtr o[4] = {THPObjectPtr(THPVariable_Wrap(std::move(indptr))), THPObjectPtr(THPVariable_Wrap(std::move(len))),
                       THPObjectPtr(THPVariable_Wrap(std::move(pos))), THPObjectPtr(THPVariable_Wrap(std::move(slots)))};
  return PyTuple_Pack(4, o[0].get(), o[1].get(), o[2].get(), o[3].get());
  SMLM_PY_END
}

// kv_free(table, length, refs, requests, page_size, status) -> whether it was done
PyObject* py_kv_free(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  TORCH_CHECK(n == 6, "kv_free takes 6 arguments");
  bool ok = plain_thread() && PyLong_CheckExact(p[4]);
  for (int i = 0; i < 4; ++i) ok = ok && plain(p[i]);
  const Tensor* status = optional(p[5], &ok);
  if (!ok) Py_RETURN_FALSE;
  const Tensor &table = THPVariable_Unpack(p[0]), &length = THPVariable_Unpack(p[1]), &refs = THPVariable_Unpack(p[2]),
               &req = THPVariable_Unpack(p[3]);
  const int64_t P = integer(p[4]);
  if (!pages(table, &length, refs, status, req, req) || P < 1 || P > (1 << 30)) Py_RETURN_FALSE;
  auto i32 = [](const Tensor& t) { return (int32_t*)t.data_ptr(); };
  check(lib.kv_free(i32(table), i32(length), i32(refs), i32(req), (int)table.size(0), (int)table.size(1), (int)refs.size(0),
                    (int)req.size(0), (int)P, status ? i32(*status) : nullptr, stream(table)),
        "kv_free");
  Py_RETURN_TRUE;
  SMLM_PY_END
}

// kv_fork(pool, table, length, refs, parents, children, status, workspace) -> whether it was done
PyObject* py_kv_fork(PyObject*, PyObject* const* p, Py_ssize_t n) {
  SMLM_PY_TRY
  TORCH_CHECK(n == 8, "kv_fork takes 8 arguments");
  bool ok = plain_thread();
  for (int i = 0; i < 6; ++i) ok = ok && plain(p[i]);
  const Tensor* status = optional(p[6], &ok);
  if (!ok) Py_RETURN_FALSE;
  const Tensor &pool = THPVariable_Unpack(p[0]), &table = THPVariable_Unpack(p[1]), &length = THPVariable_Unpack(p[2]),
               &refs = THPVariable_Unpack(p[3]), &par = THPVariable_Unpack(p[4]), &chi = THPVariable_Unpack(p[5]);
  if (!pages(table, &length, refs, status, par, chi) || pool.dim() < 3 || !pool.is_contiguous() || pool.device() != table.device() ||
      pool.numel() == 0 || pool.size(0) != refs.size(0))
    Py_RETURN_FALSE;
  const int64_t P = pool.size(-2), place = pool.size(-1) * pool.element_size(), blocks = pool.numel() / (pool.size(0) * P * pool.size(-1));
  if (place % 16 != 0 || P > (1 << 30) || place > (1 << 30) || blocks > (1 << 30)) Py_RETURN_FALSE;
  const int R = (int)table.size(0), M = (int)table.size(1), N = (int)refs.size(0), K = (int)chi.size(0);
  size_t need = 0;
  check(lib.kv_size(R, N, K, &need), "smlm_kv_workspace_size");
  const Tensor mem = scratch(p[7], need, table);
  auto i32 = [](const Tensor& t) { return (int32_t*)t.data_ptr(); };
  check(lib.kv_fork(pool.data_ptr(), i32(table), i32(length), i32(refs), i32(par), i32(chi), mem.data_ptr(), (size_t)mem.numel(), R, M, N,
                    K, (int)blocks, (int)P, (int)place, status ? i32(*status) : nullptr, stream(table)),
        "kv_fork");
  Py_RETURN_TRUE;
  SMLM_PY_END
}
