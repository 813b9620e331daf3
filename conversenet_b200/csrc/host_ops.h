// Host side of the operators around a block of any width (included by host.cpp, inside its namespace): the residual seam,
// the norm of many tensors and products in 8-bit integers.

const at::Tensor optional(PyObject* o, const char* what) {
  return o == Py_None ? at::Tensor() : cuda_tensor(o, what);
}
PyObject* wrap_or_none(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
template <class T>
T* data(const at::Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
void same_device(const at::Tensor& t, const at::Tensor& x, const char* what) {
  if (t.defined() && t.device() != x.device()) throw Failed(std::string(what) + " must be on the device of x");
}
void floating(const at::Tensor& t, const char* what) {
  if (t.defined() && !t.is_floating_point()) throw Failed(std::string(what) + " must be a floating-point tensor");
}

// (the kernels would lose it)
void no_tangent(const at::Tensor& t) {
  if (t.defined() && t._fw_grad(0).defined()) throw Failed("this operator has no forward-mode derivative, and an input is a dual tensor");
}

// The residual seam's arguments, checked, and laid out for the kernels
enum { kX, kBranch, kScale, kGate, kPostW, kPostB, kPreW, kPreB, kSeamTensors };
struct SeamConfig {
  double eps = 0;
  bool rms = false, sigmoid = false, last = false;
};
struct Seam {
  cvb_residual_norm_args A;
  std::array<at::Tensor, kSeamTensors> t;          // as given
  at::Tensor x, branch, gate, vec[kSeamTensors];   // as the kernels read them
  bool empty = false;

  Seam(std::array<at::Tensor, kSeamTensors> given, const SeamConfig& c) : t(std::move(given)) {
    static const char* names[] = {"x", "branch", "scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"};
    std::memset(&A, 0, sizeof(A));
    A.eps = (float)c.eps; A.rms = c.rms; A.gate_act = c.sigmoid; A.channels_last = c.last;
    const at::Tensor& x0 = t[kX];
    A.io_dtype = io_type(x0);
    if (c.last ? x0.dim() < 2 : x0.dim() != 4)
      throw Failed(c.last ? "x must be (...,C) with at least one token dimension" : "x must be (B,C,H,W)");
    if (!(A.eps >= 0)) throw Failed("eps must not be negative");
    const int64_t C = x0.size(c.last ? -1 : 1);
    if (C < 1 || C > 16384) throw Failed("residual_norm takes 1 to 16384 channels, got " + std::to_string(C));
    A.C = (int)C;
    if (t[kBranch].sizes() != x0.sizes()) throw Failed("branch must have the shape of x");
    if (t[kBranch].scalar_type() != x0.scalar_type()) throw Failed("branch must have the type of x");
    for (int i = kBranch; i < kSeamTensors; ++i) {
      if (!t[i].defined()) continue;
      same_device(t[i], x0, names[i]);
      floating(t[i], names[i]);
      if (i != kBranch && i != kGate && t[i].numel() != C) throw Failed(std::string(names[i]) + " must hold a value for each channel");
    }
    if ((t[kPostB].defined() && !t[kPostW].defined()) || (t[kPreB].defined() && !t[kPreW].defined()))
      throw Failed("a norm's bias needs its weight");
    empty = x0.numel() == 0;
    A.B = 1;
    A.HW = empty ? 0 : x0.numel() / C;
    if (!c.last) A.B = x0.size(0), A.HW = x0.size(2) * x0.size(3);
    const at::Tensor& g = t[kGate];
    if (!g.defined()) return;
    bool image = g.dim() == x0.dim() && g.size(0) == x0.size(0);
    for (int64_t d = 1; image && d < x0.dim(); ++d) image = g.size(d) == (d == (c.last ? x0.dim() - 1 : 1) ? C : 1);
    // (images of one pixel: both, and of any type as an image's gate)
    if (g.sizes() == x0.sizes() && (!image || g.scalar_type() == x0.scalar_type())) {
      if (g.scalar_type() != x0.scalar_type()) throw Failed("a gate for each element must have the type of x");
      A.gate_kind = CVB_GATE_FULL;
      return;
    }
    if (!image) throw Failed("gate must have the shape of x, or hold a value for each image and channel");
    A.gate_kind = CVB_GATE_IMAGE;
    if (c.last && !empty) A.B = x0.size(0), A.HW = x0.numel() / C / A.B;
  }
  // (no gradients are recorded here: the caller has none to record, or autograd's own function has switched them off)
  void lay_out() {
    x = t[kX].contiguous();
    branch = t[kBranch].contiguous();
    A.x = x.data_ptr(); A.branch = branch.data_ptr();
    for (int i = kScale; i < kSeamTensors; ++i)
      if (t[i].defined() && i != kGate) vec[i] = f32(t[i]);
    A.scale = data<const float>(vec[kScale]); A.post_w = data<const float>(vec[kPostW]); A.post_b = data<const float>(vec[kPostB]);
    A.pre_w = data<const float>(vec[kPreW]); A.pre_b = data<const float>(vec[kPreB]);
    if (A.gate_kind == CVB_GATE_FULL) gate = t[kGate].contiguous();
    if (A.gate_kind == CVB_GATE_IMAGE) gate = f32(t[kGate]);
    A.gate = data<void>(gate);
    A.stream = stream(x);
  }
};

// y, z (undefined without pre_w), the means and spreads that the gradients need (undefined unless `keep`)
std::array<at::Tensor, 3> seam_forward(Seam& s, bool keep) {
  s.lay_out();
  const auto opt = s.x.options().requires_grad(false);
  at::Tensor y = at::empty(s.x.sizes(), opt), z, stats;
  if (s.A.pre_w) z = at::empty(s.x.sizes(), opt);
  if (keep && (s.A.pre_w || s.A.post_w)) stats = at::empty({4, s.A.B * s.A.HW}, opt.dtype(at::kFloat));
  if (!s.empty) {
    s.A.y = y.data_ptr(); s.A.z = data<void>(z); s.A.stats = data<float>(stats);
    check(api.residual_norm_fwd(&s.A), "cvb_residual_norm_fwd");
  }
  return {y, z, stats};
}

// gradients of the tensors whose bit is set in `wanted`, from those of y and z (either may be undefined)
std::array<at::Tensor, kSeamTensors> seam_backward(Seam& s, const at::Tensor& stats, at::Tensor dy, at::Tensor dz, unsigned wanted) {
  std::array<at::Tensor, kSeamTensors> g;
  s.lay_out();
  const auto opt = s.x.options().requires_grad(false);
  if (!s.A.pre_w) dz = at::Tensor();
  for (int i = 0; i < kSeamTensors; ++i) {
    const bool like_x = i == kX || i == kBranch || (i == kGate && s.A.gate_kind == CVB_GATE_FULL);
    if ((wanted >> i & 1) && s.t[i].defined()) g[i] = at::empty(s.t[i].sizes(), like_x ? opt : opt.dtype(at::kFloat));
  }
  auto zero = [&](int from) {
    for (int i = from; i < kSeamTensors; ++i)
      if (g[i].defined()) g[i].zero_();
  };
  if (s.empty || (!dy.defined() && !dz.defined())) {
    zero(0);
  } else {
    for (at::Tensor* t : {&dy, &dz}) {
      if (t->defined()) *t = t->to(s.x.scalar_type()).contiguous();
      if (t->defined() && t->sizes() != s.x.sizes()) throw Failed("a gradient must have the shape of its output");
    }
    auto& A = s.A;
    A.stats = data<float>(stats); A.dy = data<void>(dy); A.dz = data<void>(dz);
    A.dx = data<void>(g[kX]); A.dbranch = data<void>(g[kBranch]); A.dscale = data<float>(g[kScale]); A.dgate = data<void>(g[kGate]);
    A.dpost_w = data<float>(g[kPostW]); A.dpost_b = data<float>(g[kPostB]);
    if (dz.defined()) A.dpre_w = data<float>(g[kPreW]), A.dpre_b = data<float>(g[kPreB]);
    else zero(kPreW);
    at::Tensor work;
    if (A.dscale || A.dpost_w || A.dpost_b || A.dpre_w || A.dpre_b || (A.dgate && A.gate_kind == CVB_GATE_IMAGE)) {
      A.workspace_bytes = api.residual_norm_workspace(A.C, A.B, A.gate_kind);
      work = bytes_like(s.x, A.workspace_bytes);
      A.workspace = work.data_ptr();
    }
    if (A.dx || A.dbranch || A.dgate || A.workspace) check(api.residual_norm_bwd(&A), "cvb_residual_norm_bwd");
  }
  for (int i = kScale; i < kSeamTensors; ++i)
    if (g[i].defined() && g[i].scalar_type() != s.t[i].scalar_type()) g[i] = g[i].to(s.t[i].scalar_type());
  return g;
}

// The seam under autograd, without the interpreter: a node of Python's took 140 us a step, of which the kernels are 30.
struct SeamFunction : torch::autograd::Function<SeamFunction> {
  using Opt = std::optional<at::Tensor>;
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& branch,
                                                const Opt& scale, const Opt& gate, const Opt& post_w, const Opt& post_b,
                                                const Opt& pre_w, const Opt& pre_b, SeamConfig c) {
    auto in = [](const Opt& t) { return t.has_value() ? *t : at::Tensor(); };
    Seam s({x, branch, in(scale), in(gate), in(post_w), in(post_b), in(pre_w), in(pre_b)}, c);
    auto out = seam_forward(s, true);
    ctx->set_materialize_grads(false);
    ctx->saved_data["eps"] = c.eps;
    ctx->saved_data["flags"] = (int64_t)(c.rms | c.sigmoid << 1 | c.last << 2);
    ctx->save_for_backward({out[2], s.t[0], s.t[1], s.t[2], s.t[3], s.t[4], s.t[5], s.t[6], s.t[7]});
    if (out[1].defined()) return {out[0], out[1]};
    return {out[0]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    SeamConfig c;
    c.eps = ctx->saved_data["eps"].toDouble();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    c.rms = flags & 1; c.sigmoid = flags >> 1 & 1; c.last = flags >> 2 & 1;
    const c10::cuda::CUDAGuard dev(saved[1].device());
    std::array<at::Tensor, kSeamTensors> t;
    unsigned wanted = 0;
    size_t edge = 0;
    for (int i = 0; i < kSeamTensors; ++i) {
      t[i] = saved[1 + i];
      if (t[i].defined() && ctx->needs_input_grad(edge++)) wanted |= 1u << i;
    }
    const bool again = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    Seam s(std::move(t), c);
    auto g = seam_backward(s, saved[0], grads[0], grads.size() > 1 ? grads[1] : at::Tensor(), wanted);
    torch::autograd::variable_list out(g.begin(), g.end());
    if (again) {          // a graph of the backward is wanted: whoever goes through it learns that there is none
      const at::AutoGradMode grad(true);
      for (auto& o : out)
        if (o.defined()) o.requires_grad_(true);
      out = (*std::make_shared<torch::autograd::DelayedError>("residual_norm can be differentiated once", (int64_t)out.size()))(std::move(out));
    }
    out.emplace_back();
    return out;
  }
};

// residual_norm(x, branch, scale, gate, post_w, post_b, pre_w, pre_b, eps, rms, sigmoid, channels_last, under autograd) ->
// (y, z or None)
PyObject* py_residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 13);
    static const char* names[] = {"x", "branch", "scale", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"};
    std::array<at::Tensor, kSeamTensors> t;
    for (int i = 0; i < kSeamTensors; ++i) t[i] = i <= kBranch ? cuda_tensor(a[i], names[i]) : optional(a[i], names[i]);
    for (const at::Tensor& one : t) no_tangent(one);
    SeamConfig c;
    c.eps = real(a[8]);
    c.rms = PyObject_IsTrue(a[9]); c.sigmoid = PyObject_IsTrue(a[10]); c.last = PyObject_IsTrue(a[11]);
    const bool graph = PyObject_IsTrue(a[12]);
    const c10::cuda::CUDAGuard dev(t[kX].device());
    at::Tensor y, z;
    {
      const Unlocked unlocked;
      if (graph) {
        auto opt = [&](int i) { return t[i].defined() ? SeamFunction::Opt(t[i]) : SeamFunction::Opt(); };
        auto out = SeamFunction::apply(t[kX], t[kBranch], opt(kScale), opt(kGate), opt(kPostW), opt(kPostB), opt(kPreW), opt(kPreB), c);
        y = out[0];
        if (out.size() > 1) z = out[1];
      } else {
        Seam s(std::move(t), c);
        auto out = seam_forward(s, false);
        y = out[0];
        z = out[1];
      }
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(y)), wrap_or_none(z));
  });
}

// ---- the norm of many tensors
// A sequence of tensors, held as Python holds it for as long as this lives (a count of its own for each would take as long as the
// rest of a call): only the interpreter's lock may be given up in between.
struct TensorList {
  PyObject* held = nullptr;
  std::vector<const at::Tensor*> t;
  TensorList() = default;
  TensorList(const TensorList&) = delete;
  ~TensorList() { Py_XDECREF(held); }
  void read(PyObject* o, const char* what) {
    held = PySequence_Tuple(o);
    if (!held) throw std::invalid_argument(what);
    const Py_ssize_t n = PyTuple_GET_SIZE(held);
    t.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) t.push_back(&tensor(PyTuple_GET_ITEM(held, i), what));
  }
  size_t size() const { return t.size(); }
};
struct Range {
  uintptr_t from, to;
  bool operator<(const Range& o) const { return from < o.from; }
};
// Outputs may not share memory with one another, nor with inputs other than their own: two blocks would write it, or one
// read what another has written.
void refuse_overlap(const std::vector<cvb_span>& s) {
  auto bytes = [](long long n, int type) { return (uintptr_t)n * (type == CVB_F32 ? 4 : 2); };
  std::vector<Range> outs;
  outs.reserve(s.size());
  bool sorted = true;
  for (const cvb_span& t : s) {
    if (!t.n) continue;
    const Range r{(uintptr_t)t.out, (uintptr_t)t.out + bytes(t.n, t.out_type)};
    if (!outs.empty() && r < outs.back()) sorted = false;
    outs.push_back(r);
  }
  if (!sorted) std::sort(outs.begin(), outs.end());
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].from < outs[i - 1].to) throw Failed("two of the tensors to be written share memory");
  if (outs.empty()) return;
  const uintptr_t low = outs.front().from, high = outs.back().to;
  for (const cvb_span& t : s) {
    if (!t.n || (t.in == t.out && t.in_type == t.out_type)) continue;      // in place: seen above
    const uintptr_t from = (uintptr_t)t.in, to = from + bytes(t.n, t.in_type);
    if (to <= low || from >= high) continue;
    auto it = std::lower_bound(outs.begin(), outs.end(), Range{from, to});
    if ((it != outs.end() && it->from < to) || (it != outs.begin() && (it - 1)->to > from))
      throw Failed("a tensor to be written shares memory with another tensor that is read");
  }
}

// clip_by_norm(tensors, out: None for new tensors, True for the tensors themselves, a sequence, or False for the norm alone,
// kind, max_norm) -> (out or None, norm)
PyObject* py_clip_by_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 4);
    TensorList in, given;
    in.read(a[0], "tensors");
    if (!in.size()) throw Failed("no tensors");
    const bool scale = a[1] != Py_False, fresh = a[1] == Py_None, self = a[1] == Py_True;
    if (scale && !fresh && !self) {
      given.read(a[1], "out");
      if (given.size() != in.size()) throw Failed("out must hold a tensor for each of the tensors");
    }
    const int kind = (int)integer(a[2]);
    const double max_norm = real(a[3]);
    if (scale && !(max_norm >= 0)) throw Failed("max_norm must not be negative");
    const at::Tensor& first = *in.t[0];
    if (!first.is_cuda()) throw Failed("the tensors must be CUDA tensors; this build has no CPU path");
    const c10::Device where = first.device();
    const c10::cuda::CUDAGuard dev(where);
    // (gradients may have one, of a double backward: they are scaled in place all the same, as torch does it)
    const bool history = !self && at::GradMode::is_enabled();
    const char* no_history = "norms and scaled tensors have no history: call it under torch.no_grad() for tensors that require gradients";
    at::Tensor norm;
    std::vector<at::Tensor> made;          // new tensors
    {
      const Unlocked unlocked;
      std::vector<cvb_span> s(in.size());
      std::vector<at::Tensor> copies;      // of tensors that are read through one
      if (fresh) made.reserve(in.size());
      // requires_grad(), which asks a view's base: of views of one buffer once (284 of them took 2 us)
      const c10::TensorImpl* asked = nullptr;
      auto recorded = [&](const c10::TensorImpl* impl) {
        const auto* meta = static_cast<const torch::autograd::AutogradMeta*>(impl->autograd_meta());
        if (!meta) return false;
        if (meta->requires_grad_ || meta->grad_fn_) return true;
        if (!meta->is_view_) return false;
        const auto* view = static_cast<const torch::autograd::DifferentiableViewMeta*>(meta);
        if (!view->has_bw_view()) return false;
        const at::Tensor& base = view->get_backward_view().base_;
        if (base.unsafeGetTensorImpl() == asked) return false;
        asked = base.unsafeGetTensorImpl();
        return base.requires_grad();
      };
      for (size_t i = 0; i < in.size(); ++i) {
        const at::Tensor& t = *in.t[i];
        const void* from = nullptr;
        auto copy = [&] {
          copies.push_back(t.contiguous());
          from = copies.back().const_data_ptr();
        };
        const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
        if (impl->layout() != at::kStrided) throw Failed("sparse tensors are not supported");
        if (impl->autograd_meta()) {          // (few have any)
          if (history && recorded(impl)) throw Failed(no_history);
          no_tangent(t);
        }
        if (impl->device() != where) throw Failed("the tensors must be on one CUDA device; this build has no CPU path");
        s[i].in_type = s[i].out_type = io_type(t);
        s[i].n = impl->numel();
        const bool whole = impl->is_contiguous(), flat = whole || t.is_non_overlapping_and_dense();
        if (fresh) made.push_back(at::empty_like(t, t.options().requires_grad(false),
                                                flat ? at::MemoryFormat::Preserve : at::MemoryFormat::Contiguous));
        if (self && !flat) throw Failed("a tensor to be scaled in place must fill its memory (no slices or expanded tensors)");
        if (fresh || given.size()) {
          const at::Tensor& o = fresh ? made[i] : *given.t[i];
          const c10::TensorImpl* to = o.unsafeGetTensorImpl();
          if (to->layout() != at::kStrided || to->sizes() != impl->sizes()) throw Failed("each tensor of out must have the shape of its tensor");
          if (to->device() != where) throw Failed("out must be on the device of the tensors");
          if (history && !fresh && recorded(to)) throw Failed(no_history);
          s[i].out_type = io_type(o);
          if (!(whole && to->is_contiguous()) && !(flat && o.strides() == t.strides())) {
            if (!to->is_contiguous()) throw Failed("a tensor of out must be contiguous or have the strides of its tensor");
            if (!whole) copy();
          }
          s[i].out = o.data_ptr();
        } else if (!flat) {
          copy();
        }
        s[i].in = from ? from : t.const_data_ptr();
        if (self) s[i].out = t.data_ptr();
      }
      if (scale) refuse_overlap(s);
      norm = at::empty({}, first.options().dtype(at::kFloat).requires_grad(false));
      const size_t ws = api.clip_workspace((int)s.size());
      at::Tensor work = bytes_like(first, ws);
      check(api.clip_by_norm(s.data(), (int)s.size(), kind, max_norm, scale, (float*)norm.data_ptr(), work.data_ptr(), ws,
                             stream(first)),
            "cvb_clip_by_norm");
      // (autograd learns that they changed)
      if (scale && !fresh)
        for (const at::Tensor* t : self ? in.t : given.t)
          if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    }
    if (!scale || self) return Py_BuildValue("(ON)", Py_None, THPVariable_Wrap(norm));
    if (!fresh) return Py_BuildValue("(ON)", a[1], THPVariable_Wrap(norm));
    PyObject* list = PyList_New((Py_ssize_t)made.size());
    for (size_t i = 0; i < made.size(); ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, THPVariable_Wrap(made[i]));
    return Py_BuildValue("(NN)", list, THPVariable_Wrap(norm));
  });
}

// ---- products in 8-bit integers
// Tokens as the kernels count them: channels_first (B,K,H,W), channels_last (...,K)
struct Tokens {
  long long B = 1, HW = 0;
  int K = 0;
  bool last = false;
  std::vector<int64_t> lead;          // the token dimensions
  Tokens(const at::Tensor& x, bool channels_last) : last(channels_last) {
    if (last ? x.dim() < 2 : x.dim() != 4)
      throw Failed(last ? "x must be (...,C) with at least one token dimension" : "x must be (B,C,H,W)");
    const int64_t k = x.size(last ? -1 : 1);
    if (k < 1 || k > 131072) throw Failed("8-bit products take 1 to 131072 channels, got " + std::to_string(k));
    K = (int)k;
    if (last) {
      HW = x.numel() / K;
      lead.assign(x.sizes().begin(), x.sizes().end() - 1);
    } else {
      B = x.size(0);
      HW = x.size(2) * x.size(3);
      lead = {x.size(0), x.size(2), x.size(3)};
    }
    if (B * HW > 0x7fffff00ll) throw Failed("too many tokens for an 8-bit product");
  }
  std::vector<int64_t> result(int64_t N) const {
    if (!last) return {lead[0], N, lead[1], lead[2]};
    std::vector<int64_t> v = lead;
    v.push_back(N);
    return v;
  }
};
// rows of 8-bit integers that begin at multiples of 16 bytes, as they are or copied; `ld` is their distance
at::Tensor int8_rows(const at::Tensor& t, long long& ld) {
  const int64_t rows = t.size(0), K = t.size(1), padded = (K + 15) / 16 * 16;
  const bool fits = (K == 1 || t.stride(1) == 1) && (size_t)t.data_ptr() % 16 == 0 &&
                    (rows == 1 || (t.stride(0) % 16 == 0 && t.stride(0) >= K));
  ld = rows == 1 ? padded : fits ? t.stride(0) : padded;
  if (fits) return t;
  at::Tensor all = at::empty({rows, padded}, t.options());
  all.narrow(1, 0, K).copy_(t);
  return all;
}
struct Int8Weight {
  at::Tensor w, scale, bias;
  long long ld = 0;
  int N = 0;
  Int8Weight(PyObject* w_, PyObject* scale_, PyObject* bias_, const at::Tensor& x, int K) {
    w = cuda_tensor(w_, "weight_q");
    scale = cuda_tensor(scale_, "weight_scale");
    bias = optional(bias_, "bias");
    if (w.scalar_type() != at::kChar || w.dim() != 2 || w.size(1) != K || w.size(0) < 1)
      throw Failed("weight_q must be int8 (N," + std::to_string(K) + ")");
    N = (int)w.size(0);
    floating(scale, "weight_scale");
    floating(bias, "bias");
    no_tangent(scale);
    no_tangent(bias);
    if (scale.numel() != N) throw Failed("weight_scale must hold a value for each output channel");
    if (bias.defined() && bias.numel() != N) throw Failed("bias must hold a value for each output channel");
    same_device(w, x, "weight_q");
    same_device(scale, x, "weight_scale");
    same_device(bias, x, "bias");
  }
  void lay_out() {
    w = int8_rows(w, ld);
    scale = f32(scale);
    if (bias.defined()) bias = f32(bias);
  }
};

// quantize_tokens(x, channels_last) -> (q int8 (tokens' dimensions, K), scale (tokens' dimensions))
PyObject* py_quantize_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 2);
    const at::Tensor& x0 = cuda_tensor(a[0], "x");
    no_tangent(x0);
    const c10::cuda::CUDAGuard dev(x0.device());
    const int io = io_type(x0);
    const Tokens t(x0, PyObject_IsTrue(a[1]));
    at::Tensor q, scale;
    {
      const Unlocked unlocked;
      const at::Tensor x = x0.contiguous();
      const int64_t padded = (t.K + 15) / 16 * 16;
      std::vector<int64_t> sizes = t.lead;
      scale = at::empty(sizes, x.options().dtype(at::kFloat).requires_grad(false));
      sizes.push_back(padded);
      q = at::empty(sizes, x.options().dtype(at::kChar).requires_grad(false));
      if (x.numel())
        check(api.quantize_tokens(x.data_ptr(), (signed char*)q.data_ptr(), (float*)scale.data_ptr(), t.B, t.HW, t.K, padded, t.last,
                                  io, stream(x)),
              "cvb_quantize_tokens");
      if (padded != t.K) q = q.narrow(-1, 0, t.K);
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(scale)));
  });
}

// int8_product(q, scale, weight_q, weight_scale, bias, bf16, channels_last) -> out; q (tokens' dimensions, K)
PyObject* py_int8_product(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 7);
    const at::Tensor &q0 = cuda_tensor(a[0], "q"), &s0 = cuda_tensor(a[1], "scale");
    const c10::cuda::CUDAGuard dev(q0.device());
    if (q0.scalar_type() != at::kChar) throw Failed("q must be int8");
    const bool bf16 = PyObject_IsTrue(a[5]), last = PyObject_IsTrue(a[6]);
    if (!last && q0.dim() != 4) throw Failed("q must be (B,H,W,K) for a channels_first result");
    Tokens t(q0, true);
    if (!last) t.B = q0.size(0), t.HW = q0.size(1) * q0.size(2), t.last = false;
    floating(s0, "scale");
    no_tangent(s0);
    same_device(s0, q0, "scale");
    if (s0.numel() != t.B * t.HW) throw Failed("scale must hold a value for each token");
    Int8Weight w(a[2], a[3], a[4], q0, t.K);
    at::Tensor out;
    {
      const Unlocked unlocked;
      out = at::empty(t.result(w.N), q0.options().dtype(bf16 ? at::kBFloat16 : at::kFloat).requires_grad(false));
      if (out.numel()) {
        w.lay_out();
        long long ld;
        const at::Tensor q = int8_rows(q0.reshape({-1, t.K}), ld), scale = f32(s0);
        check(api.int8_product((const signed char*)q.data_ptr(), ld, (const float*)scale.data_ptr(), (const signed char*)w.w.data_ptr(),
                               w.ld, (const float*)w.scale.data_ptr(), data<const float>(w.bias), out.data_ptr(), t.B, t.HW, t.K, w.N,
                               last, bf16 ? CVB_BF16 : CVB_F32, stream(q0)),
              "cvb_int8_product");
      }
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// pointwise_int8(x, weight_q, weight_scale, bias, channels_last) -> out
PyObject* py_pointwise_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 5);
    const at::Tensor& x0 = cuda_tensor(a[0], "x");
    no_tangent(x0);
    const c10::cuda::CUDAGuard dev(x0.device());
    const int io = io_type(x0);
    const Tokens t(x0, PyObject_IsTrue(a[4]));
    Int8Weight w(a[1], a[2], a[3], x0, t.K);
    at::Tensor out;
    {
      const Unlocked unlocked;
      out = at::empty(t.result(w.N), x0.options().requires_grad(false));
      if (out.numel()) {
        w.lay_out();
        const at::Tensor x = x0.contiguous();
        const size_t ws = api.pointwise_int8_workspace(t.B, t.HW, t.K, w.N, t.last, io);
        at::Tensor work;
        if (ws) work = bytes_like(x, ws);
        check(api.pointwise_int8(x.data_ptr(), (const signed char*)w.w.data_ptr(), w.ld, (const float*)w.scale.data_ptr(),
                                 data<const float>(w.bias), out.data_ptr(), t.B, t.HW, t.K, w.N, t.last, io,
                                 ws ? work.data_ptr() : nullptr, ws, stream(x)),
              "cvb_pointwise_int8");
      }
    }
    return THPVariable_Wrap(std::move(out));
  });
}
