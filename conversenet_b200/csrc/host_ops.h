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

// The arguments that both directions of the seam share, checked
struct Seam {
  cvb_residual_norm_args A;
  at::Tensor x, branch, gate, vec[5];          // vec: scale, post_w, post_b, pre_w, pre_b as given
  at::Tensor keep[5], gate_kept;               // as the kernels read them
  bool empty = false;

  // a: x-like, branch, scale, gate, post_w, post_b, pre_w, pre_b; eps, rms, sigmoid, channels_last
  void read(const at::Tensor& like, PyObject* const* a) {
    static const char* names[5] = {"scale", "post_weight", "post_bias", "pre_weight", "pre_bias"};
    std::memset(&A, 0, sizeof(A));
    x = like;
    branch = optional(a[0], "branch");
    vec[0] = optional(a[1], names[0]);
    gate = optional(a[2], "gate");
    for (int i = 1; i < 5; ++i) vec[i] = optional(a[2 + i], names[i]);
    A.eps = (float)real(a[7]);
    A.rms = PyObject_IsTrue(a[8]);
    A.gate_act = PyObject_IsTrue(a[9]);
    A.channels_last = PyObject_IsTrue(a[10]);
    A.io_dtype = io_type(x);
    if (A.channels_last ? x.dim() < 2 : x.dim() != 4)
      throw Failed(A.channels_last ? "x must be (...,C) with at least one token dimension" : "x must be (B,C,H,W)");
    if (!(A.eps >= 0)) throw Failed("eps must not be negative");
    const int64_t C = x.size(A.channels_last ? -1 : 1);
    if (C < 1 || C > 16384) throw Failed("residual_norm takes 1 to 16384 channels, got " + std::to_string(C));
    A.C = (int)C;
    same_device(branch, x, "branch");
    if (branch.defined() && branch.sizes() != x.sizes()) throw Failed("branch must have the shape of x");
    if (branch.defined() && branch.scalar_type() != x.scalar_type()) throw Failed("branch must have the type of x");
    for (int i = 0; i < 5; ++i) {
      same_device(vec[i], x, names[i]);
      floating(vec[i], names[i]);
      if (vec[i].defined() && vec[i].numel() != C) throw Failed(std::string(names[i]) + " must hold a value for each channel");
    }
    if ((vec[2].defined() && !vec[1].defined()) || (vec[4].defined() && !vec[3].defined()))
      throw Failed("a norm's bias needs its weight");
    empty = x.numel() == 0;
    A.B = 1;
    A.HW = empty ? 0 : x.numel() / C;
    if (!A.channels_last) A.B = x.size(0), A.HW = x.size(2) * x.size(3);
    if (!gate.defined()) return;
    same_device(gate, x, "gate");
    floating(gate, "gate");
    if (gate.sizes() == x.sizes()) {
      if (gate.scalar_type() != x.scalar_type()) throw Failed("a gate for each element must have the type of x");
      A.gate_kind = CVB_GATE_FULL;
      return;
    }
    bool image = gate.dim() == x.dim() && gate.size(0) == x.size(0);
    for (int64_t d = 1; image && d < x.dim(); ++d)
      image = gate.size(d) == (d == (A.channels_last ? x.dim() - 1 : 1) ? C : 1);
    if (!image) throw Failed("gate must have the shape of x, or hold a value for each image and channel");
    A.gate_kind = CVB_GATE_IMAGE;
    if (A.channels_last && !empty) A.B = x.size(0), A.HW = x.numel() / C / A.B;
  }
  // contiguous copies where they are needed (the interpreter's lock is not)
  void lay_out() {
    if (branch.defined()) branch = branch.detach().contiguous();
    A.branch = data<void>(branch);
    const float* p[5];
    for (int i = 0; i < 5; ++i) {
      if (vec[i].defined()) keep[i] = f32(vec[i].detach());
      p[i] = data<const float>(keep[i]);
    }
    A.scale = p[0]; A.post_w = p[1]; A.post_b = p[2]; A.pre_w = p[3]; A.pre_b = p[4];
    if (A.gate_kind == CVB_GATE_FULL) gate_kept = gate.detach().contiguous();
    if (A.gate_kind == CVB_GATE_IMAGE) gate_kept = f32(gate.detach());
    A.gate = data<void>(gate_kept);
  }
};

// residual_norm(x, branch, scale, gate, post_w, post_b, pre_w, pre_b, eps, rms, sigmoid, channels_last, keep) ->
// (y, z or None, stats or None)
PyObject* py_residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 13);
    const at::Tensor& x0 = cuda_tensor(a[0], "x");
    const c10::cuda::CUDAGuard dev(x0.device());
    Seam s;
    s.read(x0, a + 1);
    if (!s.branch.defined()) throw Failed("branch must be a tensor");
    const bool keep = PyObject_IsTrue(a[12]);
    at::Tensor y, z, stats;
    {
      const Unlocked unlocked;
      s.lay_out();
      const at::Tensor x = x0.detach().contiguous();
      const auto opt = x.options().requires_grad(false);
      y = at::empty(x.sizes(), opt);
      if (s.A.pre_w) z = at::empty(x.sizes(), opt);
      if (keep && (s.A.pre_w || s.A.post_w)) stats = at::empty({4, s.A.B * s.A.HW}, opt.dtype(at::kFloat));
      if (!s.empty) {
        s.A.x = x.data_ptr(); s.A.y = y.data_ptr(); s.A.z = data<void>(z); s.A.stats = data<float>(stats);
        s.A.stream = stream(x);
        check(api.residual_norm_fwd(&s.A), "cvb_residual_norm_fwd");
      }
    }
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(y)), wrap_or_none(z), wrap_or_none(stats));
  });
}

// residual_norm_backward(x, branch, scale, gate, post_w, post_b, pre_w, pre_b, eps, rms, sigmoid, channels_last, stats, dy or
// None, dz or None, wanted) -> gradients of (x, branch, scale, gate, post_w, post_b, pre_w, pre_b), None where the bit of
// `wanted` is not set
PyObject* py_residual_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 16);
    const at::Tensor& x0 = cuda_tensor(a[0], "x");
    const c10::cuda::CUDAGuard dev(x0.device());
    Seam s;
    s.read(x0, a + 1);
    const at::Tensor stats = optional(a[12], "stats");
    at::Tensor dy = optional(a[13], "dy"), dz = optional(a[14], "dz");
    const long wanted = integer(a[15]);
    at::Tensor g[8];
    {
      const Unlocked unlocked;
      s.lay_out();
      const auto opt = x0.options().requires_grad(false);
      const at::Tensor* given[8] = {&x0, &s.branch, &s.vec[0], &s.gate, &s.vec[1], &s.vec[2], &s.vec[3], &s.vec[4]};
      auto make = [&](int i, bool fp32) {
        if ((wanted >> i & 1) && given[i]->defined())
          g[i] = at::empty(given[i]->sizes(), fp32 ? opt.dtype(at::kFloat) : opt);
      };
      for (int i = 0; i < 8; ++i) make(i, i == 2 || i > 3 || (i == 3 && s.A.gate_kind == CVB_GATE_IMAGE));
      if (s.empty || (!dy.defined() && !dz.defined())) {
        for (auto& t : g)
          if (t.defined()) t.zero_();
      } else {
        const at::Tensor x = x0.detach().contiguous();
        auto like = [&](at::Tensor& t) {
          if (t.defined()) t = t.detach().to(x.scalar_type()).contiguous();
          if (t.defined() && t.sizes() != x.sizes()) throw Failed("a gradient must have the shape of its output");
        };
        like(dy);
        like(dz);
        auto& A = s.A;
        A.x = x.data_ptr(); A.stats = data<float>(stats); A.dy = data<void>(dy); A.dz = data<void>(dz);
        A.dx = data<void>(g[0]); A.dbranch = data<void>(g[1]); A.dscale = data<float>(g[2]); A.dgate = data<void>(g[3]);
        A.dpost_w = data<float>(g[4]); A.dpost_b = data<float>(g[5]);
        if (dz.defined()) {
          A.dpre_w = data<float>(g[6]); A.dpre_b = data<float>(g[7]);
        } else {
          for (int i = 6; i < 8; ++i)
            if (g[i].defined()) g[i].zero_();
        }
        at::Tensor work;
        if (A.dscale || A.dpost_w || A.dpost_b || A.dpre_w || A.dpre_b || (A.dgate && A.gate_kind == CVB_GATE_IMAGE)) {
          A.workspace_bytes = api.residual_norm_workspace(A.C, A.B, A.gate_kind);
          work = bytes_like(x, A.workspace_bytes);
          A.workspace = work.data_ptr();
        }
        A.stream = stream(x);
        if (A.dx || A.dbranch || A.dgate || A.workspace) check(api.residual_norm_bwd(&A), "cvb_residual_norm_bwd");
      }
      for (int i = 2; i < 8; ++i)
        if (g[i].defined() && g[i].scalar_type() != given[i]->scalar_type()) g[i] = g[i].to(given[i]->scalar_type());
    }
    return Py_BuildValue("(NNNNNNNN)", wrap_or_none(g[0]), wrap_or_none(g[1]), wrap_or_none(g[2]), wrap_or_none(g[3]),
                         wrap_or_none(g[4]), wrap_or_none(g[5]), wrap_or_none(g[6]), wrap_or_none(g[7]));
  });
}

// ---- the norm of many tensors
std::vector<at::Tensor> tensor_list(PyObject* o, const char* what) {
  PyObject* fast = PySequence_Fast(o, "a sequence of tensors is wanted");
  if (!fast) throw std::invalid_argument(what);
  std::vector<at::Tensor> v;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
  v.reserve(n);
  try {
    for (Py_ssize_t i = 0; i < n; ++i) v.push_back(tensor(PySequence_Fast_GET_ITEM(fast, i), what));
  } catch (...) {
    Py_DECREF(fast);
    throw;
  }
  Py_DECREF(fast);
  return v;
}
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
    std::vector<at::Tensor> in = tensor_list(a[0], "tensors"), out;
    if (in.empty()) throw Failed("no tensors");
    const bool scale = a[1] != Py_False, fresh = a[1] == Py_None, self = a[1] == Py_True;
    if (scale && !fresh && !self) {
      out = tensor_list(a[1], "out");
      if (out.size() != in.size()) throw Failed("out must hold a tensor for each of the tensors");
    }
    const int kind = (int)integer(a[2]);
    const double max_norm = real(a[3]);
    if (scale && !(max_norm >= 0)) throw Failed("max_norm must not be negative");
    for (const at::Tensor& t : in) {
      if (!t.is_cuda()) throw Failed("the tensors must be CUDA tensors; this build has no CPU path");
      if (t.layout() != at::kStrided) throw Failed("sparse tensors are not supported");
      if (t.device() != in[0].device()) throw Failed("the tensors must be on one device");
    }
    const c10::cuda::CUDAGuard dev(in[0].device());
    at::Tensor norm;
    {
      const Unlocked unlocked;
      std::vector<cvb_span> s(in.size());
      if (fresh) out.reserve(in.size());
      for (size_t i = 0; i < in.size(); ++i) {
        at::Tensor& t = in[i];
        s[i].in_type = s[i].out_type = io_type(t);
        s[i].n = t.numel();
        const bool flat = t.is_contiguous() || t.is_non_overlapping_and_dense();
        if (fresh) out.push_back(at::empty_like(t, t.options().requires_grad(false),
                                                flat ? at::MemoryFormat::Preserve : at::MemoryFormat::Contiguous));
        if (self && !flat) throw Failed("a tensor to be scaled in place must fill its memory (no slices or expanded tensors)");
        if (!out.empty()) {
          const at::Tensor& o = out[i];
          if (!o.is_cuda() || o.device() != t.device()) throw Failed("out must be on the device of the tensors");
          if (o.layout() != at::kStrided || o.sizes() != t.sizes()) throw Failed("each tensor of out must have the shape of its tensor");
          s[i].out_type = io_type(o);
          if (!(flat && o.strides() == t.strides())) {
            if (!o.is_contiguous()) throw Failed("a tensor of out must be contiguous or have the strides of its tensor");
            if (!t.is_contiguous()) t = t.contiguous();
          }
          s[i].out = o.data_ptr();
        } else if (!flat) {
          t = t.contiguous();
        }
        s[i].in = t.data_ptr();
        if (self) s[i].out = t.data_ptr();
      }
      if (scale) refuse_overlap(s);
      norm = at::empty({}, in[0].options().dtype(at::kFloat).requires_grad(false));
      const size_t ws = api.clip_workspace((int)s.size());
      at::Tensor work = bytes_like(in[0], ws);
      check(api.clip_by_norm(s.data(), (int)s.size(), kind, max_norm, scale, (float*)norm.data_ptr(), work.data_ptr(), ws,
                             stream(in[0])),
            "cvb_clip_by_norm");
      // (autograd learns that they changed)
      if (scale && !fresh)
        for (const at::Tensor& t : self ? in : out)
          if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    if (!scale || self) return Py_BuildValue("(ON)", Py_None, THPVariable_Wrap(norm));
    if (!fresh) return Py_BuildValue("(ON)", a[1], THPVariable_Wrap(norm));
    PyObject* list = PyList_New((Py_ssize_t)out.size());
    for (size_t i = 0; i < out.size(); ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, THPVariable_Wrap(out[i]));
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
    if (scale.numel() != N) throw Failed("weight_scale must hold a value for each output channel");
    if (bias.defined() && bias.numel() != N) throw Failed("bias must hold a value for each output channel");
    same_device(w, x, "weight_q");
    same_device(scale, x, "weight_scale");
    same_device(bias, x, "bias");
  }
  void lay_out() {
    w = int8_rows(w.detach(), ld);
    scale = f32(scale.detach());
    if (bias.defined()) bias = f32(bias.detach());
  }
};

// quantize_tokens(x, channels_last) -> (q int8 (tokens' dimensions, K), scale (tokens' dimensions))
PyObject* py_quantize_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n, 2);
    const at::Tensor& x0 = cuda_tensor(a[0], "x");
    const c10::cuda::CUDAGuard dev(x0.device());
    const int io = io_type(x0);
    const Tokens t(x0, PyObject_IsTrue(a[1]));
    at::Tensor q, scale;
    {
      const Unlocked unlocked;
      const at::Tensor x = x0.detach().contiguous();
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
        const at::Tensor q = int8_rows(q0.detach().reshape({-1, t.K}), ld), scale = f32(s0.detach());
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
        const at::Tensor x = x0.detach().contiguous();
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
