// Host side of the operators of the model (dion_amd/model_ops.py): argument checks, results, calls of the library, and the nodes of
// autograd.  Included by host.cpp, whose helpers it uses.  A call allocates its workspace from PyTorch's caching allocator on the
// current stream: calls on different streams share nothing.
//
// What computes takes tensors and throws Refused, without the interpreter: autograd calls it from threads that do not hold its lock.

struct OpsApi {
  decltype(&dion_amd_embedding) embedding;
  decltype(&dion_amd_embedding_grad_workspace_bytes) embedding_grad_bytes;
  decltype(&dion_amd_embedding_grad) embedding_grad;
  decltype(&dion_amd_qk_norm_rope) qk_norm_rope;
  decltype(&dion_amd_qk_norm_rope_grad_workspace_bytes) qk_norm_rope_grad_bytes;
  decltype(&dion_amd_qk_norm_rope_grad) qk_norm_rope_grad;
  decltype(&dion_amd_cross_entropy_workspace_bytes) cross_entropy_bytes;
  decltype(&dion_amd_cross_entropy) cross_entropy;
  decltype(&dion_amd_cross_entropy_grad) cross_entropy_grad;
} ops;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const char* op, const std::string& why) { throw Refused(std::string(op) + ": " + why); }

// The status of a call of the library.
void status(int rc, const char* what) {
  if (rc == 0) return;
  static const char* const why[] = {"bad argument", "alignment", "workspace too small", "unsupported dtype", "size beyond a documented limit"};
  throw Refused(std::string(what) + ": " +
                (rc < 0 && rc >= -5 ? std::string(why[-rc - 1]) + " (code " + std::to_string(rc) + ")" : "HIP error " + std::to_string(rc)));
}

// The interpreter lock is released, if this thread holds it, while the library is called.
struct Released {
  PyThreadState* saved = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
  ~Released() { if (saved) PyEval_RestoreThread(saved); }
};

int float_code(const at::Tensor& t, const char* op, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return DION_AMD_BF16;
  if (t.scalar_type() == at::kFloat) return DION_AMD_F32;
  refuse(op, std::string(name) + " must be bfloat16 or float32, got " + c10::toString(t.scalar_type()));
}

// A tensor that is only the outside of others (a DTensor) has no memory of its own; the values of one that waits to be negated (the
// imaginary part of a conjugate) are not those in its memory.
void plain(const at::Tensor& t, const char* op, const char* name) {
  if (t.unsafeGetTensorImpl()->is_python_dispatch() || !t.has_storage() || t.layout() != at::kStrided || t.is_neg() || t._is_zerotensor())
    refuse(op, std::string(name) + " must be a plain dense tensor (of a DTensor: its to_local())");
}

void on_gpu(const at::Tensor& t, const char* op, const char* name) {
  if (!t.is_cuda())
    refuse(op, std::string(name) + " is on " + t.device().str() + "; the MI355X kernels need a GPU tensor (no CPU fallback)");
  plain(t, op, name);
}

void same_device(const at::Tensor& t, const at::Tensor& first, const char* op, const char* name) {
  if (t.device() != first.device()) refuse(op, std::string(name) + " is on " + t.device().str() + ", not on " + first.device().str());
  plain(t, op, name);
}

int index_bits(const at::Tensor& t, const char* op, const char* name) {
  if (t.scalar_type() == at::kLong) return 64;
  if (t.scalar_type() == at::kInt) return 32;
  refuse(op, std::string(name) + " must be int64 or int32, got " + c10::toString(t.scalar_type()));
}

// A 2-D tensor whose rows lie at a pitch of at least their length, a copy where its own do not.
at::Tensor rows_of(const at::Tensor& t) {
  const bool fits = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
  return fits ? t : t.contiguous();
}
long long pitch(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// A tensor of the caller's is about to be written over: what autograd has kept of it must not go unnoticed.
void written(const at::Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

// Memory of the current device and stream for the length of a call: what is enqueued later on the stream may have it next.  (The
// allocator itself, without a tensor around it: 1 us less a call.)
at::DataPtr scratch(size_t nbytes) { return nbytes ? c10::hip::HIPCachingAllocator::get()->allocate(nbytes) : at::DataPtr(); }

// ---- embedding

at::Tensor run_embedding(const at::Tensor& weight, const at::Tensor& ids, float scale, at::ScalarType out_type) {
  static const char op[] = "embedding";
  on_gpu(weight, op, "weight");
  same_device(ids, weight, op, "tokens");
  if (weight.dim() != 2 || weight.numel() == 0) refuse(op, "weight must be a matrix with at least one row and column");
  const int wc = float_code(weight, op, "weight"), bits = index_bits(ids, op, "tokens");
  const at::Tensor w = rows_of(weight), t = ids.contiguous();
  const long long dim = w.size(1);
  if (dim > 0x7fffffff) refuse(op, "rows of 2^31 columns or more");
  std::vector<int64_t> sizes = ids.sizes().vec();
  sizes.push_back(dim);
  const c10::DeviceGuard guard(w.device());
  const at::Tensor out = at::empty(sizes, w.options().dtype(out_type));
  const int oc = float_code(out, op, "the result");
  int rc;
  {
    const Released released;
    rc = ops.embedding(w.data_ptr(), wc, pitch(w), w.size(0), (int)dim, t.data_ptr(), bits, t.numel(), out.data_ptr(), oc, dim, scale,
                       stream_of(w.device()));
  }
  status(rc, "dion_amd_embedding");
  return out;
}

// out: undefined, or the tensor to write
at::Tensor run_embedding_grad(const at::Tensor& grad, const at::Tensor& ids, long long vocab, long long padding, float scale,
                              at::ScalarType type, at::Tensor out, bool accumulate) {
  static const char op[] = "embedding_backward";
  on_gpu(grad, op, "grad");
  same_device(ids, grad, op, "tokens");
  const int gc = float_code(grad, op, "grad"), bits = index_bits(ids, op, "tokens");
  if (grad.dim() != ids.dim() + 1 || !grad.sizes().slice(0, ids.dim()).equals(ids.sizes()) || grad.size(-1) == 0)
    refuse(op, "grad must have the shape of tokens and a last dimension of at least one column");
  const long long dim = grad.size(-1);
  if (vocab <= 0 || dim > 0x7fffffff) refuse(op, "the table needs at least one row, and fewer than 2^31 columns");
  if (out.defined()) {
    on_gpu(out, op, "out");
    same_device(out, grad, op, "out");
    if (out.dim() != 2 || out.size(0) != vocab || out.size(1) != dim || (dim > 1 && out.stride(1) != 1) || (vocab > 1 && out.stride(0) < dim))
      refuse(op, "out must be (num_embeddings, columns) with contiguous rows");
    if (out.scalar_type() != type) refuse(op, "dtype is not that of out");
    for (const at::Tensor* t : {&grad, &ids}) {   // (tables with gaps may lie between the rows of others)
      const at::MemOverlapStatus over = at::get_overlap_status(out, *t);
      if (over == at::MemOverlapStatus::Full || over == at::MemOverlapStatus::Partial) refuse(op, "out and an input overlap");
    }
  } else if (accumulate) {
    refuse(op, "accumulate needs out");
  }
  const at::Tensor g = rows_of(grad.reshape({ids.numel(), dim})), t = ids.contiguous();
  const c10::DeviceGuard guard(grad.device());
  if (out.defined()) written(out);
  else out = at::empty({vocab, dim}, grad.options().dtype(type));
  const int wc = float_code(out, op, "the result");
  const size_t need = ops.embedding_grad_bytes(t.numel(), vocab, (int)dim);
  const at::DataPtr ws = scratch(need);
  int rc;
  {
    const Released released;
    rc = ops.embedding_grad(g.data_ptr(), gc, pitch(g), t.data_ptr(), bits, t.numel(), out.data_ptr(), wc, pitch(out), vocab, (int)dim,
                            padding, scale, accumulate, ws.get(), need, stream_of(grad.device()));
  }
  status(rc, "dion_amd_embedding_grad");
  return out;
}

// ---- norm and rotation of queries and keys

struct QkInputs {
  at::Tensor x[2], cos, sin, gain[2], positions;   // gains and positions may be undefined
  float eps;
  bool interleaved;
};

// Checked inputs as the library takes them; the tensors live as long as this does.
struct QkCall {
  at::Tensor x[2], gain[2], cos, sin, positions;
  long long batch, length, dim, rotary, pos_batch = 0;
  int code, gain_code = DION_AMD_F32, bits = 64;
  float eps;
  bool interleaved;
  dion_amd_heads heads[2] = {};

  // strides of a (batch, length, heads, dim) tensor with contiguous channels
  static void strides(const at::Tensor& t, long long& b, long long& l, long long& h) {
    b = t.stride(0);
    l = t.stride(1);
    h = t.stride(2);
  }
  static at::Tensor channels(const at::Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

  QkCall(const QkInputs& in, const char* op) : cos(in.cos), sin(in.sin), positions(in.positions), eps(in.eps), interleaved(in.interleaved) {
    static const char* const names[2] = {"q", "k"};
    static const char* const gain_names[2] = {"q_gain", "k_gain"};
    const at::Tensor& first = in.x[0];
    for (int w = 0; w < 2; ++w) {
      const at::Tensor& t = in.x[w];
      on_gpu(t, op, names[w]);
      same_device(t, first, op, names[w]);
      code = float_code(t, op, names[w]);
      if (t.dim() != 4) refuse(op, "q and k must be (batch, length, heads, channels)");
      if (t.scalar_type() != first.scalar_type() || t.size(0) != first.size(0) || t.size(1) != first.size(1) || t.size(3) != first.size(3))
        refuse(op, "q and k differ in dtype, batch, length or channels");
      x[w] = channels(t);
      strides(x[w], heads[w].x_batch, heads[w].x_token, heads[w].x_head);
      heads[w].x = x[w].data_ptr();
      if (t.size(2) > 0x7fffffff) refuse(op, "2^31 heads or more");
      heads[w].heads = (int)t.size(2);
    }
    batch = first.size(0); length = first.size(1); dim = first.size(3);
    if (dim < 1 || batch > 0x7fffffff || length > 0x7fffffff || dim > 0x7fffffff) refuse(op, "no channels, or a dimension of 2^31 or more");
    for (const at::Tensor* t : {&cos, &sin}) {
      same_device(*t, first, op, "cos or sin");
      if (t->dim() != 2 || t->scalar_type() != at::kFloat) refuse(op, "cos and sin must be float32 matrices (positions, rotary / 2)");
    }
    if (!cos.sizes().equals(sin.sizes())) refuse(op, "cos and sin differ in shape");
    rotary = 2 * cos.size(1);
    if (rotary > dim) refuse(op, "the tables turn more channels than a head has");
    cos = rows_of(cos);
    sin = rows_of(sin);
    if (pitch(cos) != pitch(sin)) {
      cos = cos.contiguous();
      sin = sin.contiguous();
    }
    if (cos.size(0) > 0x7fffffff) refuse(op, "more than 2^31 positions");
    for (int w = 0; w < 2; ++w) {
      if (!in.gain[w].defined()) continue;
      same_device(in.gain[w], first, op, gain_names[w]);
      gain_code = float_code(in.gain[w], op, gain_names[w]);
      if (in.gain[w].dim() != 1 || in.gain[w].size(0) != dim) refuse(op, std::string(gain_names[w]) + " must have one factor a channel");
      if (w && in.gain[0].defined() && in.gain[0].scalar_type() != in.gain[1].scalar_type()) refuse(op, "q_gain and k_gain differ in dtype");
      gain[w] = in.gain[w].contiguous();
      heads[w].gain = gain[w].data_ptr();
    }
    if (positions.defined()) {
      same_device(positions, first, op, "positions");
      bits = index_bits(positions, op, "positions");
      const bool shared = positions.dim() == 1 && positions.size(0) == length;
      if (!shared && !(positions.dim() == 2 && positions.size(0) == batch && positions.size(1) == length))
        refuse(op, "positions must be (length) or (batch, length)");
      if (length > 1 && positions.stride(-1) != 1) positions = positions.contiguous();
      pos_batch = shared || batch <= 1 ? 0 : positions.stride(0);
    } else if (rotary && length > cos.size(0)) {
      refuse(op, "the tables have fewer positions than the sequences");
    }
  }

  at::Tensor result(int w) {
    const at::Tensor y = at::empty(x[w].sizes(), x[w].options());
    strides(y, heads[w].y_batch, heads[w].y_token, heads[w].y_head);
    heads[w].y = y.data_ptr();
    return y;
  }
  const float* table(const at::Tensor& t) const { return rotary ? t.data_ptr<float>() : nullptr; }
  const void* pos() const { return positions.defined() ? positions.data_ptr() : nullptr; }
};

void run_qk_norm_rope(const QkInputs& in, at::Tensor (&out)[2]) {
  QkCall c(in, "qk_norm_rope");
  const c10::DeviceGuard guard(c.x[0].device());
  for (int w = 0; w < 2; ++w) out[w] = c.result(w);
  int rc;
  {
    const Released released;
    rc = ops.qk_norm_rope(&c.heads[0], &c.heads[1], (int)c.batch, (int)c.length, (int)c.dim, (int)c.rotary, c.interleaved, c.code,
                          c.gain_code, c.table(c.cos), c.table(c.sin), pitch(c.cos), (int)c.cos.size(0), c.pos(), c.bits, c.pos_batch,
                          c.eps, stream_of(c.x[0].device()));
  }
  status(rc, "dion_amd_qk_norm_rope");
}

// out: dq, dk, and of the gains that are there dq_gain, dk_gain
void run_qk_norm_rope_grad(const QkInputs& in, const at::Tensor (&dy)[2], at::Tensor (&out)[4]) {
  static const char op[] = "qk_norm_rope_backward";
  QkCall c(in, op);
  at::Tensor d[2];
  for (int w = 0; w < 2; ++w) {
    same_device(dy[w], c.x[0], op, w ? "dk" : "dq");
    if (!dy[w].sizes().equals(c.x[w].sizes()) || dy[w].scalar_type() != c.x[w].scalar_type())
      refuse(op, "dq and dk must have the shapes and the dtype of q and k");
    d[w] = QkCall::channels(dy[w]);
    QkCall::strides(d[w], c.heads[w].dy_batch, c.heads[w].dy_token, c.heads[w].dy_head);
    c.heads[w].dy = d[w].data_ptr();
  }
  const c10::DeviceGuard guard(c.x[0].device());
  size_t need = 0;
  for (int w = 0; w < 2; ++w) {
    out[w] = c.result(w);
    if (!c.gain[w].defined()) continue;
    out[2 + w] = at::empty_like(c.gain[w]);
    c.heads[w].dgain = out[2 + w].data_ptr();
    need = ops.qk_norm_rope_grad_bytes((int)c.batch, (int)c.length, (int)c.dim, c.heads[0].heads + c.heads[1].heads);
  }
  const at::DataPtr ws = scratch(need);
  int rc;
  {
    const Released released;
    rc = ops.qk_norm_rope_grad(&c.heads[0], &c.heads[1], (int)c.batch, (int)c.length, (int)c.dim, (int)c.rotary, c.interleaved, c.code,
                               c.gain_code, c.table(c.cos), c.table(c.sin), pitch(c.cos), (int)c.cos.size(0), c.pos(), c.bits,
                               c.pos_batch, c.eps, ws.get(), need, stream_of(c.x[0].device()));
  }
  status(rc, "dion_amd_qk_norm_rope_grad");
}

// ---- cross entropy

struct LossOptions {
  long long ignore;
  double cap;   // as the caller gave it: what float32 rounds to zero would be no cap
  float z_loss;
  int reduction;
};

struct LossCall {
  at::Tensor x, t;
  long long rows, vocab;
  int code, bits;
  LossCall(const at::Tensor& logits, const at::Tensor& targets, const LossOptions& o) {
    static const char op[] = "cross_entropy";
    on_gpu(logits, op, "logits");
    same_device(targets, logits, op, "targets");
    code = float_code(logits, op, "logits");
    bits = index_bits(targets, op, "targets");
    if (logits.dim() != targets.dim() + 1 || !logits.sizes().slice(0, targets.dim()).equals(targets.sizes()) || logits.size(-1) == 0)
      refuse(op, "logits must have the shape of targets and a last dimension of at least one class");
    vocab = logits.size(-1);
    rows = targets.numel();
    x = rows_of(logits.reshape({rows, vocab}));
    t = targets.contiguous();
    if (o.cap != 0.0 && !(o.cap >= 1e-30 && o.cap <= 1e30)) refuse(op, "softcap must be zero or a positive number between 1e-30 and 1e30");
  }
};

// out: loss; the rows' normalisers if `keep`; the gradient: `gradient` 0 none, 1 into a new tensor, 2 over the logits
void run_cross_entropy(const at::Tensor& logits, const at::Tensor& targets, const LossOptions& o, bool keep, int gradient, float scale,
                       at::Tensor (&out)[3]) {
  const LossCall c(logits, targets, o);
  const auto f32 = c.x.options().dtype(at::kFloat);
  const c10::DeviceGuard guard(c.x.device());
  out[0] = o.reduction == DION_AMD_REDUCE_NONE ? at::empty(targets.sizes(), f32) : at::empty({}, f32);
  if (keep) out[1] = at::empty({c.rows + 1}, f32);
  long long ldd = c.vocab;
  if (gradient == 1) {
    out[2] = at::empty(logits.sizes(), c.x.options());
  } else if (gradient == 2) {
    if (c.rows && c.x.data_ptr() != logits.data_ptr()) refuse("cross_entropy", "inplace needs logits whose rows lie at one pitch");
    out[2] = logits;
    ldd = pitch(c.x);
  }
  const size_t need = ops.cross_entropy_bytes(c.rows, c.vocab, c.code);
  const at::DataPtr ws = scratch(need);
  int rc;
  {
    const Released released;
    rc = ops.cross_entropy(c.x.data_ptr(), c.code, pitch(c.x), c.t.data_ptr(), c.bits, c.rows, c.vocab, o.ignore, (float)o.cap, o.z_loss,
                           o.reduction, out[0].data_ptr<float>(), keep ? out[1].data_ptr<float>() : nullptr,
                           gradient ? out[2].data_ptr() : nullptr, ldd, scale, ws.get(), need, stream_of(c.x.device()));
  }
  status(rc, "dion_amd_cross_entropy");
  if (gradient == 2) logits.unsafeGetTensorImpl()->bump_version();   // an earlier use of the logits must not go unnoticed
}

at::Tensor run_cross_entropy_grad(const at::Tensor& logits, const at::Tensor& targets, const LossOptions& o, const at::Tensor& lse,
                                  const at::Tensor& dloss) {
  const LossCall c(logits, targets, o);
  const at::Tensor d = dloss.to(at::kFloat).contiguous().resolve_neg();
  same_device(d, logits, "cross_entropy", "the upstream gradient");
  const c10::DeviceGuard guard(c.x.device());
  const at::Tensor out = at::empty(logits.sizes(), c.x.options());
  int rc;
  {
    const Released released;
    rc = ops.cross_entropy_grad(c.x.data_ptr(), c.code, pitch(c.x), c.t.data_ptr(), c.bits, c.rows, c.vocab, o.ignore, (float)o.cap, o.z_loss,
                                o.reduction, lse.data_ptr<float>(), d.data_ptr<float>(), out.data_ptr(), c.vocab,
                                stream_of(c.x.device()));
  }
  status(rc, "dion_amd_cross_entropy_grad");
  return out;
}

// ---- autograd: a node an operator, whose gradients are not differentiated again

using torch::autograd::SavedVariable;
using torch::autograd::collect_next_edges;
using torch::autograd::deleteNode;
using torch::autograd::edge_list;
using torch::autograd::set_history;
using torch::autograd::variable_list;

// A tangent would be lost.
void no_tangent(const at::Tensor& t, const std::string& op) {
  if (t.defined() && t._fw_grad(0).defined()) refuse(op.c_str(), "no gradient in forward mode");
}

struct OperatorNode : torch::autograd::Node {
  // the gradients of the inputs, from those of the outputs; called with gradients off
  virtual variable_list gradients(const variable_list& grads) = 0;
  // lets go of what was kept for them
  virtual void forget() = 0;

  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    forget();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (const at::Tensor& g : grads) no_tangent(g, name());
    const bool twice = at::GradMode::is_enabled();   // a graph of the gradients is wanted
    variable_list out;
    {
      const at::NoGradGuard no_grad;
      out = gradients(grads);
    }
    if (twice) {
      const std::shared_ptr<Node> error(new torch::autograd::Error(name() + " is not differentiable twice", edge_list(next_edges())), deleteNode);
      for (const at::Tensor& t : out)
        if (t.defined()) set_history(t, error);
    }
    return out;
  }
};

struct EmbeddingBackward : OperatorNode {
  SavedVariable tokens;
  long long vocab, padding;
  float scale;
  at::ScalarType type;
  std::string name() const override { return "EmbeddingBackward"; }
  void forget() override { tokens.reset_data(); }
  variable_list gradients(const variable_list& grads) override {
    if (!grads[0].defined()) return {at::Tensor()};
    return {run_embedding_grad(grads[0], tokens.unpack(), vocab, padding, scale, type, at::Tensor(), false)};
  }
};

struct QkNormRopeBackward : OperatorNode {
  SavedVariable x[2], cos, sin, gain[2], positions;
  float eps;
  bool interleaved;
  std::string name() const override { return "QkNormRopeBackward"; }
  void forget() override {
    for (SavedVariable* v : {x, x + 1, &cos, &sin, gain, gain + 1, &positions}) v->reset_data();
  }
  variable_list gradients(const variable_list& grads) override {
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
    const QkInputs in{{x[0].unpack(), x[1].unpack()}, cos.unpack(), sin.unpack(), {gain[0].unpack(), gain[1].unpack()}, positions.unpack(),
                      eps, interleaved};
    const at::Tensor dy[2] = {grads[0].defined() ? grads[0] : at::zeros_like(in.x[0]), grads[1].defined() ? grads[1] : at::zeros_like(in.x[1])};
    at::Tensor out[4];
    run_qk_norm_rope_grad(in, dy, out);
    return {out[0], out[1], out[2], out[3]};
  }
};

struct CrossEntropyBackward : OperatorNode {
  SavedVariable logits, targets, lse;
  LossOptions options;
  std::string name() const override { return "CrossEntropyBackward"; }
  void forget() override {
    for (SavedVariable* v : {&logits, &targets, &lse}) v->reset_data();
  }
  variable_list gradients(const variable_list& grads) override {
    if (!grads[0].defined()) return {at::Tensor()};
    return {run_cross_entropy_grad(logits.unpack(), targets.unpack(), options, lse.unpack(), grads[0])};
  }
};

template <typename N>
std::shared_ptr<N> make_node() { return {new N(), deleteNode}; }   // (a long graph is not taken down by recursion)

bool wants_grad(const char* op, std::initializer_list<const at::Tensor*> inputs) {
  bool wants = false;
  for (const at::Tensor* t : inputs) {
    no_tangent(*t, op);
    wants = wants || (t->defined() && t->requires_grad());
  }
  return wants && at::GradMode::is_enabled();
}

// ---- Python

const at::Tensor& tensor_arg(PyObject* o, const char* op, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: %s must be a tensor", op, name);
    throw Failed();
  }
  return THPVariable_Unpack(o);
}
// None stands for an undefined tensor.
at::Tensor optional_arg(PyObject* o, const char* op, const char* name) { return o == Py_None ? at::Tensor() : tensor_arg(o, op, name); }

at::ScalarType dtype_arg(PyObject* o, at::ScalarType fallback, const char* op) {
  if (o == Py_None) return fallback;
  if (!THPDtype_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: expected a torch.dtype", op);
    throw Failed();
  }
  const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  if (t != at::kBFloat16 && t != at::kFloat) refuse(op, std::string("the result is bfloat16 or float32, not ") + c10::toString(t));
  return t;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Failed();
  return v;
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Failed();
  return v == 1;
}

PyObject* wrap(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
template <size_t N>
PyObject* wrap_all(const at::Tensor (&ts)[N]) {
  PyObject* out = PyTuple_New(N);
  if (!out) throw Failed();
  for (size_t i = 0; i < N; ++i) {
    PyObject* o = wrap(ts[i]);
    if (!o) { Py_DECREF(out); throw Failed(); }
    PyTuple_SET_ITEM(out, (Py_ssize_t)i, o);
  }
  return out;
}

// Runs `body` with the exceptions of C++ turned into Python's: ATen's as its own operators do, those of Python (a hook's) as they are.
template <typename F>
PyObject* guarded(const char* op, Py_ssize_t want, Py_ssize_t got, F&& body) {
  if (want != got) {
    PyErr_Format(PyExc_TypeError, "%s: %zd arguments", op, want);
    return nullptr;
  }
  try {
    return body();
  } catch (const Failed&) {
  } catch (const Refused& e) {
    PyErr_SetString(g_error, e.what());
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// embedding(weight, tokens, scale, padding, out_dtype) -> out
PyObject* op_embedding(PyObject*, PyObject* const* a, Py_ssize_t na) {
  static const char op[] = "embedding";
  return guarded(op, 5, na, [&] {
    const at::Tensor &weight = tensor_arg(a[0], op, "weight"), &tokens = tensor_arg(a[1], op, "tokens");
    const float scale = (float)number(a[2]);
    const long long padding = integer(a[3]);
    const bool track = wants_grad(op, {&weight});
    at::Tensor out;
    {
      const at::NoGradGuard no_grad;
      out = run_embedding(weight, tokens, scale, dtype_arg(a[4], weight.scalar_type(), op));
    }
    if (track) {
      const auto node = make_node<EmbeddingBackward>();
      node->set_next_edges(collect_next_edges(weight));
      node->tokens = SavedVariable(tokens, false);
      node->vocab = weight.size(0);
      node->padding = padding;
      node->scale = scale;
      node->type = weight.scalar_type();
      set_history(out, node);
    }
    return wrap(out);
  });
}

// embedding_grad(grad, tokens, num_embeddings, padding, scale, dtype, out, accumulate) -> gradient of the table
PyObject* op_embedding_grad(PyObject*, PyObject* const* a, Py_ssize_t na) {
  static const char op[] = "embedding_backward";
  return guarded(op, 8, na, [&] {
    const at::NoGradGuard no_grad;
    const at::Tensor &grad = tensor_arg(a[0], op, "grad"), &tokens = tensor_arg(a[1], op, "tokens");
    const at::Tensor out = optional_arg(a[6], op, "out");
    for (const at::Tensor* t : {&grad, &out}) no_tangent(*t, op);
    const at::ScalarType type = dtype_arg(a[5], out.defined() ? out.scalar_type() : grad.scalar_type(), op);
    return wrap(run_embedding_grad(grad, tokens, integer(a[2]), integer(a[3]), (float)number(a[4]), type, out, truth(a[7])));
  });
}

// the arguments q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved
QkInputs qk_args(PyObject* const* a, const char* op) {
  return {{tensor_arg(a[0], op, "q"), tensor_arg(a[1], op, "k")}, tensor_arg(a[2], op, "cos"), tensor_arg(a[3], op, "sin"),
          {optional_arg(a[4], op, "q_gain"), optional_arg(a[5], op, "k_gain")}, optional_arg(a[6], op, "positions"), (float)number(a[7]),
          truth(a[8])};
}

// qk_norm_rope(q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved) -> (q, k)
PyObject* op_qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t na) {
  static const char op[] = "qk_norm_rope";
  return guarded(op, 9, na, [&] {
    const QkInputs in = qk_args(a, op);
    const bool track = wants_grad(op, {in.x, in.x + 1, in.gain, in.gain + 1});
    if (wants_grad(op, {&in.cos, &in.sin})) refuse(op, "cos and sin are constants, without a gradient of their own (detach them)");
    at::Tensor out[2];
    {
      const at::NoGradGuard no_grad;
      run_qk_norm_rope(in, out);
    }
    if (track) {
      const auto node = make_node<QkNormRopeBackward>();
      node->set_next_edges(collect_next_edges(in.x[0], in.x[1], in.gain[0], in.gain[1]));
      for (int w = 0; w < 2; ++w) {
        node->x[w] = SavedVariable(in.x[w], false);
        node->gain[w] = SavedVariable(in.gain[w], false);
      }
      node->cos = SavedVariable(in.cos, false);
      node->sin = SavedVariable(in.sin, false);
      node->positions = SavedVariable(in.positions, false);
      node->eps = in.eps;
      node->interleaved = in.interleaved;
      for (const at::Tensor& t : out) set_history(t, node);
    }
    return wrap_all(out);
  });
}

// qk_norm_rope_grad(q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved, dq, dk) -> (dq, dk, dq_gain, dk_gain)
PyObject* op_qk_norm_rope_grad(PyObject*, PyObject* const* a, Py_ssize_t na) {
  static const char op[] = "qk_norm_rope_backward";
  return guarded(op, 11, na, [&] {
    const at::NoGradGuard no_grad;
    const QkInputs in = qk_args(a, op);
    const at::Tensor dy[2] = {tensor_arg(a[9], op, "dq"), tensor_arg(a[10], op, "dk")};
    for (const at::Tensor* t : {in.x, in.x + 1, &in.cos, &in.sin, in.gain, in.gain + 1, dy, dy + 1}) no_tangent(*t, op);
    at::Tensor out[4];
    run_qk_norm_rope_grad(in, dy, out);
    return wrap_all(out);
  });
}

// the arguments ignore_index, softcap, z_loss, reduction
LossOptions loss_args(PyObject* const* a) { return {integer(a[0]), number(a[1]), (float)number(a[2]), (int)integer(a[3])}; }

// cross_entropy(logits, targets, ignore_index, softcap, z_loss, reduction) -> loss
PyObject* op_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t na) {
  static const char op[] = "cross_entropy";
  return guarded(op, 6, na, [&] {
    const at::Tensor &logits = tensor_arg(a[0], op, "logits"), &targets = tensor_arg(a[1], op, "targets");
    const LossOptions options = loss_args(a + 2);
    const bool track = wants_grad(op, {&logits});
    at::Tensor out[3];
    {
      const at::NoGradGuard no_grad;
      run_cross_entropy(logits, targets, options, track, 0, 1.f, out);
    }
    if (track) {
      const auto node = make_node<CrossEntropyBackward>();
      node->set_next_edges(collect_next_edges(logits));
      node->logits = SavedVariable(logits, false);
      node->targets = SavedVariable(targets, false);
      node->lse = SavedVariable(out[1], false);
      node->options = options;
      set_history(out[0], node);
    }
    return wrap(out[0]);
  });
}

// cross_entropy_with_grad(logits, targets, ignore_index, softcap, z_loss, reduction, grad_scale, inplace) -> (loss, dlogits)
PyObject* op_cross_entropy_with_grad(PyObject*, PyObject* const* a, Py_ssize_t na) {
  static const char op[] = "cross_entropy_with_grad";
  return guarded(op, 8, na, [&] {
    const at::NoGradGuard no_grad;
    const at::Tensor &logits = tensor_arg(a[0], op, "logits"), &targets = tensor_arg(a[1], op, "targets");
    const LossOptions options = loss_args(a + 2);
    const bool inplace = truth(a[7]);
    no_tangent(logits, op);
    at::Tensor out[3];
    // (the gradient is no part of the logits' graph, also where it takes their place)
    run_cross_entropy(inplace ? logits.detach() : logits, targets, options, false, inplace ? 2 : 1, (float)number(a[6]), out);
    const at::Tensor both[2] = {out[0], out[2]};
    return wrap_all(both);
  });
}

// bind_ops(addresses of the entry points in the order of OpsApi)
PyObject* bind_ops(PyObject*, PyObject* args) {
  unsigned long long f[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6, f + 7, f + 8)) return nullptr;
  ops.embedding = reinterpret_cast<decltype(ops.embedding)>(f[0]);
  ops.embedding_grad_bytes = reinterpret_cast<decltype(ops.embedding_grad_bytes)>(f[1]);
  ops.embedding_grad = reinterpret_cast<decltype(ops.embedding_grad)>(f[2]);
  ops.qk_norm_rope = reinterpret_cast<decltype(ops.qk_norm_rope)>(f[3]);
  ops.qk_norm_rope_grad_bytes = reinterpret_cast<decltype(ops.qk_norm_rope_grad_bytes)>(f[4]);
  ops.qk_norm_rope_grad = reinterpret_cast<decltype(ops.qk_norm_rope_grad)>(f[5]);
  ops.cross_entropy_bytes = reinterpret_cast<decltype(ops.cross_entropy_bytes)>(f[6]);
  ops.cross_entropy = reinterpret_cast<decltype(ops.cross_entropy)>(f[7]);
  ops.cross_entropy_grad = reinterpret_cast<decltype(ops.cross_entropy_grad)>(f[8]);
  Py_RETURN_NONE;
}
