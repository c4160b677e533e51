// Autograd nodes of the operators at a language model's ends (layer norm, embedding, distillation loss), in C++: their
// kernels take 5 to 30 us on small batches, and the same nodes as Python functions took 90 to 100 us of host time for a
// forward and a backward, of which about 50 went into calling a Python function from the engine and back.
// Arguments come checked (`ops/elementwise.py`, `ops/embedding.py`, `ops/top_logits.py`); memory comes from torch's
// allocator, the kernels run on the current stream, which in a backward the engine has set to the forward's.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <atomic>

extern "C" {
int pd_layer_norm_partial_rows(long long rows, int d);
int pd_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, long long rows, int d,
                      float eps, int x_fp32, int p_fp32, void* stream);
int pd_layer_norm_bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, void* dw,
                      void* db, float* partial, long long rows, int d, int x_fp32, int p_fp32, void* stream);
int pd_embedding(const void* tokens, int wide, const void* table, void* y, int* ids, long long n, long long V, int d,
                 float scale, int table_fp32, int y_fp32, int* status, int* refused, void* stream);
long long pd_embedding_grad_ints(long long n, long long V);
long long pd_embedding_grad_floats(long long n, int d);
int pd_embedding_grad(const int* ids, const void* dy, void* dE, long long n, long long V, int d, float scale, int dy_fp32,
                      int table_fp32, int* ints, float* partial, void* stream);
int pd_top_logits(const void* z, long long rows, int V, long long ld, int k, float inv_t, void* values, int* indices,
                  float* tail, int z_fp32, int* status, void* stream);
int pd_top_kl(const void* z, long long rows, int V, long long ld, const void* indices, int wide, const void* values,
              int values_fp32, int K, const float* tail, double inv_t, float* loss, void* dz, long long ldo,
              const float* scale, float* sums, const float* known, int z_fp32, int* status, int* refused, void* stream);
}

namespace {

using at::Tensor;
using torch::autograd::edge_list;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

std::atomic<long long> launches{0};

void* current_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
void check(int rc, const char* what, int kernels = 1) {
  launches += kernels;
  TORCH_CHECK(rc == 0, what, " failed to launch (code ", rc, ")");
}
bool fp32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
const void* at_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* data_or_null(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor given(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
Tensor floats(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }

// The kernels' gradients are not differentiable again: a second derivative with respect to what `node` has its edges to
// raises, where it would otherwise lack a term.
variable_list once(variable_list grads, const Node& node, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  std::shared_ptr<Node> error(
      new torch::autograd::Error(std::string(what) + " is not differentiable twice", edge_list(node.next_edges())),
      torch::autograd::deleteNode);
  for (Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, error);
  return grads;
}
template <typename N, typename... T>
std::shared_ptr<N> node_of(const T&... inputs) {
  std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}
template <typename... T>
bool wanted(const T&... inputs) {
  for (const Tensor& t : {inputs...})
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t), "the kernels have no forward-mode derivative");
  return at::GradMode::is_enabled() && torch::autograd::any_variable_requires_grad(variable_list{inputs...});
}

// ---- layer norm

struct LayerNormBackward : Node {
  SavedVariable x, w;
  Tensor stats;
  at::ScalarType p_type;

  std::string name() const override { return "LayerNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    w.reset_data();
    stats.reset();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(3);
    const Tensor x_back = x.unpack(), w_back = w.unpack();
    Tensor dx, dw, db;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor xs = dense(x_back), ws = dense(w_back);  // what a saved-tensor hook gives back may lie otherwise
      const int d = static_cast<int>(xs.size(-1));
      const long long rows = xs.numel() / d;
      const auto p_options = xs.options().dtype(p_type);
      if (task_should_compute_output(0)) dx = at::empty(xs.sizes(), xs.options());
      if (task_should_compute_output(1)) dw = at::empty({d}, p_options);
      if (task_should_compute_output(2)) db = at::empty({d}, p_options);
      if (rows > 0) {
        const Tensor dy = grads[0].contiguous();
        const bool params = dw.defined() || db.defined();
        const Tensor partial = params ? floats({pd_layer_norm_partial_rows(rows, d), 2, d}, xs) : Tensor();
        const float* mean = stats.const_data_ptr<float>();
        check(pd_layer_norm_bwd(xs.const_data_ptr(), at_or_null(ws), dy.const_data_ptr(), mean, mean + rows, data_or_null(dx),
                                data_or_null(dw), data_or_null(db), static_cast<float*>(data_or_null(partial)), rows, d,
                                fp32(xs), p_type == at::kFloat, current_stream()),
              "layer_norm_bwd", params ? 2 : 1);
      } else {
        for (const Tensor& g : {dw, db})
          if (g.defined()) g.zero_();
      }
    }
    return once({dx, dw, db}, *this, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x_in, const std::optional<Tensor>& w_in, const std::optional<Tensor>& b_in, double eps) {
  const Tensor w_var = given(w_in), b_var = given(b_in);
  std::shared_ptr<LayerNormBackward> node;
  if (wanted(x_in, w_var, b_var)) node = node_of<LayerNormBackward>(x_in, w_var, b_var);
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor x = x_in.contiguous(), w = dense(w_var), b = dense(b_var);
    const int d = static_cast<int>(x.size(-1));
    const long long rows = x.numel() / d;
    y = at::empty(x.sizes(), x.options());
    Tensor stats;
    if (node) stats = floats({2, rows}, x);
    const at::ScalarType p_type = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
    if (rows > 0) {
      float* mean = node ? stats.mutable_data_ptr<float>() : nullptr;
      check(pd_layer_norm_fwd(x.const_data_ptr(), at_or_null(w), at_or_null(b), y.mutable_data_ptr(), mean,
                              node ? mean + rows : nullptr, rows, d, static_cast<float>(eps), fp32(x), p_type == at::kFloat,
                              current_stream()),
            "layer_norm_fwd");
    }
    if (node) {
      node->x = SavedVariable(x, false);
      node->w = SavedVariable(w, false);
      node->stats = stats;
      node->p_type = p_type;
    }
  }
  if (node) torch::autograd::set_history(y, node);
  return y;
}

// ---- embedding

struct EmbeddingBackward : Node {
  Tensor ids;
  long long rows;
  double scale;
  at::ScalarType type;

  std::string name() const override { return "EmbeddingBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids.reset();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    TORCH_CHECK(ids.defined(), "embedding: its saved tokens have been freed (a second backward needs retain_graph=True)");
    Tensor dE;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor dy = grads[0].contiguous();
      const int d = static_cast<int>(dy.size(-1));
      const long long n = ids.numel(), whole = pd_embedding_grad_floats(n, d);
      dE = at::empty({rows, d}, dy.options().dtype(type));
      const Tensor scratch = floats({whole + pd_embedding_grad_ints(n, rows)}, dy);
      float* partial = scratch.mutable_data_ptr<float>();
      check(pd_embedding_grad(ids.const_data_ptr<int>(), dy.const_data_ptr(), dE.mutable_data_ptr(), n, rows, d,
                              static_cast<float>(scale), fp32(dy), type == at::kFloat, reinterpret_cast<int*>(partial + whole),
                              partial, current_stream()),
            "embedding_grad", 2);
    }
    return once({dE}, *this, "embedding");
  }
};

Tensor embedding(const Tensor& tokens_in, const Tensor& table_in, double scale, bool out_fp32, int64_t status, int64_t refused) {
  std::shared_ptr<EmbeddingBackward> node;
  if (wanted(table_in)) node = node_of<EmbeddingBackward>(table_in);
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor tokens = tokens_in.contiguous(), table = table_in.contiguous();
    const long long n = tokens.numel(), rows = table.size(0);
    const int d = static_cast<int>(table.size(1));
    c10::SmallVector<int64_t, 4> sizes(tokens.sizes().begin(), tokens.sizes().end());
    sizes.push_back(d);
    y = at::empty(sizes, table.options().dtype(out_fp32 ? at::kFloat : at::kBFloat16));
    Tensor ids;
    if (node) ids = at::empty({n}, table.options().dtype(at::kInt));
    if (n > 0)
      check(pd_embedding(tokens.const_data_ptr(), tokens.scalar_type() == at::kLong, table.const_data_ptr(),
                         y.mutable_data_ptr(), node ? ids.mutable_data_ptr<int>() : nullptr, n, rows, d,
                         static_cast<float>(scale), fp32(table), out_fp32, reinterpret_cast<int*>(status),
                         reinterpret_cast<int*>(refused), current_stream()),
            "embedding");
    if (node) {
      node->ids = ids;
      node->rows = rows;
      node->scale = scale;
      node->type = table.scalar_type();
    }
  }
  if (node) torch::autograd::set_history(y, node);
  return y;
}

// ---- top logits and distillation loss

// [rows, V] whose rows start at the same address modulo 16 bytes as the rows of z.
Tensor grad_like(const Tensor& z, long long pitch_in) {
  const long long size = z.element_size(), per = 16 / size, rows = z.size(0), V = z.size(1);
  const long long pitch = V + (pitch_in - V) % per;
  const long long first = static_cast<long long>(reinterpret_cast<uintptr_t>(z.const_data_ptr()) % 16) / size;
  return at::empty({first + rows * pitch}, z.options()).as_strided({rows, V}, {pitch, 1}, first);
}
// A single row's stride may be anything; where it is that of a padded matrix, the gradient is laid out like it too: products
// that read it want rows of whole 16 bytes, of one row as of many.
long long pitch_of(const Tensor& z) { return z.size(0) > 1 || z.stride(0) > z.size(1) ? z.stride(0) : z.size(1); }

// Neighbouring columns, rows that do not overlap.
bool in_rows(const Tensor& z) {
  return (z.size(1) == 1 || z.stride(1) == 1) && (z.size(0) <= 1 || z.stride(0) >= z.size(1));
}

// z [rows, V], neighbouring columns; the results in the shape `lead`, which holds as many rows.
std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& z, std::vector<int64_t> lead, int64_t k, double temperature,
                                              int64_t status) {
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor tail = floats(lead, z);
  lead.push_back(k);
  const Tensor values = at::empty(lead, z.options()), indices = at::empty(lead, z.options().dtype(at::kInt));
  if (z.size(0) > 0)
    check(pd_top_logits(z.const_data_ptr(), z.size(0), static_cast<int>(z.size(1)), pitch_of(z), static_cast<int>(k),
                        static_cast<float>(1.0 / temperature), values.mutable_data_ptr(), indices.mutable_data_ptr<int>(),
                        tail.mutable_data_ptr<float>(), fp32(z), reinterpret_cast<int*>(status), current_stream()),
          "top_logits");
  return {values, indices, tail};
}

struct Teacher {
  Tensor indices, values, tail;
  double temperature;
  int64_t status, refused;
};
void run_top_kl(const Tensor& z, const Teacher& t, const Tensor& loss, const Tensor& dz, const Tensor& scale,
                const Tensor& sums, const Tensor& known) {
  if (z.size(0) == 0) return;
  check(pd_top_kl(z.const_data_ptr(), z.size(0), static_cast<int>(z.size(1)), pitch_of(z), t.indices.const_data_ptr(),
                  t.indices.scalar_type() == at::kLong, t.values.const_data_ptr(), fp32(t.values),
                  static_cast<int>(t.indices.size(1)), static_cast<const float*>(at_or_null(t.tail)), 1.0 / t.temperature,
                  static_cast<float*>(data_or_null(loss)), data_or_null(dz), dz.defined() ? dz.stride(0) : 0,
                  static_cast<const float*>(at_or_null(scale)),
                  static_cast<float*>(data_or_null(sums)), static_cast<const float*>(at_or_null(known)), fp32(z),
                  reinterpret_cast<int*>(t.status),
                  reinterpret_cast<int*>(t.refused), current_stream()),
        "top_kl");
}

// The backward reads the logits again, with the rows' sums that the forward kept: 2 reads and a write of the logits for
// both passes, against a read and two writes had the forward kept an unscaled gradient.
struct TopKLBackward : Node {
  SavedVariable z, indices, values, tail;
  Tensor sums;
  double temperature;
  int64_t status, refused;

  std::string name() const override { return "TopKLBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&z, &indices, &values, &tail}) s->reset_data();
    sums.reset();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    const Tensor z_back = z.unpack(), indices_back = indices.unpack(), values_back = values.unpack(), tail_back = tail.unpack();
    Tensor dz;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      // what a saved-tensor hook gives back may lie otherwise than what was saved
      const Tensor zs = in_rows(z_back) ? z_back : z_back.contiguous();
      const Teacher t{dense(indices_back), dense(values_back), dense(tail_back), temperature, status, refused};
      dz = grad_like(zs, pitch_of(zs));
      run_top_kl(zs, t, Tensor(), dz, grads[0].contiguous(), Tensor(), sums);
    }
    return once({dz}, *this, "top_kl");
  }
};

// z [rows, V], neighbouring columns; indices, values [rows, K] and tail [rows] contiguous.
Tensor top_kl(const Tensor& z, const Tensor& indices, const Tensor& values, const std::optional<Tensor>& tail,
              double temperature, int64_t status, int64_t refused) {
  std::shared_ptr<TopKLBackward> node;
  if (wanted(z)) node = node_of<TopKLBackward>(z);
  const Teacher t{indices, values, given(tail), temperature, status, refused};
  Tensor loss;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    loss = floats({z.size(0)}, z);
    if (node) node->sums = floats({z.size(0), 4}, z);
    run_top_kl(z, t, loss, Tensor(), Tensor(), node ? node->sums : Tensor(), Tensor());
  }
  if (node) {
    node->z = SavedVariable(z, false);
    node->indices = SavedVariable(indices, false);
    node->values = SavedVariable(values, false);
    node->tail = SavedVariable(t.tail, false);
    node->temperature = temperature;
    node->status = status;
    node->refused = refused;
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

std::tuple<Tensor, Tensor> top_kl_rows(const Tensor& z, const Tensor& indices, const Tensor& values,
                                       const std::optional<Tensor>& tail, double temperature, bool want_grad, int64_t status,
                                       int64_t refused) {
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor loss = floats({z.size(0)}, z), dz = want_grad ? grad_like(z, pitch_of(z)) : Tensor();
  run_top_kl(z, Teacher{indices, values, given(tail), temperature, status, refused}, loss, dz, Tensor(),
             Tensor(), Tensor());
  return {loss, dz};
}

}  // namespace

PYBIND11_MODULE(pd_autograd, m) {
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("layer_norm", &layer_norm, free);
  m.def("embedding", &embedding, free);
  m.def("top_logits", &top_logits, free);
  m.def("top_kl", &top_kl, free);
  m.def("top_kl_rows", &top_kl_rows, free);
  m.def("launches", [] { return launches.load(); });
}
