// PyTorch side of the token operators: layer norm, three-axis rotary positions, cross attention.  Autograd nodes, argument
// checks and allocations over the C ABI, as torch_ops.cpp has them for the convolutions.
#include <array>
#include <mutex>

#include "torch_common.h"

namespace d2c_torch {
namespace {

int token_dtype(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat: return D2C_F32;
    case at::kHalf: return D2C_F16;
    case at::kBFloat16: return D2C_BF16;
    default: TORCH_CHECK(false, "\"", op, "\" not implemented for '", t.scalar_type(), "'");
  }
}

void same_device(const char* op, const Tensor& a, const Tensor& b, const char* name) {
  TORCH_CHECK(!b.defined() || b.device() == a.device(), op, ": expected ", name, " on ", a.device(), " but found it on ",
              b.defined() ? b.device() : a.device());
}

// ---- layer norm ---------------------------------------------------------------------------------------------

struct LayerNormNode : public Node {
  d2c_layer_norm_desc desc;
  bool has_bias, empty;
  at::TensorOptions param_options;
  std::vector<int64_t> shape;
  Saved x, weight;
  Tensor stats;

  std::string name() const override { return "D2CLayerNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x.reset(); weight.reset();
    stats = Tensor();
  }

  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return variable_list(3);
    Tensor xv, wv, sv, gx, gw, gb;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      xv = x.unpack(); wv = weight.unpack();
      sv = stats;
    }
    {
      at::AutoGradMode no_grad(false);
      c10::cuda::CUDAGuard guard(xv.device());
      xv = xv.contiguous(); wv = contiguous(wv);
      if (task_should_compute_output(0)) gx = at::empty(shape, xv.options().requires_grad(false));
      if (wv.defined() && task_should_compute_output(1)) gw = at::empty({desc.channels}, param_options);
      if (has_bias && task_should_compute_output(2)) gb = at::empty({desc.channels}, param_options);
      if (empty) {
        if (gw.defined()) gw.zero_();
        if (gb.defined()) gb.zero_();
      } else {
        const Tensor gy = grads[0].contiguous();
        const size_t n = gw.defined() || gb.defined() ? d2c_layer_norm_bwd_workspace_bytes(&desc) : 0;
        const Tensor ws = bytes_on(n, xv);
        check(d2c_layer_norm_bwd(&desc, ptr(gy), ptr(xv), ptr(wv), ptr(sv), ptr(gx), ptr(gw), ptr(gb), ptr(ws), n,
                                 stream_of(xv)), "layer_norm backward");
      }
    }
    return once_differentiable({gx, gw, gb});
  }
};

Tensor layer_norm(const Tensor& input, const OptTensor& weight_, const OptTensor& bias_, double eps, int64_t layout) {
  const Tensor weight = get(weight_), bias = get(bias_);
  refuse_tangents("layer_norm", {&input, &weight, &bias});
  D2C_REQUIRE(input.is_cuda(), "input.device().is_cuda()");
  same_device("layer_norm", input, weight, "weight");
  same_device("layer_norm", input, bias, "bias");
  d2c_layer_norm_desc d{};
  d.dtype = token_dtype(input, "layer_norm");
  d.layout = (int32_t)layout;
  d.eps = (float)eps;
  const bool rows = layout == D2C_NORM_ROWS;
  TORCH_CHECK(rows ? input.dim() >= 1 : input.dim() >= 2, "layer_norm: input has too few dimensions, got ", input.sizes());
  const int64_t channels = input.size(rows ? -1 : 1);
  TORCH_CHECK(channels > 0 && channels <= 0x7fffffff, "layer_norm: bad number of channels, got ", input.sizes());
  for (const Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->dim() == 1 && t->size(0) == channels, "layer_norm: weight and bias must be [", channels, "], got ", t->sizes());
    TORCH_CHECK(t->scalar_type() == at::kFloat || t->scalar_type() == input.scalar_type(),
                "layer_norm: weight and bias must be float32 or of the input's type, got ", t->scalar_type());
  }
  TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
              "layer_norm: weight and bias must have the same type");
  const Tensor& p = weight.defined() ? weight : bias;
  d.param_dtype = p.defined() ? token_dtype(p, "layer_norm") : d.dtype;
  d.channels = (int32_t)channels;
  int64_t batch = 1, positions = 1;
  if (rows) {
    positions = input.numel() / channels;
  } else {
    batch = input.size(0);
    for (int64_t i = 2; i < input.dim(); ++i) positions *= input.size(i);
  }
  const bool empty = input.numel() == 0;
  TORCH_CHECK(batch <= 0x7fffffff, "layer_norm: batch too large");
  d.batch = (int32_t)batch;
  d.positions = positions;
  std::vector<int64_t> out = layout == D2C_NORM_VOLUME_TO_ROWS ? std::vector<int64_t>{batch, positions, channels}
                                                               : input.sizes().vec();
  const bool record = torch::autograd::compute_requires_grad(input, weight, bias);
  Tensor x, w, b, y, stats;
  {
    at::AutoGradMode no_grad(false);
    c10::cuda::CUDAGuard guard(input.device());
    x = input.contiguous(); w = contiguous(weight); b = contiguous(bias);
    y = at::empty(out, x.options().requires_grad(false));
    if (!empty) {
      if (record) stats = at::empty({batch * positions, 2}, x.options().dtype(at::kFloat).requires_grad(false));
      check(d2c_layer_norm_fwd(&d, ptr(x), ptr(w), ptr(b), ptr(y), ptr(stats), stream_of(x)), "layer_norm forward");
    }
  }
  if (record) {
    auto node = std::shared_ptr<LayerNormNode>(new LayerNormNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(input, weight, bias));
    node->desc = d; node->has_bias = bias.defined(); node->empty = empty;
    node->shape = input.sizes().vec();
    if (p.defined()) node->param_options = p.options().requires_grad(false);
    node->x = Saved(x, false);
    if (w.defined()) node->weight = Saved(w, false);
    node->stats = stats;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- rotary positions -----------------------------------------------------------------------------------------

struct Rotary {
  d2c_rotary_desc desc;
  Tensor positions;
};

// Dimensions of one element have no stride that matters.
int64_t stride_or_zero(const Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

Tensor rotate(const Tensor& input, Rotary r, bool inverse) {
  Tensor x = input;
  const int64_t pair = r.desc.interleaved ? 2 : 1;
  auto fits = [&](const Tensor& t) {
    if (t.size(3) > 1 && t.stride(3) != 1) return false;
    for (int64_t d = 0; d < 3; ++d)
      if (stride_or_zero(t, d) % pair) return false;
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % (pair * t.element_size()) == 0;
  };
  if (!fits(x)) x = x.clone(at::MemoryFormat::Contiguous);
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  if (x.numel() == 0) return y;
  r.desc.stride_batch = stride_or_zero(x, 0);
  r.desc.stride_token = stride_or_zero(x, 1);
  r.desc.stride_head = stride_or_zero(x, 2);
  r.desc.inverse = inverse;
  check(d2c_rotary(&r.desc, ptr(x), ptr(r.positions), ptr(y), stream_of(x)), "rotary_embedding_3d");
  return y;
}

struct RotaryNode : public Node {
  d2c_rotary_desc desc;
  Saved positions;

  std::string name() const override { return "D2CRotaryEmbedding3dBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    positions.reset();
  }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return variable_list(1);
    Rotary r{desc, Tensor()};
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      r.positions = positions.unpack();
    }
    Tensor gx;
    {
      at::AutoGradMode no_grad(false);
      c10::cuda::CUDAGuard guard(grads[0].device());
      r.positions = contiguous(r.positions);
      gx = rotate(grads[0], r, true);
    }
    return once_differentiable({gx});
  }
};

Tensor rotary(const Tensor& x, const OptTensor& positions_, const std::array<int64_t, 3>& grid, const std::array<double, 3>& step,
              const std::array<int64_t, 3>& axis_dims, double base, bool interleaved) {
  const Tensor positions = get(positions_);
  refuse_tangents("rotary_embedding_3d", {&x, &positions});
  D2C_REQUIRE(x.is_cuda(), "x.device().is_cuda()");
  D2C_REQUIRE(x.dim() == 4, "x.ndimension() == 4");
  Rotary r{};
  d2c_rotary_desc& d = r.desc;
  d.dtype = token_dtype(x, "rotary_embedding_3d");
  for (int64_t i = 0; i < 4; ++i) TORCH_CHECK(x.size(i) <= 0x7fffffff, "rotary_embedding_3d: x too large");
  d.batch = (int32_t)x.size(0); d.length = (int32_t)x.size(1); d.heads = (int32_t)x.size(2); d.dim = (int32_t)x.size(3);
  int64_t sum = 0;
  for (int k = 0; k < 3; ++k) {
    TORCH_CHECK(axis_dims[k] >= 0 && axis_dims[k] % 2 == 0 && axis_dims[k] <= x.size(3),
                "rotary_embedding_3d: axis_dims must be even and not negative, got ", axis_dims[k]);
    sum += axis_dims[k];
    d.axis_dims[k] = (int32_t)axis_dims[k];
  }
  TORCH_CHECK(sum <= x.size(3), "rotary_embedding_3d: axis_dims take ", sum, " channels of a head's ", x.size(3));
  TORCH_CHECK(x.size(3) % 2 == 0 && x.size(3) >= 2 && x.size(3) <= 512, "rotary_embedding_3d: a head has an even number of channels up to 512, got ",
              x.size(3));
  TORCH_CHECK(base > 0, "rotary_embedding_3d: base must be positive");
  d.base = base;
  d.interleaved = interleaved;
  if (positions.defined()) {
    same_device("rotary_embedding_3d", x, positions, "positions");
    TORCH_CHECK((positions.dim() == 2 || (positions.dim() == 3 && (positions.size(0) == x.size(0) || positions.size(0) == 1))) &&
                    positions.size(-2) == x.size(1) && positions.size(-1) == 3,
                "rotary_embedding_3d: positions must be [", x.size(1), ", 3] or [", x.size(0), ", ", x.size(1), ", 3], got ",
                positions.sizes());
    switch (positions.scalar_type()) {
      case at::kInt: d.pos_kind = D2C_POS_I32; break;
      case at::kLong: d.pos_kind = D2C_POS_I64; break;
      case at::kFloat: d.pos_kind = D2C_POS_F32; break;
      default: TORCH_CHECK(false, "rotary_embedding_3d: positions must be int32, int64 or float32, got ", positions.scalar_type());
    }
    TORCH_CHECK(!positions.requires_grad(), "rotary_embedding_3d: not differentiable in positions");
    d.pos_batch_stride = positions.dim() == 3 && positions.size(0) > 1 ? x.size(1) * 3 : 0;
  } else {
    int64_t n = 1;
    for (int k = 0; k < 3; ++k) {
      TORCH_CHECK(grid[k] >= 0 && grid[k] <= 0x7fffffff, "rotary_embedding_3d: bad grid");
      n *= grid[k];
      TORCH_CHECK(n <= 0x7fffffff, "rotary_embedding_3d: bad grid");
      d.grid[k] = (int32_t)grid[k];
      d.grid_step[k] = step[k];
    }
    TORCH_CHECK(n == x.size(1), "rotary_embedding_3d: a grid of ", n, " positions for ", x.size(1), " tokens");
    d.pos_kind = D2C_POS_GRID;
  }
  const bool record = torch::autograd::compute_requires_grad(x);
  Tensor y;
  {
    at::AutoGradMode no_grad(false);
    c10::cuda::CUDAGuard guard(x.device());
    r.positions = contiguous(positions);
    y = rotate(x, r, false);
  }
  if (record) {
    auto node = std::shared_ptr<RotaryNode>(new RotaryNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->desc = d;
    if (r.positions.defined()) node->positions = Saved(r.positions, false);
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- cross attention --------------------------------------------------------------------------------------------

// [B, L, H, D] with contiguous channels; any strides otherwise, but where the fast kernels could read a head's rows 16 bytes at a
// time if they were laid out so (or if a repeated dimension were written out), they are: a copy costs less than the slow kernels.
Tensor attention_rows(const Tensor& t) {
  if (t.size(3) > 1 && t.stride(3) != 1) return t.contiguous();
  const int64_t piece = 16 / t.element_size();
  if (t.size(3) % piece) return t;
  bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d < 3; ++d) fits &= t.size(d) == 1 || (t.stride(d) > 0 && t.stride(d) % piece == 0);
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
void take_strides(int64_t (&out)[3], const Tensor& t) {
  for (int64_t d = 0; d < 3; ++d) out[d] = stride_or_zero(t, d);
}

struct AttentionNode : public Node {
  d2c_attention_desc desc;
  bool empty;
  Saved q, k, v, lengths, o;
  Tensor lse;

  std::string name() const override { return "D2CCrossAttentionBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    q.reset(); k.reset(); v.reset(); lengths.reset(); o.reset();
    lse = Tensor();
  }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return variable_list(3);
    Tensor qv, kv, vv, nv, ov, lv, gq, gk, gv;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      qv = q.unpack(); kv = k.unpack(); vv = v.unpack(); nv = lengths.unpack(); ov = o.unpack(shared_from_this());
      lv = lse;
    }
    {
      at::AutoGradMode no_grad(false);
      c10::cuda::CUDAGuard guard(qv.device());
      // saved-tensor hooks may have laid the tensors out anew: the strides are those of what came back
      qv = attention_rows(qv); kv = attention_rows(kv); vv = attention_rows(vv); nv = contiguous(nv); ov = ov.contiguous();
      gq = at::empty(qv.sizes(), qv.options().requires_grad(false));
      gk = at::empty(kv.sizes(), kv.options().requires_grad(false));
      gv = at::empty(vv.sizes(), vv.options().requires_grad(false));
      if (empty) {
        gq.zero_(); gk.zero_(); gv.zero_();
      } else {
        const Tensor g = attention_rows(grads[0]);
        d2c_attention_desc d = desc;
        take_strides(d.q_stride, qv); take_strides(d.k_stride, kv); take_strides(d.v_stride, vv); take_strides(d.g_stride, g);
        const size_t n = d2c_attention_bwd_workspace_bytes(&d);
        const Tensor ws = bytes_on(n, qv);
        check(d2c_attention_bwd(&d, ptr(g), ptr(qv), ptr(kv), ptr(vv), ptr(nv), ptr(ov), ptr(lv), ptr(gq), ptr(gk), ptr(gv),
                                ptr(ws), n, stream_of(qv)), "cross_attention backward");
      }
    }
    return once_differentiable({gq, gk, gv});
  }
};

Tensor cross_attention(const Tensor& query, const Tensor& key, const Tensor& value, const OptTensor& lengths_, double scale) {
  const Tensor lengths = get(lengths_);
  refuse_tangents("cross_attention", {&query, &key, &value});
  D2C_REQUIRE(query.is_cuda(), "query.device().is_cuda()");
  D2C_REQUIRE(query.dim() == 4, "query.ndimension() == 4");
  D2C_REQUIRE(key.dim() == 4, "key.ndimension() == 4");
  same_device("cross_attention", query, key, "key");
  same_device("cross_attention", query, value, "value");
  same_device("cross_attention", query, lengths, "key_lengths");
  TORCH_CHECK(key.scalar_type() == query.scalar_type() && value.scalar_type() == query.scalar_type(),
              "cross_attention: query, key and value must have the same type");
  TORCH_CHECK(key.size(0) == query.size(0) && key.size(3) == query.size(3), "cross_attention: key ", key.sizes(),
              " does not match query ", query.sizes());
  TORCH_CHECK(value.sizes() == key.sizes(), "cross_attention: value ", value.sizes(), " does not match key ", key.sizes());
  TORCH_CHECK(key.size(2) > 0 && query.size(2) > 0 && query.size(2) % key.size(2) == 0, "cross_attention: ", query.size(2),
              " query heads cannot share ", key.size(2), " key heads");
  TORCH_CHECK(query.size(3) >= 1 && query.size(3) <= 128, "cross_attention: a head has 1 to 128 channels, got ", query.size(3));
  if (lengths.defined()) {
    TORCH_CHECK(lengths.dim() == 1 && lengths.size(0) == query.size(0), "cross_attention: key_lengths must be [", query.size(0),
                "], got ", lengths.sizes());
    TORCH_CHECK(lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong,
                "cross_attention: key_lengths must be int32 or int64, got ", lengths.scalar_type());
  }
  d2c_attention_desc d{};
  d.dtype = token_dtype(query, "cross_attention");
  for (const Tensor* t : {&query, &key})
    for (int64_t i = 0; i < 4; ++i) TORCH_CHECK(t->size(i) <= 0x7fffffff, "cross_attention: tensor too large");
  d.batch = (int32_t)query.size(0); d.queries = (int32_t)query.size(1); d.keys = (int32_t)key.size(1);
  d.q_heads = (int32_t)query.size(2); d.kv_heads = (int32_t)key.size(2); d.dim = (int32_t)query.size(3);
  d.lengths_i64 = lengths.defined() && lengths.scalar_type() == at::kLong;
  d.scale = (float)scale;
  const bool empty = query.numel() == 0 || key.numel() == 0;
  const bool record = torch::autograd::compute_requires_grad(query, key, value);
  Tensor q, k, v, n, o, lse;
  {
    at::AutoGradMode no_grad(false);
    c10::cuda::CUDAGuard guard(query.device());
    q = attention_rows(query); k = attention_rows(key); v = attention_rows(value); n = contiguous(lengths);
    take_strides(d.q_stride, q); take_strides(d.k_stride, k); take_strides(d.v_stride, v);
    o = at::empty(query.sizes(), query.options().requires_grad(false));
    if (empty) {
      o.zero_();
    } else {
      if (record) lse = at::empty({d.batch, d.q_heads, d.queries}, q.options().dtype(at::kFloat).requires_grad(false));
      const size_t bytes = d2c_attention_fwd_workspace_bytes(&d);
      const Tensor ws = bytes_on(bytes, q);
      check(d2c_attention_fwd(&d, ptr(q), ptr(k), ptr(v), ptr(n), ptr(o), ptr(lse), ptr(ws), bytes, stream_of(q)),
            "cross_attention forward");
    }
  }
  if (record) {
    auto node = std::shared_ptr<AttentionNode>(new AttentionNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(query, key, value));
    node->desc = d; node->empty = empty;
    node->q = Saved(q, false);
    node->k = Saved(k, false);
    node->v = Saved(v, false);
    if (n.defined()) node->lengths = Saved(n, false);
    node->lse = lse;
    torch::autograd::set_history(o, node);
    node->o = Saved(o, true);
  }
  return o;
}

}  // namespace

void bind_token_ops(py::module_& m) {
  m.def("layer_norm", torch::wrap_pybind_function_no_gil(layer_norm));
  m.def("rotary_embedding_3d", torch::wrap_pybind_function_no_gil(rotary));
  m.def("cross_attention", torch::wrap_pybind_function_no_gil(cross_attention));
}

}  // namespace d2c_torch
