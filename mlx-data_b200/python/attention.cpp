// The module `_attention`: the attention operators on torch tensors - checks, results and workspaces, calls of the C ABI.
//
// A module of its own because it is built against torch: a call of a few microseconds has no time for reading tensors through
// their Python methods.  The pipeline's module `_c` knows nothing of torch.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <pybind11/pybind11.h>

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/mlxd_b200.h"

namespace py = pybind11;

namespace {

[[noreturn]] void bad(const char* op, const std::string& what) {
  throw std::invalid_argument(std::string(op) + ": " + what);
}

void check(int rc) {
  if (rc == MLXD_OK) {
    return;
  }
  if (rc == MLXD_ERR_INVALID) {
    throw std::invalid_argument(mlxd_last_error());
  }
  throw std::runtime_error(std::string("mlx-data GPU path: ") + mlxd_last_error());
}

// A gradient that would not be worked out is refused.
void constant(const char* op, const char* name, const at::Tensor& t) {
  if (t.requires_grad() && c10::GradMode::is_enabled()) {
    bad(op, std::string(name) + " has no gradient here but requires one; pass " + name + ".detach()");
  }
}

// A Python number; what is none, or does not fit, is a wrong argument like any other.
template <class T>
T number(const char* op, const char* name, const py::handle& o) {
  if (!PyLong_CheckExact(o.ptr()) && !PyFloat_CheckExact(o.ptr()) && THPVariable_Check(o.ptr())) {
    constant(op, name, THPVariable_Unpack(o.ptr()));
  }
  try {
    return o.cast<T>();
  } catch (const py::cast_error&) {
    bad(op, std::string(name) + (std::is_integral<T>::value ? " must be whole numbers" : " must be a number"));
  }
}

// Work is queued on torch's current stream of the tensors' device.
void* stream_of(int device) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

py::object wrapped(const at::Tensor& t) {
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(t));
}

constexpr int kMaxDims = 4;

// A tensor in GPU memory.
struct Tensor {
  at::Tensor t;
  char* data = nullptr;
  int device = -1, dims = 0;
  int64_t size[kMaxDims], stride[kMaxDims];

  void read(const char* op, const char* name, const py::object& o) {
    if (!THPVariable_Check(o.ptr())) {
      bad(op, std::string(name) + " must be a torch tensor");
    }
    set(op, name, THPVariable_Unpack(o.ptr()));
  }

  void set(const char* op, const char* name, const at::Tensor& from) {
    t = from;
    if (!t.is_cuda()) {
      bad(op, std::string(name) + " must be in GPU memory (there is no CPU path)");
    }
    if (t._fw_grad(0).defined()) {
      bad(op, std::string(name) + " carries a tangent: there is no forward-mode derivative here");
    }
    if (t.layout() != at::kStrided || t.is_conj() || t.is_neg()) {
      bad(op, std::string(name) + " must be an ordinary strided tensor");
    }
    device = t.get_device();
    data = static_cast<char*>(t.data_ptr());
    const auto sizes = t.sizes(), strides = t.strides();
    if (sizes.size() < 1 || sizes.size() > kMaxDims) {
      bad(op, std::string(name) + " has " + std::to_string(sizes.size()) + " dimensions");
    }
    dims = static_cast<int>(sizes.size());
    for (int i = 0; i < dims; i++) {
      size[i] = sizes[i];
      stride[i] = strides[i];
    }
  }

  int kind() const {   // mlxd_dtype; -1: another type
    switch (t.scalar_type()) {
      case at::kBFloat16: return MLXD_BF16;
      case at::kHalf: return MLXD_F16;
      case at::kFloat: return MLXD_F32;
      case at::kLong: return MLXD_I64;
      case at::kInt: return MLXD_I32;
      case at::kByte: case at::kBool: return MLXD_U8;
      default: return -1;
    }
  }

  std::string text() const {
    std::string s = "(";
    for (int i = 0; i < dims; i++) {
      s += (i ? ", " : "") + std::to_string(size[i]);
    }
    return s + ")";
  }
};

// [batch, tokens, heads, dim] or [tokens, heads, dim]
struct HeadsTensor : Tensor {
  int64_t batch, tokens, heads, dim;

  void layout(const char* op, const char* name) {
    if (dims != 3 && dims != 4) {
      bad(op, std::string(name) + " must be [batch, tokens, heads, head_dim] or [tokens, heads, head_dim], got " + text());
    }
    const int o = dims - 3;
    batch = o ? size[0] : 1;
    tokens = size[o];
    heads = size[o + 1];
    dim = size[o + 2];
    if (batch > INT32_MAX || tokens > INT32_MAX || heads > INT32_MAX || dim > INT32_MAX) {
      bad(op, std::string(name) + " is too large");
    }
  }

  // Rows have to be contiguous; with `units` they start on 16 bytes too.  Others are copied.
  void take(const char* op, const char* name, const py::object& o, bool units) {
    read(op, name, o);
    layout(op, name);
    bool fits = stride[dims - 1] == 1 || dim <= 1;
    if (units) {
      fits = fits && reinterpret_cast<uintptr_t>(data) % 16 == 0;
      for (int i = 0; i < dims - 1; i++) {
        fits = fits && (size[i] <= 1 || (stride[i] % 8 == 0 && stride[i] > 0));
      }
    }
    if (!fits) {
      const at::Tensor copy = t.is_contiguous() ? t.clone() : t.contiguous();
      set(op, name, copy);
      layout(op, name);
    }
  }

  mlxd_heads view() const {
    const int o = dims - 3;
    return mlxd_heads{data, o ? stride[0] : 0, stride[o], stride[o + 1]};
  }

  void same_shape(const char* op, const char* name, const HeadsTensor& like, const char* other) const {
    bool same = dims == like.dims;
    for (int i = 0; same && i < dims; i++) {
      same = size[i] == like.size[i];
    }
    if (!same) {
      bad(op, std::string(name) + " must have the shape of " + other + ": " + text() + " and " + like.text());
    }
    same_kind(op, name, like, other);
  }

  void same_kind(const char* op, const char* name, const HeadsTensor& like, const char* other) const {
    if (t.scalar_type() != like.t.scalar_type() || device != like.device) {
      bad(op, std::string(name) + " must have the type and device of " + other);
    }
  }
};

// A new tensor of `like`'s shape, type and device, contiguous.
at::Tensor empty_like(const HeadsTensor& like, mlxd_heads* view) {
  at::Tensor o = at::empty(like.t.sizes(), like.t.options().requires_grad(false));
  view->data = o.data_ptr();
  view->stride_head = like.dim;
  view->stride_token = like.heads * like.dim;
  view->stride_batch = like.tokens * view->stride_token;
  return o;
}

at::Tensor empty_bytes(const HeadsTensor& like, size_t bytes, void** data) {
  at::Tensor o = at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(like.t.device()));
  *data = o.data_ptr();
  return o;
}

// ---------------------------------------------------------------- rotary
struct Rotary {
  const char* op;
  mlxd_rotary_desc d{};
  HeadsTensor q, k;
  Tensor positions, frequencies, q_weight, k_weight;
  bool has_k = false;

  void inputs(const py::object& q_, const py::object& k_) {
    q.take(op, "q", q_, false);
    d.dtype = q.kind();
    if (d.dtype != MLXD_F32 && d.dtype != MLXD_BF16 && d.dtype != MLXD_F16) {
      bad(op, "tensors must be float32, bfloat16 or float16");
    }
    d.batch = static_cast<int32_t>(q.batch);
    d.tokens = static_cast<int32_t>(q.tokens);
    d.q_heads = static_cast<int32_t>(q.heads);
    d.head_dim = static_cast<int32_t>(q.dim);
    d.q = q.view();
    has_k = !k_.is_none();
    if (has_k) {
      k.take(op, "k", k_, false);
      k.same_kind(op, "k", q, "q");
      if (k.dims != q.dims || k.batch != q.batch || k.tokens != q.tokens || k.dim != q.dim) {
        bad(op, "q and k must agree in all but the number of heads: " + q.text() + " and " + k.text());
      }
      d.k_heads = static_cast<int32_t>(k.heads);
      d.k = k.view();
    }
  }

  void places(const py::object& positions_, const py::object& frequencies_, const py::sequence& sections, bool adjacent, bool interleaved) {
    positions.read(op, "positions", positions_);
    constant(op, "positions", positions.t);
    if (positions.dims != q.dims - 1) {
      bad(op, "positions must be [axes, batch, tokens] (or [axes, tokens] beside [tokens, heads, head_dim]), got " + positions.text());
    }
    const bool batched = positions.dims == 3;
    if ((batched && positions.size[1] != q.batch) || positions.size[positions.dims - 1] != q.tokens) {
      bad(op, "positions of " + positions.text() + " do not belong to q of " + q.text());
    }
    d.n_axes = static_cast<int32_t>(std::min<int64_t>(positions.size[0], 1 << 20));
    d.positions = positions.data;
    d.positions_dtype = positions.kind();
    d.positions_stride_axis = positions.stride[0];
    d.positions_stride_batch = batched ? positions.stride[1] : 0;
    d.positions_stride_token = positions.stride[positions.dims - 1];
    const size_t n = py::len(sections);
    if (static_cast<int64_t>(n) != positions.size[0]) {
      bad(op, "one section for each axis: " + std::to_string(n) + " sections, positions of " + positions.text());
    }
    int64_t pairs = 0;
    for (size_t i = 0; i < n && i < MLXD_ROTARY_MAX_AXES; i++) {
      pairs += d.sections[i] = number<int32_t>(op, "sections", sections[i]);
    }
    frequencies.read(op, "frequencies", frequencies_);
    constant(op, "frequencies", frequencies.t);
    if (frequencies.kind() != MLXD_F32 || frequencies.dims != 1 || (frequencies.size[0] > 1 && frequencies.stride[0] != 1)) {
      bad(op, "frequencies must be a contiguous float32 vector");
    }
    if (n <= MLXD_ROTARY_MAX_AXES && frequencies.size[0] != pairs) {
      bad(op, "one frequency for each pair: " + std::to_string(frequencies.size[0]) + " frequencies, " + std::to_string(pairs) + " pairs in the sections");
    }
    if (positions.device != q.device || frequencies.device != q.device) {
      bad(op, "positions and frequencies must be on q's device");
    }
    d.frequencies = reinterpret_cast<const float*>(frequencies.data);
    d.adjacent = adjacent;
    d.interleaved = interleaved;
  }

  void weight(const char* name, const py::object& o, Tensor& w, const void** at) {
    if (o.is_none()) {
      return;
    }
    w.read(op, name, o);
    if (w.dims != 1 || w.size[0] != q.dim || (w.size[0] > 1 && w.stride[0] != 1) || w.device != q.device) {
      bad(op, std::string(name) + " must be a contiguous vector of head_dim values on q's device");
    }
    *at = w.data;
  }

  void weights(const py::object& q_weight_, const py::object& k_weight_, const py::object& eps) {
    weight("q_weight", q_weight_, q_weight, &d.q_weight);
    weight("k_weight", k_weight_, k_weight, &d.k_weight);
    if (d.q_weight && d.k_weight && q_weight.t.scalar_type() != k_weight.t.scalar_type()) {
      bad(op, "q_weight and k_weight must have one type");
    }
    d.weight_dtype = d.q_weight ? q_weight.kind() : d.k_weight ? k_weight.kind() : MLXD_F32;
    d.eps = static_cast<float>(number<double>(op, "eps", eps));
  }

  py::tuple results(int (*call)(int, void*, const mlxd_rotary_desc*)) {
    const at::Tensor q_out = empty_like(q, &d.q_out);
    at::Tensor k_out;
    if (has_k) {
      k_out = empty_like(k, &d.k_out);
    }
    check(call(q.device, stream_of(q.device), &d));
    return py::make_tuple(wrapped(q_out), has_k ? wrapped(k_out) : py::none());
  }
};

py::tuple rotary(const py::object& q, const py::object& k, const py::object& positions, const py::object& frequencies,
                 const py::sequence& sections, bool inverse, bool adjacent, bool interleaved) {
  Rotary r{"rotary"};
  r.inputs(q, k);
  r.places(positions, frequencies, sections, adjacent, interleaved);
  r.d.inverse = inverse;
  return r.results(mlxd_rotary);
}

py::tuple qk_norm_rotary(const py::object& q, const py::object& k, const py::object& positions, const py::object& frequencies,
                         const py::sequence& sections, const py::object& q_weight, const py::object& k_weight, const py::object& eps,
                         bool adjacent, bool interleaved) {
  Rotary r{"qk_norm_rotary"};
  r.inputs(q, k);
  r.places(positions, frequencies, sections, adjacent, interleaved);
  r.weights(q_weight, k_weight, eps);
  return r.results(mlxd_qk_norm_rotary);
}

py::tuple qk_norm_rotary_backward(const py::object& q_grad, const py::object& k_grad, const py::object& q, const py::object& k,
                                  const py::object& positions, const py::object& frequencies, const py::sequence& sections,
                                  const py::object& q_weight, const py::object& k_weight, const py::object& eps, bool adjacent, bool interleaved) {
  Rotary r{"qk_norm_rotary_backward"};
  r.inputs(q, k);
  r.places(positions, frequencies, sections, adjacent, interleaved);
  r.weights(q_weight, k_weight, eps);
  HeadsTensor gq, gk;
  gq.take(r.op, "q_grad", q_grad, false);
  gq.same_shape(r.op, "q_grad", r.q, "q");
  r.d.q_grad = gq.view();
  if (r.has_k != !k_grad.is_none()) {
    bad(r.op, "k and its gradient come together");
  }
  if (r.has_k) {
    gk.take(r.op, "k_grad", k_grad, false);
    gk.same_shape(r.op, "k_grad", r.k, "k");
    r.d.k_grad = gk.view();
  }
  at::Tensor wq, wk;
  const auto grad_of = [&](const Tensor& w, void** at) {
    at::Tensor o = at::empty(w.t.sizes(), w.t.options().requires_grad(false));
    *at = o.data_ptr();
    return o;
  };
  if (r.d.q_weight) {
    wq = grad_of(r.q_weight, &r.d.q_weight_grad);
  }
  if (r.d.k_weight) {
    wk = grad_of(r.k_weight, &r.d.k_weight_grad);
  }
  check(mlxd_qk_norm_rotary_workspace(r.q.device, &r.d, &r.d.workspace_bytes));
  const at::Tensor work = empty_bytes(r.q, r.d.workspace_bytes, &r.d.workspace);
  const py::tuple x = r.results(mlxd_qk_norm_rotary_backward);
  return py::make_tuple(x[0], x[1], wq.defined() ? wrapped(wq) : py::none(), wk.defined() ? wrapped(wk) : py::none());
}

// ---------------------------------------------------------------- cross attention
struct Cross {
  const char* op;
  mlxd_cross_desc d{};
  HeadsTensor q, k, v;
  Tensor lengths, mask;

  void inputs(const py::object& q_, const py::object& k_, const py::object& v_, const py::object& lengths_, const py::object& mask_,
              const py::object& scale) {
    q.take(op, "q", q_, true);
    k.take(op, "k", k_, true);
    v.take(op, "v", v_, true);
    d.dtype = q.kind();
    if (d.dtype != MLXD_BF16 && d.dtype != MLXD_F16) {
      bad(op, "tensors must be bfloat16 or float16");
    }
    k.same_kind(op, "k", q, "q");
    v.same_shape(op, "v", k, "k");
    if (q.dims != 4 || k.dims != 4 || k.batch != q.batch || k.dim != q.dim) {
      bad(op, "q must be [batch, tokens, q_heads, head_dim] and k, v [batch, keys, kv_heads, head_dim], got " + q.text() + " and " + k.text());
    }
    d.batch = static_cast<int32_t>(q.batch);
    d.q_tokens = static_cast<int32_t>(q.tokens);
    d.kv_tokens = static_cast<int32_t>(k.tokens);
    d.q_heads = static_cast<int32_t>(q.heads);
    d.kv_heads = static_cast<int32_t>(k.heads);
    d.head_dim = static_cast<int32_t>(q.dim);
    d.scale = scale.is_none() ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(q.dim))) : number<float>(op, "scale", scale);
    d.q = q.view();
    d.k = k.view();
    d.v = v.view();
    if (!lengths_.is_none()) {
      lengths.read(op, "lengths", lengths_);
      d.lengths_dtype = lengths.kind();
      if ((d.lengths_dtype != MLXD_I32 && d.lengths_dtype != MLXD_I64) || lengths.dims != 1 || lengths.size[0] != q.batch ||
          (q.batch > 1 && lengths.stride[0] != 1) || lengths.device != q.device) {
        bad(op, "lengths must be a contiguous int32 or int64 vector of one number for each sample, on q's device");
      }
      d.lengths = lengths.data;
    }
    if (!mask_.is_none()) {
      mask.read(op, "key_mask", mask_);
      if (mask.kind() != MLXD_U8 || mask.dims != 2 || mask.size[0] != k.batch || mask.size[1] != k.tokens || mask.device != q.device) {
        bad(op, "key_mask must be bool [batch, keys] on q's device");
      }
      if (mask.size[1] > 1 && mask.stride[1] != 1) {
        mask.set(op, "key_mask", at::Tensor(mask.t.contiguous()));
      }
      d.key_mask = reinterpret_cast<const uint8_t*>(mask.data);
      d.key_mask_stride = mask.stride[0];
    }
  }

  at::Tensor workspace(bool backward) {
    check(mlxd_cross_attention_workspace(q.device, &d, backward, &d.workspace_bytes));
    return d.workspace_bytes ? empty_bytes(q, d.workspace_bytes, &d.workspace) : at::Tensor();
  }
};

py::object cross_attention(const py::object& q, const py::object& k, const py::object& v, const py::object& lengths,
                           const py::object& key_mask, const py::object& scale, bool return_lse) {
  Cross c{"cross_attention"};
  c.inputs(q, k, v, lengths, key_mask, scale);
  const at::Tensor work = c.workspace(false);
  const at::Tensor out = empty_like(c.q, &c.d.out);
  at::Tensor lse;
  if (return_lse) {
    lse = at::empty({c.d.batch, c.d.q_heads, c.d.q_tokens}, at::TensorOptions().dtype(at::kFloat).device(c.q.t.device()));
    c.d.lse = static_cast<float*>(lse.data_ptr());
  }
  check(mlxd_cross_attention(c.q.device, stream_of(c.q.device), &c.d));
  if (return_lse) {
    return py::make_tuple(wrapped(out), wrapped(lse));
  }
  return wrapped(out);
}

py::tuple cross_attention_backward(const py::object& dout, const py::object& q, const py::object& k, const py::object& v,
                                   const py::object& out, const py::object& lse, const py::object& lengths,
                                   const py::object& key_mask, const py::object& scale, const py::object& lse_grad) {
  Cross c{"cross_attention_backward"};
  c.inputs(q, k, v, lengths, key_mask, scale);
  HeadsTensor o, g;
  o.take(c.op, "out", out, true);
  o.same_shape(c.op, "out", c.q, "q");
  g.take(c.op, "dout", dout, true);
  g.same_shape(c.op, "dout", c.q, "q");
  c.d.out = o.view();
  c.d.dout = g.view();
  Tensor l;
  l.read(c.op, "lse", lse);
  if (l.kind() != MLXD_F32 || l.dims != 3 || l.size[0] != c.d.batch || l.size[1] != c.d.q_heads || l.size[2] != c.d.q_tokens ||
      l.device != c.q.device || !l.t.is_contiguous()) {
    bad(c.op, "lse must be what cross_attention returned: contiguous float32 [batch, q_heads, tokens]");
  }
  c.d.lse = reinterpret_cast<float*>(l.data);
  Tensor lg;
  if (!lse_grad.is_none()) {
    lg.read(c.op, "lse_grad", lse_grad);
    if (lg.kind() != MLXD_F32 || lg.t.sizes() != l.t.sizes() || lg.device != c.q.device) {
      bad(c.op, "lse_grad must have lse's shape, type and device");
    }
    if (!lg.t.is_contiguous()) {
      lg.set(c.op, "lse_grad", at::Tensor(lg.t.contiguous()));
    }
  }
  const at::Tensor work = c.workspace(true);
  const at::Tensor dq = empty_like(c.q, &c.d.dq), dk = empty_like(c.k, &c.d.dk), dv = empty_like(c.v, &c.d.dv);
  check(mlxd_cross_attention_backward_lse(c.q.device, stream_of(c.q.device), &c.d, reinterpret_cast<const float*>(lg.data)));
  return py::make_tuple(wrapped(dq), wrapped(dk), wrapped(dv));
}

}  // namespace

PYBIND11_MODULE(_attention, a) {
  a.doc() = "The attention operators without gradients of their own; see attention.py";
  a.def("rotary", &rotary, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("frequencies"), py::arg("sections"),
        py::arg("inverse"), py::arg("adjacent"), py::arg("interleaved"));
  a.def("qk_norm_rotary", &qk_norm_rotary, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("frequencies"),
        py::arg("sections"), py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"), py::arg("adjacent"), py::arg("interleaved"));
  a.def("qk_norm_rotary_backward", &qk_norm_rotary_backward, py::arg("q_grad"), py::arg("k_grad"), py::arg("q"), py::arg("k"),
        py::arg("positions"), py::arg("frequencies"), py::arg("sections"), py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"),
        py::arg("adjacent"), py::arg("interleaved"));
  a.def("cross_attention", &cross_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("lengths"), py::arg("key_mask"),
        py::arg("scale"), py::arg("return_lse"));
  a.def("cross_attention_backward", &cross_attention_backward, py::arg("dout"), py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("out"), py::arg("lse"), py::arg("lengths"), py::arg("key_mask"), py::arg("scale"), py::arg("lse_grad"));
}
