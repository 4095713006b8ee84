// The module `_attention`: the attention operators on torch tensors - checks, results and workspaces, calls of the C ABI.
//
// A module of its own because it is built against torch: a call of a few microseconds has no time for reading tensors through
// their Python methods.  The pipeline's module `_c` knows nothing of torch.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <pybind11/pybind11.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <utility>

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
  const char* q_name = "q";     // what the caller calls them
  const char* k_name = "k";

  void inputs(const py::object& q_, const py::object& k_) {
    q.take(op, q_name, q_, false);
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
      k.take(op, k_name, k_, false);
      k.same_kind(op, k_name, q, q_name);
      if (k.dims != q.dims || k.batch != q.batch || k.tokens != q.tokens || k.dim != q.dim) {
        bad(op, "q and k must agree in all but the number of heads: " + q.text() + " and " + k.text());
      }
      d.k_heads = static_cast<int32_t>(k.heads);
      d.k = k.view();
    }
  }

  void places(const py::object& positions_, const py::object& frequencies_, const py::sequence& sections, bool adjacent, bool interleaved) {
    places_of(positions_, sections);
    turns(frequencies_, sections, adjacent, interleaved);
  }

  void places_of(const py::object& positions_, const py::sequence& sections) {
    positions.read(op, "positions", positions_);
    constant(op, "positions", positions.t);
    if (positions.dims != q.dims - 1) {
      bad(op, "positions must be [axes, batch, tokens] (or [axes, tokens] beside [tokens, heads, head_dim]), got " + positions.text());
    }
    const bool batched = positions.dims == 3;
    if ((batched && positions.size[1] != q.batch) || positions.size[positions.dims - 1] != q.tokens) {
      bad(op, "positions of " + positions.text() + " do not belong to " + q_name + " of " + q.text());
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
    if (positions.device != q.device) {
      bad(op, std::string("positions and frequencies must be on ") + q_name + "'s device");
    }
  }

  void turns(const py::object& frequencies_, const py::sequence& sections, bool adjacent, bool interleaved) {
    const size_t n = py::len(sections);
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
    if (frequencies.device != q.device) {
      bad(op, std::string("positions and frequencies must be on ") + q_name + "'s device");
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

// ---------------------------------------------------------------- a cache in pages
// [pages, page_size, heads, dim]: never copied.
struct PagesTensor : Tensor {
  void take(const char* op, const char* name, const py::object& o, const HeadsTensor& like, const char* other, int64_t heads) {
    read(op, name, o);
    constant(op, name, t);
    if (dims != 4 || size[2] != heads || size[3] != like.dim || size[0] > INT32_MAX || size[1] > INT32_MAX) {
      bad(op, std::string(name) + " must be [pages, page_size, kv_heads, head_dim], got " + text() + " beside " + other + " of " + like.text());
    }
    if (t.scalar_type() != like.t.scalar_type() || device != like.device) {
      bad(op, std::string(name) + " must have the type and device of " + other);
    }
    if (stride[3] != 1 && size[3] > 1) {
      bad(op, std::string(name) + " must have contiguous heads");
    }
  }

  mlxd_pages view() const { return mlxd_pages{data, stride[0], stride[1], stride[2]}; }
};

struct Cache {
  const char* op;
  PagesTensor k, v;
  Tensor table, lengths, counts;

  void vector(const char* name, const py::object& o, const HeadsTensor& like, Tensor& x, const void** data, int32_t* dtype) {
    x.read(op, name, o);
    *dtype = x.kind();
    if ((*dtype != MLXD_I32 && *dtype != MLXD_I64) || x.dims != 1 || x.size[0] != like.batch || (like.batch > 1 && x.stride[0] != 1) ||
        x.device != like.device) {
      bad(op, std::string(name) + " must be a contiguous int32 or int64 vector of one number for each sample, on the cache's device");
    }
    *data = x.data;
  }

  void take(const HeadsTensor& like, const char* other, int64_t heads, const py::object& k_, const py::object& v_, const py::object& table_,
            const py::object& lengths_, const py::object& counts_, mlxd_cache* c) {
    k.take(op, "k_pages", k_, like, other, heads);
    v.take(op, "v_pages", v_, like, other, heads);
    if (k.size[0] != v.size[0] || k.size[1] != v.size[1]) {
      bad(op, "k_pages and v_pages must have one shape: " + k.text() + " and " + v.text());
    }
    c->k = k.view();
    c->v = v.view();
    c->pages = static_cast<int32_t>(k.size[0]);
    c->page_size = static_cast<int32_t>(k.size[1]);
    table.read(op, "page_table", table_);
    c->page_table_dtype = table.kind();
    if ((c->page_table_dtype != MLXD_I32 && c->page_table_dtype != MLXD_I64) || table.dims != 2 || table.size[0] != like.batch ||
        table.size[1] > INT32_MAX || table.device != like.device) {
      bad(op, "page_table must be int32 or int64 [batch, pages of a sample] on the cache's device");
    }
    if (table.size[1] > 1 && table.stride[1] != 1) {
      table.set(op, "page_table", at::Tensor(table.t.contiguous()));
    }
    c->page_table = table.data;
    c->table_width = static_cast<int32_t>(table.size[1]);
    c->page_table_stride = table.stride[0];
    vector("lengths", lengths_, like, lengths, &c->lengths, &c->lengths_dtype);
    if (!counts_.is_none()) {
      vector("counts", counts_, like, counts, &c->counts, &c->counts_dtype);
    }
  }

  // Pools that are written: no element may lie where another one does.
  void written() {
    const auto reach = [](const PagesTensor& x) {
      int64_t n = 1;
      for (int i = 0; i < 4; i++) {
        n += (x.size[i] - 1) * x.stride[i];
      }
      return n * x.t.element_size();
    };
    const auto apart = [](std::array<std::pair<int64_t, int64_t>, 5> dims) {   // strides and sizes
      std::sort(dims.begin(), dims.end());
      int64_t end = 1;
      for (const auto& d : dims) {
        if (d.second > 1) {
          if (d.first < end) {
            return false;
          }
          end += (d.second - 1) * d.first;
        }
      }
      return true;
    };
    if (!k.t.numel()) {
      return;
    }
    const auto dims_of = [](const PagesTensor& x, int64_t stride, int64_t size) {
      return std::array<std::pair<int64_t, int64_t>, 5>{
          {{x.stride[0], x.size[0]}, {x.stride[1], x.size[1]}, {x.stride[2], x.size[2]}, {1, x.size[3]}, {stride, size}}};
    };
    bool fine = apart(dims_of(k, 0, 1)) && apart(dims_of(v, 0, 1));
    if (fine && k.data < v.data + reach(v) && v.data < k.data + reach(k)) {   // one allocation: keys and values as one more dimension of it
      const int64_t bytes = k.data < v.data ? v.data - k.data : k.data - v.data, item = k.t.element_size();
      fine = bytes % item == 0 && k.t.strides() == v.t.strides() && apart(dims_of(k, bytes / item, 2));
    }
    if (!fine) {
      bad(op, "k_pages and v_pages are written and must overlap neither themselves nor each other");
    }
    k.t.unsafeGetTensorImpl()->bump_version();
    v.t.unsafeGetTensorImpl()->bump_version();
  }
};

py::object append_rotary(const py::object& q, const py::object& k, const py::object& v, const py::object& positions, const py::object& frequencies,
                         const py::sequence& sections, const py::object& k_pages, const py::object& v_pages, const py::object& page_table,
                         const py::object& lengths, const py::object& counts, bool adjacent, bool interleaved) {
  Rotary r{"append_rotary"};
  r.q_name = "k";               // there may be no queries
  r.k_name = "q";
  r.inputs(k, q);
  constant(r.op, "k", r.q.t);
  if (r.has_k) {
    constant(r.op, "q", r.k.t);
  }
  if (r.q.dims != 4) {
    bad(r.op, "k must be [batch, tokens, kv_heads, head_dim], got " + r.q.text());
  }
  if (positions.is_none()) {
    r.d.n_axes = static_cast<int32_t>(std::min<size_t>(py::len(sections), 1 << 20));
  } else {
    r.places_of(positions, sections);
  }
  r.turns(frequencies, sections, adjacent, interleaved);
  std::swap(r.d.q, r.d.k);
  std::swap(r.d.q_heads, r.d.k_heads);
  mlxd_append_desc d{};
  d.r = r.d;
  HeadsTensor values;
  values.take(r.op, "v", v, false);
  values.same_shape(r.op, "v", r.q, "k");
  constant(r.op, "v", values.t);
  d.v = values.view();
  Cache c{r.op};
  c.take(r.q, "k", r.q.heads, k_pages, v_pages, page_table, lengths, counts, &d.cache);
  c.written();
  at::Tensor q_out;
  if (r.has_k) {
    q_out = empty_like(r.k, &d.r.q_out);
  }
  check(mlxd_append_rotary(r.q.device, stream_of(r.q.device), &d));
  return r.has_k ? wrapped(q_out) : py::none();
}

// ---------------------------------------------------------------- cached and window attention
// What both take alike; `Desc` is one of their descriptors.
template <class Desc>
void attention_inputs(const char* op, Desc& d, const HeadsTensor& q, int64_t kv_heads, const py::object& window, const py::object& sinks,
                      const py::object& scale) {
  d.dtype = q.kind();
  if (d.dtype != MLXD_BF16 && d.dtype != MLXD_F16) {
    bad(op, "tensors must be bfloat16 or float16");
  }
  d.batch = static_cast<int32_t>(q.batch);
  d.tokens = static_cast<int32_t>(q.tokens);
  d.q_heads = static_cast<int32_t>(q.heads);
  d.kv_heads = static_cast<int32_t>(kv_heads);
  d.head_dim = static_cast<int32_t>(q.dim);
  if (!window.is_none()) {
    const int64_t n = number<int64_t>(op, "window", window);
    if (n < 1) {
      bad(op, "window must be at least 1, or None");
    }
    d.window = static_cast<int32_t>(std::min<int64_t>(n, INT32_MAX));
  }
  const int64_t first = number<int64_t>(op, "sinks", sinks);
  if (first < 0) {
    bad(op, "sinks must not be negative");
  }
  d.sinks = static_cast<int32_t>(std::min<int64_t>(first, INT32_MAX));
  d.scale = scale.is_none() ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(q.dim))) : number<float>(op, "scale", scale);
  d.q = q.view();
}

at::Tensor lse_like(const HeadsTensor& q) {
  return at::empty({q.batch, q.heads, q.tokens}, at::TensorOptions().dtype(at::kFloat).device(q.t.device()));
}

py::object cached_attention(const py::object& q_, const py::object& k_pages, const py::object& v_pages, const py::object& page_table,
                            const py::object& lengths, const py::object& counts, const py::object& tree_, const py::object& window,
                            const py::object& sinks, const py::object& scale, bool return_lse) {
  const char* op = "cached_attention";
  mlxd_cached_desc d{};
  HeadsTensor q;
  q.take(op, "q", q_, true);
  constant(op, "q", q.t);
  if (q.dims != 4) {
    bad(op, "q must be [batch, tokens, q_heads, head_dim], got " + q.text());
  }
  Tensor pages;
  pages.read(op, "k_pages", k_pages);
  const int64_t kv_heads = pages.dims == 4 && pages.size[2] <= INT32_MAX ? pages.size[2] : 0;
  attention_inputs(op, d, q, kv_heads, window, sinks, scale);
  Cache c{op};
  c.take(q, "q", kv_heads, k_pages, v_pages, page_table, lengths, counts, &d.cache);
  Tensor tree;
  if (!tree_.is_none()) {
    tree.read(op, "tree", tree_);
    const int o = tree.dims - 2;
    if (tree.kind() != MLXD_U8 || (tree.dims != 2 && tree.dims != 3) || (o && tree.size[0] != q.batch) || tree.size[o] != q.tokens ||
        tree.size[o + 1] != q.tokens || tree.device != q.device) {
      bad(op, "tree must be bool [batch, tokens, tokens] or [tokens, tokens] on q's device");
    }
    if (tree.size[o + 1] > 1 && tree.stride[o + 1] != 1) {
      tree.set(op, "tree", at::Tensor(tree.t.contiguous()));
    }
    d.tree = reinterpret_cast<const uint8_t*>(tree.data);
    d.tree_stride_batch = o ? tree.stride[0] : 0;
    d.tree_stride_token = tree.stride[o];
  }
  check(mlxd_cached_attention_workspace(q.device, &d, &d.workspace_bytes));
  const at::Tensor work = d.workspace_bytes ? empty_bytes(q, d.workspace_bytes, &d.workspace) : at::Tensor();
  const at::Tensor out = empty_like(q, &d.out);
  at::Tensor lse;
  if (return_lse) {
    lse = lse_like(q);
    d.lse = static_cast<float*>(lse.data_ptr());
  }
  check(mlxd_cached_attention(q.device, stream_of(q.device), &d));
  return return_lse ? py::object(py::make_tuple(wrapped(out), wrapped(lse))) : wrapped(out);
}

struct Window {
  const char* op;
  mlxd_window_desc d{};
  HeadsTensor q, k, v;
  Tensor lengths;

  void inputs(const py::object& q_, const py::object& k_, const py::object& v_, const py::object& window, const py::object& sinks,
              const py::object& lengths_, const py::object& scale) {
    q.take(op, "q", q_, true);
    k.take(op, "k", k_, true);
    v.take(op, "v", v_, true);
    k.same_kind(op, "k", q, "q");
    v.same_shape(op, "v", k, "k");
    if (q.dims != 4 || k.dims != 4 || k.batch != q.batch || k.tokens != q.tokens || k.dim != q.dim) {
      bad(op, "q must be [batch, tokens, q_heads, head_dim] and k, v [batch, tokens, kv_heads, head_dim], got " + q.text() + " and " + k.text());
    }
    attention_inputs(op, d, q, k.heads, window, sinks, scale);
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
  }

  at::Tensor workspace(bool backward) {
    check(mlxd_window_attention_workspace(q.device, &d, backward, &d.workspace_bytes));
    return d.workspace_bytes ? empty_bytes(q, d.workspace_bytes, &d.workspace) : at::Tensor();
  }
};

py::object window_attention(const py::object& q, const py::object& k, const py::object& v, const py::object& window, const py::object& sinks,
                            const py::object& lengths, const py::object& scale, bool return_lse) {
  Window w{"window_attention"};
  w.inputs(q, k, v, window, sinks, lengths, scale);
  const at::Tensor work = w.workspace(false);
  const at::Tensor out = empty_like(w.q, &w.d.out);
  at::Tensor lse;
  if (return_lse) {
    lse = lse_like(w.q);
    w.d.lse = static_cast<float*>(lse.data_ptr());
  }
  check(mlxd_window_attention(w.q.device, stream_of(w.q.device), &w.d));
  return return_lse ? py::object(py::make_tuple(wrapped(out), wrapped(lse))) : wrapped(out);
}

py::tuple window_attention_backward(const py::object& dout, const py::object& q, const py::object& k, const py::object& v, const py::object& out,
                                    const py::object& lse, const py::object& window, const py::object& sinks, const py::object& lengths,
                                    const py::object& scale, const py::object& lse_grad) {
  Window w{"window_attention_backward"};
  w.inputs(q, k, v, window, sinks, lengths, scale);
  HeadsTensor o, g;
  o.take(w.op, "out", out, true);
  o.same_shape(w.op, "out", w.q, "q");
  g.take(w.op, "dout", dout, true);
  g.same_shape(w.op, "dout", w.q, "q");
  w.d.out = o.view();
  w.d.dout = g.view();
  Tensor l, lg;
  l.read(w.op, "lse", lse);
  if (l.kind() != MLXD_F32 || l.dims != 3 || l.size[0] != w.d.batch || l.size[1] != w.d.q_heads || l.size[2] != w.d.tokens ||
      l.device != w.q.device || !l.t.is_contiguous()) {
    bad(w.op, "lse must be what window_attention returned: contiguous float32 [batch, q_heads, tokens]");
  }
  w.d.lse = reinterpret_cast<float*>(l.data);
  if (!lse_grad.is_none()) {
    lg.read(w.op, "lse_grad", lse_grad);
    if (lg.kind() != MLXD_F32 || lg.t.sizes() != l.t.sizes() || lg.device != w.q.device) {
      bad(w.op, "lse_grad must have lse's shape, type and device");
    }
    if (!lg.t.is_contiguous()) {
      lg.set(w.op, "lse_grad", at::Tensor(lg.t.contiguous()));
    }
    w.d.lse_grad = reinterpret_cast<const float*>(lg.data);
  }
  const at::Tensor work = w.workspace(true);
  const at::Tensor dq = empty_like(w.q, &w.d.dq), dk = empty_like(w.k, &w.d.dk), dv = empty_like(w.v, &w.d.dv);
  check(mlxd_window_attention_backward(w.q.device, stream_of(w.q.device), &w.d));
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
  a.def("append_rotary", &append_rotary, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("positions"), py::arg("frequencies"),
        py::arg("sections"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"), py::arg("lengths"), py::arg("counts"),
        py::arg("adjacent"), py::arg("interleaved"));
  a.def("cached_attention", &cached_attention, py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
        py::arg("lengths"), py::arg("counts"), py::arg("tree"), py::arg("window"), py::arg("sinks"), py::arg("scale"), py::arg("return_lse"));
  a.def("window_attention", &window_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("window"), py::arg("sinks"),
        py::arg("lengths"), py::arg("scale"), py::arg("return_lse"));
  a.def("window_attention_backward", &window_attention_backward, py::arg("dout"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("out"),
        py::arg("lse"), py::arg("window"), py::arg("sinks"), py::arg("lengths"), py::arg("scale"), py::arg("lse_grad"));
}
