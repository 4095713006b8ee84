// The attention operators on torch tensors: checks, results and workspaces, calls of the C ABI.
//
// Tensors are read through their Python methods (torch is no build dependency); results and workspaces come from the
// tensors' own allocator (new_empty), so torch's rules for memory and streams hold for them.
#include "python/attention.h"

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

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

py::object steal(PyObject* o) {
  if (!o) {
    throw py::error_already_set();
  }
  return py::reinterpret_steal<py::object>(o);
}

// What is asked of torch, looked up once.  Never freed: it outlives the interpreter's own teardown.
struct Torch {
  py::object bf16, f16, f32, i32, i64, u8, boolean, raw_stream, current_stream, empty;
  PyObject *shape, *stride, *dtype, *data_ptr, *get_device, *is_contiguous, *contiguous, *clone, *new_empty, *cuda_stream, *is_cuda;

  Torch() {
    const py::module_ t = py::module_::import("torch");
    bf16 = t.attr("bfloat16");
    f16 = t.attr("float16");
    f32 = t.attr("float32");
    i32 = t.attr("int32");
    i64 = t.attr("int64");
    u8 = t.attr("uint8");
    boolean = t.attr("bool");
    empty = t.attr("empty");
    current_stream = t.attr("cuda").attr("current_stream");
    const py::object c = t.attr("_C");
    raw_stream = py::getattr(c, "_cuda_getCurrentRawStream", py::none());
    shape = PyUnicode_InternFromString("shape");
    stride = PyUnicode_InternFromString("stride");
    dtype = PyUnicode_InternFromString("dtype");
    data_ptr = PyUnicode_InternFromString("data_ptr");
    get_device = PyUnicode_InternFromString("get_device");
    is_contiguous = PyUnicode_InternFromString("is_contiguous");
    contiguous = PyUnicode_InternFromString("contiguous");
    clone = PyUnicode_InternFromString("clone");
    new_empty = PyUnicode_InternFromString("new_empty");
    cuda_stream = PyUnicode_InternFromString("cuda_stream");
    is_cuda = PyUnicode_InternFromString("is_cuda");
  }

  // Work is queued on torch's current stream of the tensors' device.
  void* stream_of(int device) const {
    if (!raw_stream.is_none()) {
      return reinterpret_cast<void*>(raw_stream(device).cast<uintptr_t>());
    }
    return reinterpret_cast<void*>(current_stream(device).attr("cuda_stream").cast<uintptr_t>());
  }
};

const Torch& torch() {
  static const Torch* t = new Torch();
  return *t;
}

constexpr int kMaxDims = 4;

// A tensor in GPU memory.
struct Tensor {
  py::object obj;
  PyObject* dtype = nullptr;   // of torch, kept alive there
  char* data = nullptr;
  int device = -1, dims = 0;
  int64_t size[kMaxDims], stride[kMaxDims];

  void read(const char* op, const char* name, const py::object& o) {
    const Torch& t = torch();
    obj = o;
    if (!PyObject_HasAttr(o.ptr(), t.data_ptr) || !PyObject_HasAttr(o.ptr(), t.get_device)) {
      bad(op, std::string(name) + " must be a torch tensor");
    }
    device = static_cast<int>(PyLong_AsLong(steal(PyObject_CallMethodNoArgs(o.ptr(), t.get_device)).ptr()));
    if (device < 0) {
      bad(op, std::string(name) + " must be in GPU memory (there is no CPU path)");
    }
    data = reinterpret_cast<char*>(PyLong_AsUnsignedLongLong(steal(PyObject_CallMethodNoArgs(o.ptr(), t.data_ptr)).ptr()));
    dtype = steal(PyObject_GetAttr(o.ptr(), t.dtype)).ptr();
    const py::object shape = steal(PyObject_GetAttr(o.ptr(), t.shape));
    const py::object strides = steal(PyObject_CallMethodNoArgs(o.ptr(), t.stride));
    const Py_ssize_t n = PyTuple_Size(shape.ptr());
    if (n < 1 || n > kMaxDims || PyTuple_Size(strides.ptr()) != n) {
      PyErr_Clear();
      bad(op, std::string(name) + " has " + std::to_string(n) + " dimensions");
    }
    dims = static_cast<int>(n);
    for (int i = 0; i < dims; i++) {
      size[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape.ptr(), i));
      stride[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(strides.ptr(), i));
    }
    if (PyErr_Occurred()) {
      throw py::error_already_set();
    }
  }

  int kind() const {   // mlxd_dtype; -1: another type
    const Torch& t = torch();
    if (dtype == t.bf16.ptr()) return MLXD_BF16;
    if (dtype == t.f16.ptr()) return MLXD_F16;
    if (dtype == t.f32.ptr()) return MLXD_F32;
    if (dtype == t.i64.ptr()) return MLXD_I64;
    if (dtype == t.i32.ptr()) return MLXD_I32;
    if (dtype == t.u8.ptr() || dtype == t.boolean.ptr()) return MLXD_U8;
    return -1;
  }

  std::string text() const {
    return py::str(py::tuple(obj.attr("shape"))).cast<std::string>();
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
      const Torch& t = torch();
      const bool dense = steal(PyObject_CallMethodNoArgs(o.ptr(), t.is_contiguous)).ptr() == Py_True;
      read(op, name, steal(PyObject_CallMethodNoArgs(o.ptr(), dense ? t.clone : t.contiguous)));
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
    if (dtype != like.dtype || device != like.device) {
      bad(op, std::string(name) + " must have the type and device of " + other);
    }
  }
};

// A new tensor of `like`'s shape, type and device, contiguous.
py::object empty_like(const HeadsTensor& like, mlxd_heads* view) {
  const Torch& t = torch();
  const py::object shape = steal(PyObject_GetAttr(like.obj.ptr(), t.shape));
  py::object o = steal(PyObject_CallMethodOneArg(like.obj.ptr(), t.new_empty, shape.ptr()));
  view->data = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(steal(PyObject_CallMethodNoArgs(o.ptr(), t.data_ptr)).ptr()));
  view->stride_head = like.dim;
  view->stride_token = like.heads * like.dim;
  view->stride_batch = like.tokens * view->stride_token;
  return o;
}

py::object empty_bytes(const HeadsTensor& like, size_t bytes, const py::object& dtype, void** data) {
  py::object o = torch().empty(py::make_tuple(bytes), py::arg("dtype") = dtype, py::arg("device") = like.obj.attr("device"));
  *data = reinterpret_cast<void*>(o.attr("data_ptr")().cast<uintptr_t>());
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
      pairs += d.sections[i] = sections[i].cast<int32_t>();
    }
    frequencies.read(op, "frequencies", frequencies_);
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

  void weights(const py::object& q_weight_, const py::object& k_weight_, double eps) {
    weight("q_weight", q_weight_, q_weight, &d.q_weight);
    weight("k_weight", k_weight_, k_weight, &d.k_weight);
    if (d.q_weight && d.k_weight && q_weight.dtype != k_weight.dtype) {
      bad(op, "q_weight and k_weight must have one type");
    }
    d.weight_dtype = d.q_weight ? q_weight.kind() : d.k_weight ? k_weight.kind() : MLXD_F32;
    d.eps = static_cast<float>(eps);
  }

  py::tuple results(int (*call)(int, void*, const mlxd_rotary_desc*)) {
    py::object q_out = empty_like(q, &d.q_out), k_out = py::none();
    if (has_k) {
      k_out = empty_like(k, &d.k_out);
    }
    check(call(q.device, torch().stream_of(q.device), &d));
    return py::make_tuple(q_out, k_out);
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
                         const py::sequence& sections, const py::object& q_weight, const py::object& k_weight, double eps,
                         bool adjacent, bool interleaved) {
  Rotary r{"qk_norm_rotary"};
  r.inputs(q, k);
  r.places(positions, frequencies, sections, adjacent, interleaved);
  r.weights(q_weight, k_weight, eps);
  return r.results(mlxd_qk_norm_rotary);
}

py::tuple qk_norm_rotary_backward(const py::object& q_grad, const py::object& k_grad, const py::object& q, const py::object& k,
                                  const py::object& positions, const py::object& frequencies, const py::sequence& sections,
                                  const py::object& q_weight, const py::object& k_weight, double eps, bool adjacent, bool interleaved) {
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
  const Torch& t = torch();
  py::object wq = py::none(), wk = py::none(), work;
  const auto grad_of = [&](const Tensor& w, void** at) {
    const py::object shape = steal(PyObject_GetAttr(w.obj.ptr(), t.shape));
    py::object o = steal(PyObject_CallMethodOneArg(w.obj.ptr(), t.new_empty, shape.ptr()));
    *at = reinterpret_cast<void*>(PyLong_AsUnsignedLongLong(steal(PyObject_CallMethodNoArgs(o.ptr(), t.data_ptr)).ptr()));
    return o;
  };
  if (r.d.q_weight) {
    wq = grad_of(r.q_weight, &r.d.q_weight_grad);
  }
  if (r.d.k_weight) {
    wk = grad_of(r.k_weight, &r.d.k_weight_grad);
  }
  check(mlxd_qk_norm_rotary_workspace(r.q.device, &r.d, &r.d.workspace_bytes));
  work = empty_bytes(r.q, r.d.workspace_bytes, t.u8, &r.d.workspace);
  const py::tuple x = r.results(mlxd_qk_norm_rotary_backward);
  return py::make_tuple(x[0], x[1], wq, wk);
}

// ---------------------------------------------------------------- cross attention
struct Cross {
  const char* op;
  mlxd_cross_desc d{};
  HeadsTensor q, k, v;
  Tensor lengths, mask;
  py::object copied_mask;

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
    d.scale = scale.is_none() ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(q.dim))) : scale.cast<float>();
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
        mask.read(op, "key_mask", steal(PyObject_CallMethodNoArgs(mask_.ptr(), torch().contiguous)));
      }
      d.key_mask = reinterpret_cast<const uint8_t*>(mask.data);
      d.key_mask_stride = mask.stride[0];
    }
  }

  py::object workspace(bool backward) {
    check(mlxd_cross_attention_workspace(q.device, &d, backward, &d.workspace_bytes));
    return d.workspace_bytes ? empty_bytes(q, d.workspace_bytes, torch().u8, &d.workspace) : py::object(py::none());
  }
};

py::object cross_attention(const py::object& q, const py::object& k, const py::object& v, const py::object& lengths,
                           const py::object& key_mask, const py::object& scale, bool return_lse) {
  Cross c{"cross_attention"};
  c.inputs(q, k, v, lengths, key_mask, scale);
  const py::object work = c.workspace(false);
  const py::object out = empty_like(c.q, &c.d.out);
  py::object lse;
  if (return_lse) {
    void* at = nullptr;
    lse = torch().empty(py::make_tuple(c.d.batch, c.d.q_heads, c.d.q_tokens), py::arg("dtype") = torch().f32,
                        py::arg("device") = c.q.obj.attr("device"));
    at = reinterpret_cast<void*>(lse.attr("data_ptr")().cast<uintptr_t>());
    c.d.lse = static_cast<float*>(at);
  }
  check(mlxd_cross_attention(c.q.device, torch().stream_of(c.q.device), &c.d));
  if (return_lse) {
    return py::make_tuple(out, lse);
  }
  return out;
}

py::tuple cross_attention_backward(const py::object& dout, const py::object& q, const py::object& k, const py::object& v,
                                   const py::object& out, const py::object& lse, const py::object& lengths,
                                   const py::object& key_mask, const py::object& scale) {
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
      l.device != c.q.device || steal(PyObject_CallMethodNoArgs(lse.ptr(), torch().is_contiguous)).ptr() != Py_True) {
    bad(c.op, "lse must be what cross_attention returned: contiguous float32 [batch, q_heads, tokens]");
  }
  c.d.lse = reinterpret_cast<float*>(l.data);
  const py::object work = c.workspace(true);
  const py::object dq = empty_like(c.q, &c.d.dq), dk = empty_like(c.k, &c.d.dk), dv = empty_like(c.v, &c.d.dv);
  check(mlxd_cross_attention_backward(c.q.device, torch().stream_of(c.q.device), &c.d));
  return py::make_tuple(dq, dk, dv);
}

}  // namespace

void bind_attention(py::module_& m) {
  py::module_ a = m.def_submodule("attention", "The attention operators without gradients of their own; see the package's attention.py");
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
        py::arg("out"), py::arg("lse"), py::arg("lengths"), py::arg("key_mask"), py::arg("scale"));
}
