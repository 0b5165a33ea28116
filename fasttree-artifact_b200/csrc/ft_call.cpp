// The Python call path of the decode entry points: checks the tensors, fills ft_decode_args and calls the C ABI.
//
// A decode step of a few requests is about ten microseconds of GPU work, launched once per layer and step, with a query
// and an output that are new tensors each time.  Done in Python, the checks and the forty-odd argument fields took
// 13.6 us per call (18 us in fp32), so small steps were bound by the host; here they take well under a microsecond beside
// the two launches, which is cheap enough to do for every call: nothing is remembered from one call for the next,
// the argument block lives on the stack, and the GIL is released around the launch.
//
// Built as an extension module of its own (ft_b200/build.py): libfasttree_b200.so stays free of Python and torch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>

#include "fasttree_b200.h"

namespace {

typedef int (*DecodeFn)(const ft_decode_args*);
DecodeFn g_entry[3] = {nullptr, nullptr, nullptr};  // ft_decode, ft_stage1, ft_stage2
int (*g_append)(const ft_append_args*) = nullptr;
int (*g_extend)(const ft_extend_args*) = nullptr;

struct Refused {};  // a Python error has been set

[[noreturn]] void refuse(const char* fmt, const char* name, const char* more = "") {
  PyErr_Format(PyExc_ValueError, fmt, name, more);
  throw Refused();
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse("%s must be a torch.Tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda())
    refuse("%s is on %s; the engine has no CPU path - tensors must live on a CUDA device", name, t.device().str().c_str());
  return t;
}

const at::Tensor& table(const char* name, PyObject* o) {
  const at::Tensor& t = tensor(name, o);
  if (t.scalar_type() != at::kInt) refuse("%s must be int32, got %s", name, c10::toString(t.scalar_type()));
  if (!t.is_contiguous()) refuse("%s must be contiguous", name);
  return t;
}

void pair(const char* name, PyObject* o, int64_t (&out)[2]) {
  PyObject* seq = PySequence_Fast(o, "expected a pair of integers");
  if (seq == nullptr) throw Refused();
  if (PySequence_Fast_GET_SIZE(seq) != 2) {
    Py_DECREF(seq);
    refuse("%s must have two entries (one per phase)", name);
  }
  for (int i = 0; i < 2; ++i) {
    PyObject* v = PyNumber_Long(PySequence_Fast_GET_ITEM(seq, i));
    out[i] = v != nullptr ? PyLong_AsLongLong(v) : -1;
    Py_XDECREF(v);
    if (PyErr_Occurred()) {
      Py_DECREF(seq);
      throw Refused();
    }
  }
  Py_DECREF(seq);
}

// The task sizes that a plan's vnode_to_kv_lens tensor carries as an attribute (ft_b200.planner.task_sizes), with the plan's
// partial rows behind them where the scratch buffers hold more; without it none are known.
void task_sizes(PyObject* table, ft_decode_args& a) {
  static PyObject* const name = PyUnicode_InternFromString("task_sizes");
  PyObject* sizes = nullptr;
  if (_PyObject_LookupAttr(table, name, &sizes) < 0) throw Refused();
  if (sizes == nullptr) return;
  long long n[5] = {0, 0, 0, 0, 0};
  const int count = PyTuple_Check(sizes) ? (int)PyTuple_GET_SIZE(sizes) : 0;
  for (int i = 0; (count == 4 || count == 5) && i < count; ++i) n[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(sizes, i));
  Py_DECREF(sizes);
  if (PyErr_Occurred()) throw Refused();
  a.few_tokens = n[0];
  a.few_longest = (int32_t)n[1];
  a.few_over_8_rows = (int32_t)n[2];
  a.many_longest = (int32_t)n[3];
  a.plan_rows = (int32_t)n[4];
}

// Positional arguments of the reference's fasttree_decode (kernel_bench/fasttree.py:582-601), in order.
enum { Q, K, V, O, KV_ENTRIES, KV_OFFS, KV_LENS, Q_ENTRIES, Q_OFFS, Q_LENS, R2V_ENTRIES, R2V_OFFS, R2V_LENS, MID_O, MID_LSE,
       NODE_NUMS, NODE_OFFSETS, Q_TILES, KV_TILES, SM_SCALE, N_ARGS };

// (args tuple, logit_cap, path, o_lse | None, row ranges | None, partial rows named by q_entries or -1,
//  phase_info | None, kv_entries_aux | None, stream or -1 for torch's current one)
void fill(PyObject* const* x, ft_decode_args& a, c10::DeviceIndex& device) {
  memset(&a, 0, sizeof(a));
  if (!PyTuple_Check(x[0]) || PyTuple_GET_SIZE(x[0]) != N_ARGS) {
    PyErr_Format(PyExc_TypeError, "expected %d positional arguments", (int)N_ARGS);
    throw Refused();
  }
  auto arg = [&](int i) { return PyTuple_GET_ITEM(x[0], i); };
  const at::Tensor &q = tensor("q", arg(Q)), &k = tensor("k_buffer", arg(K)), &v = tensor("v_buffer", arg(V)),
                   &o = tensor("o", arg(O)), &mid_o = tensor("mid_o", arg(MID_O)), &mid_lse = tensor("mid_lse", arg(MID_LSE));
  if (q.dim() != 3 || o.dim() != 3 || k.dim() != 3 || v.dim() != 3)
    refuse("%s", "q, o must be [batch, heads, head_dim] and k/v buffers [rows, kv_heads, head_dim]");
  const at::ScalarType dtype = q.scalar_type();
  if (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat) refuse("unsupported dtype %s", c10::toString(dtype));
  if (k.scalar_type() != dtype || v.scalar_type() != dtype || o.scalar_type() != dtype)
    refuse("%s", "q, k_buffer, v_buffer and o must share one dtype");
  if (q.size(2) != k.size(2) || q.size(2) != v.size(2)) refuse("%s", "head_dim of q, k_buffer and v_buffer differ");
  if (o.sizes() != q.sizes()) refuse("%s", "o must have the shape of q");
  if (mid_o.scalar_type() != at::kFloat || mid_lse.scalar_type() != at::kFloat) refuse("%s", "mid_o / mid_lse must be float32");
  if (mid_o.dim() != 3 || mid_lse.dim() != 2 || mid_lse.stride(1) != 1)
    refuse("%s", "mid_o must be [rows, heads, head_dim] and mid_lse [rows, heads]");
  const at::Tensor* rows[] = {&q, &k, &v, &o, &mid_o};
  const char* row_names[] = {"q", "k_buffer", "v_buffer", "o", "mid_o"};
  for (int i = 0; i < 5; ++i)
    if (rows[i]->stride(2) != 1) refuse("%s: the head_dim axis must be contiguous", row_names[i]);
  const int64_t batch = q.size(0), heads = q.size(1);
  if (mid_o.size(1) < heads || mid_o.size(2) != q.size(2) || mid_lse.size(1) < heads)
    refuse("%s", "mid_o / mid_lse are too small for the head count of q");
  if (k.sizes() != v.sizes()) refuse("%s", "k_buffer and v_buffer differ in shape");

  static const char* const table_names[] = {"vnode_to_kv_entries", "vnode_to_kv_offs",     "vnode_to_kv_lens",
                                            "vnode_to_q_entries",  "vnode_to_q_offs",      "vnode_to_q_lens",
                                            "req_to_vnode_entries", "req_to_vnode_offs",   "req_to_vnode_lens"};
  const int32_t* tab[9];
  int64_t len[9];
  for (int i = 0; i < 9; ++i) {
    const at::Tensor& t = table(table_names[i], arg(KV_ENTRIES + i));
    tab[i] = static_cast<const int32_t*>(t.data_ptr());
    len[i] = t.numel();
  }
  int64_t nums[2], offs[2], q_tiles[2], kv_tiles[2];
  pair("phase_node_nums", arg(NODE_NUMS), nums);
  task_sizes(arg(KV_LENS), a);
  pair("phase_node_offsets", arg(NODE_OFFSETS), offs);
  pair("phase_q_tile_sizes", arg(Q_TILES), q_tiles);
  pair("phase_kv_tile_sizes", arg(KV_TILES), kv_tiles);
  const bool on_device = x[6] != Py_None;
  if (on_device) {
    const at::Tensor& t = table("phase_info", x[6]);
    if (t.numel() < 4) refuse("%s", "phase_info needs four entries: n0, n1, o0, o1");
    a.device_phase_info = static_cast<const int32_t*>(t.data_ptr());
  }
  if (x[7] != Py_None) {
    const at::Tensor& t = table("kv_entries_aux", x[7]);
    a.vnode_to_kv_entries_aux = static_cast<const int32_t*>(t.data_ptr());
    a.kv_entries_aux_len = t.numel();
  }
  const int64_t vnodes = len[1];
  for (int ph = 0; ph < 2; ++ph)
    if (!on_device && (nums[ph] < 0 || offs[ph] < 0 || offs[ph] + nums[ph] > vnodes))
      refuse("%s", "phase_node_nums / phase_node_offsets do not fit the vnode tables");
  if (std::min({len[2], len[4], len[5]}) < vnodes) refuse("%s", "vnode tables differ in length");
  if (len[7] < batch || len[8] < batch) refuse("%s", "request tables are shorter than the batch");
  if (x[3] != Py_None) {
    const at::Tensor& t = tensor("o_lse", x[3]);
    if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.numel() < batch * heads)
      refuse("%s", "o_lse must be a contiguous float32 [batch, heads] tensor");
    a.o_lse = static_cast<float*>(t.data_ptr());
  }
  int64_t q_rows = PyLong_AsLongLong(x[5]);
  if (q_rows < 0) q_rows = len[3];
  if (x[4] != Py_None) {
    const at::Tensor& t = table("row ranges", x[4]);
    if (t.numel() < 2 * q_rows) refuse("%s", "the row-range table needs two entries per partial row");
    a.vnode_q_kv_ranges = static_cast<const int32_t*>(t.data_ptr());
  }

  a.q = q.data_ptr();
  a.k_buffer = k.data_ptr();
  a.v_buffer = v.data_ptr();
  a.o = o.data_ptr();
  a.dtype = dtype == at::kHalf ? FT_F16 : dtype == at::kBFloat16 ? FT_BF16 : FT_F32;
  a.batch = (int32_t)batch;
  a.num_qo_heads = (int32_t)heads;
  a.head_dim = (int32_t)q.size(2);
  a.num_kv_heads = (int32_t)k.size(1);
  a.path = (int32_t)PyLong_AsLong(x[2]);
  a.kv_rows = k.size(0);
  a.q_stride0 = q.stride(0), a.q_stride1 = q.stride(1);
  a.k_stride0 = k.stride(0), a.k_stride1 = k.stride(1);
  a.v_stride0 = v.stride(0), a.v_stride1 = v.stride(1);
  a.o_stride0 = o.stride(0), a.o_stride1 = o.stride(1);
  a.vnode_to_kv_entries = tab[0];
  a.vnode_to_kv_offs = tab[1];
  a.vnode_to_kv_lens = const_cast<int32_t*>(tab[2]);
  a.vnode_to_q_entries = tab[3];
  a.vnode_to_q_offs = tab[4];
  a.vnode_to_q_lens = tab[5];
  a.req_to_vnode_entries = tab[6];
  a.req_to_vnode_offs = tab[7];
  a.req_to_vnode_lens = tab[8];
  a.kv_entries_len = len[0];
  a.num_partial_rows = std::min({mid_o.size(0), mid_lse.size(0), q_rows});
  for (int ph = 0; ph < 2; ++ph) {
    a.phase_node_nums[ph] = (int32_t)nums[ph];
    a.phase_node_offsets[ph] = (int32_t)offs[ph];
    a.phase_q_tile_sizes[ph] = (int32_t)q_tiles[ph];
    a.phase_kv_tile_sizes[ph] = (int32_t)kv_tiles[ph];
  }
  a.mid_o = static_cast<float*>(mid_o.data_ptr());
  a.mid_lse = static_cast<float*>(mid_lse.data_ptr());
  a.mid_o_stride0 = mid_o.stride(0), a.mid_o_stride1 = mid_o.stride(1);
  a.mid_lse_stride0 = mid_lse.stride(0);
  a.sm_scale = (float)PyFloat_AsDouble(arg(SM_SCALE));
  a.logit_cap = (float)PyFloat_AsDouble(x[1]);
  const long long stream = PyLong_AsLongLong(x[8]);
  if (PyErr_Occurred()) throw Refused();
  device = q.device().index();
  a.stream = stream != -1 ? reinterpret_cast<void*>(stream) : static_cast<void*>(c10::cuda::getCurrentCUDAStream(device).stream());
}

constexpr int N_FILL = 9;

// args(...) -> bytes of the filled ft_decode_args
PyObject* py_args(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != N_FILL) return PyErr_Format(PyExc_TypeError, "args() takes %d arguments", N_FILL);
  try {
    ft_decode_args a;
    c10::DeviceIndex device;
    fill(x, a, device);
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&a), sizeof(a));
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

// call(entry, ...as args()) -> status of the C-ABI call, on the device of q
PyObject* py_call(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 1 + N_FILL) return PyErr_Format(PyExc_TypeError, "call() takes %d arguments", 1 + N_FILL);
  const long entry = PyLong_AsLong(x[0]);
  if (entry < 0 || entry > 2 || g_entry[entry] == nullptr) return PyErr_Format(PyExc_ValueError, "unknown entry");
  try {
    ft_decode_args a;
    c10::DeviceIndex device;
    fill(x + 1, a, device);
    int rc;
    {
      const c10::cuda::CUDAGuard guard(device);
      Py_BEGIN_ALLOW_THREADS
      rc = g_entry[entry](&a);
      Py_END_ALLOW_THREADS
    }
    return PyLong_FromLong(rc);
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

// ---- new tokens (ft_append, ft_extend)

int dtype_code(at::ScalarType t) {
  if (t != at::kHalf && t != at::kBFloat16 && t != at::kFloat) refuse("unsupported dtype %s", c10::toString(t));
  return t == at::kHalf ? FT_F16 : t == at::kBFloat16 ? FT_BF16 : FT_F32;
}

// a [rows, heads, head_dim] tensor of the call's dtype and device
const at::Tensor& rows_of(const char* name, PyObject* o, const at::Tensor* like) {
  const at::Tensor& t = tensor(name, o);
  if (t.dim() != 3) refuse("%s must have three axes: rows, heads, head_dim", name);
  if (t.size(2) > 1 && t.stride(2) != 1) refuse("%s: the head_dim axis must be contiguous", name);
  if (like != nullptr && t.scalar_type() != like->scalar_type()) refuse("%s: all of the call's tensors must share one dtype", name);
  if (like != nullptr && t.device() != like->device()) refuse("%s is on another device than the call's other tensors", name);
  return t;
}

const at::Tensor& on_device_of(const char* name, const at::Tensor& t, const at::Tensor& like) {
  if (t.device() != like.device()) refuse("%s is on another device than the call's other tensors", name);
  return t;
}

// int32 or int64, the last axis contiguous
const at::Tensor& indices(const char* name, PyObject* o, const at::Tensor& like) {
  const at::Tensor& t = on_device_of(name, tensor(name, o), like);
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) refuse("%s must be int32 or int64, got %s", name, c10::toString(t.scalar_type()));
  if (t.dim() < 1 || (t.size(-1) > 1 && t.stride(-1) != 1)) refuse("%s must be contiguous along its tokens", name);
  return t;
}

template <typename Args, typename Fn>
PyObject* launch_on(const at::Tensor& like, Args& a, Fn fn) {
  const c10::DeviceIndex device = like.device().index();
  a.stream = static_cast<void*>(c10::cuda::getCurrentCUDAStream(device).stream());
  int rc;
  {
    const c10::cuda::CUDAGuard guard(device);
    Py_BEGIN_ALLOW_THREADS
    rc = fn(&a);
    Py_END_ALLOW_THREADS
  }
  return PyLong_FromLong(rc);
}

// append(q | None, k, v, k_buffer, v_buffer, slots, q_out | None, positions | None, cos_sin | None, sections | None, interleaved)
PyObject* py_append(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 11) return PyErr_Format(PyExc_TypeError, "append() takes 11 arguments");
  try {
    ft_append_args a;
    memset(&a, 0, sizeof(a));
    const at::Tensor& k = rows_of("k", x[1], nullptr);
    const at::Tensor &v = rows_of("v", x[2], &k), &kb = rows_of("k_buffer", x[3], &k), &vb = rows_of("v_buffer", x[4], &k);
    a.dtype = dtype_code(k.scalar_type());
    if (v.sizes() != k.sizes()) refuse("%s", "k and v differ in shape");
    if (kb.sizes() != vb.sizes()) refuse("%s", "k_buffer and v_buffer differ in shape");
    if (kb.size(1) != k.size(1) || kb.size(2) != k.size(2)) refuse("%s", "k and k_buffer differ in heads or head_dim");
    const int64_t tokens = k.size(0);
    if (tokens > INT32_MAX) refuse("%s", "too many tokens for one call");
    if (x[0] != Py_None) {
      const at::Tensor& q = rows_of("q", x[0], &k);
      const at::Tensor& qo = x[6] != Py_None ? rows_of("q_out", x[6], &k) : q;
      if (q.size(0) != tokens || q.size(2) != k.size(2)) refuse("%s", "q and k differ in tokens or head_dim");
      if (qo.sizes() != q.sizes()) refuse("%s", "q_out must have the shape of q");
      a.q = q.data_ptr(), a.q_out = qo.data_ptr();
      a.num_qo_heads = (int32_t)q.size(1);
      a.q_stride0 = q.stride(0), a.q_stride1 = q.stride(1), a.q_out_stride0 = qo.stride(0), a.q_out_stride1 = qo.stride(1);
    } else if (x[6] != Py_None) {
      refuse("%s", "q_out is given without q");
    }
    const at::Tensor& slots = indices("slots", x[5], k);
    if (slots.dim() != 1 || slots.size(0) != tokens) refuse("%s", "slots must have one entry per token");
    a.slots = slots.data_ptr(), a.slots_64 = slots.scalar_type() == at::kLong;
    if ((x[7] == Py_None) != (x[8] == Py_None)) refuse("%s", "positions and cos_sin go together");
    if (x[7] != Py_None) {
      const at::Tensor& pos = indices("positions", x[7], k);
      const at::Tensor& table = on_device_of("cos_sin", tensor("cos_sin", x[8]), k);
      if (table.scalar_type() != at::kFloat || table.dim() != 2 || (table.size(1) > 1 && table.stride(1) != 1))
        refuse("%s", "cos_sin must be a float32 [positions, rot_dim] tensor with contiguous rows");
      if (pos.dim() > 2 || pos.size(-1) != tokens) refuse("%s", "positions must be [tokens] or [axes, tokens]");
      const int64_t axes = pos.dim() == 2 ? pos.size(0) : 1;
      if (axes < 1 || axes > 4) refuse("%s", "positions have one to four axes");
      if (table.size(1) > k.size(2) || table.size(1) % 2 != 0 || table.size(1) == 0)
        refuse("%s", "cos_sin: rot_dim must be even and at most head_dim");
      a.rot_dim = (int32_t)table.size(1), a.num_axes = (int32_t)axes;
      if (x[9] != Py_None) {
        PyObject* seq = PySequence_Fast(x[9], "sections must be a sequence of integers");
        if (seq == nullptr) throw Refused();
        const Py_ssize_t len = PySequence_Fast_GET_SIZE(seq);
        for (Py_ssize_t i = 0; i < len && i < 4; ++i) {
          const long s = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
          a.sections[i] = s < 0 ? -1 : s > 1 << 20 ? 1 << 20 : (int32_t)s;
        }
        Py_DECREF(seq);
        if (PyErr_Occurred()) throw Refused();
        if (len != axes) refuse("%s", "sections must have one entry per axis of positions");
      } else {
        if (axes != 1) refuse("%s", "positions with several axes need sections");
        a.sections[0] = a.rot_dim / 2;
      }
      int64_t pairs = 0;
      for (int i = 0; i < 4; ++i) {
        if (a.sections[i] < 0) refuse("%s", "sections must not be negative");
        pairs += a.sections[i];
      }
      if (pairs != a.rot_dim / 2) refuse("%s", "the sections must hold rot_dim / 2 pairs together");
      a.positions = pos.data_ptr(), a.positions_64 = pos.scalar_type() == at::kLong;
      a.positions_stride0 = pos.dim() == 2 ? pos.stride(0) : 0;
      a.cos_sin = static_cast<const float*>(table.data_ptr()), a.cos_sin_rows = table.size(0), a.cos_sin_stride0 = table.stride(0);
    } else if (x[9] != Py_None) {
      refuse("%s", "sections without positions");
    }
    a.interleaved = PyObject_IsTrue(x[10]);
    a.k = k.data_ptr(), a.v = v.data_ptr(), a.k_buffer = kb.data_ptr(), a.v_buffer = vb.data_ptr();
    a.tokens = (int32_t)tokens, a.num_kv_heads = (int32_t)k.size(1), a.head_dim = (int32_t)k.size(2), a.kv_rows = kb.size(0);
    a.k_stride0 = k.stride(0), a.k_stride1 = k.stride(1), a.v_stride0 = v.stride(0), a.v_stride1 = v.stride(1);
    a.k_buffer_stride0 = kb.stride(0), a.k_buffer_stride1 = kb.stride(1), a.v_buffer_stride0 = vb.stride(0), a.v_buffer_stride1 = vb.stride(1);
    if (PyErr_Occurred()) throw Refused();
    return launch_on(k, a, g_append);
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

// (q, k_buffer, v_buffer, o, kv_entries, plan table, plan info as bytes, sm_scale, logit_cap, o_lse | None, path) -> filled
// argument block; the scratch of a plan with partial rows is the call's own, from torch's allocator (`hold`)
void fill_extend(PyObject* const* x, ft_extend_args& a, at::Tensor& hold) {
  memset(&a, 0, sizeof(a));
  const at::Tensor& q = rows_of("q", x[0], nullptr);
  const at::Tensor &k = rows_of("k_buffer", x[1], &q), &v = rows_of("v_buffer", x[2], &q), &o = rows_of("o", x[3], &q);
  a.dtype = dtype_code(q.scalar_type());
  if (k.sizes() != v.sizes()) refuse("%s", "k_buffer and v_buffer differ in shape");
  if (o.sizes() != q.sizes()) refuse("%s", "o must have the shape of q");
  if (o.numel() > 0 && o.data_ptr() == q.data_ptr()) refuse("%s", "o must not be q: rows of q are read after rows of o are written");
  if (q.size(2) != k.size(2)) refuse("%s", "head_dim of q and k_buffer differ");
  const at::Tensor& entries = on_device_of("kv_entries", table("kv_entries", x[4]), q);
  const at::Tensor& plan = on_device_of("the plan", table("the plan", x[5]), q);
  char* info = nullptr;
  Py_ssize_t len = 0;
  if (PyBytes_AsStringAndSize(x[6], &info, &len) != 0) throw Refused();
  if (len != (Py_ssize_t)sizeof(a.plan)) refuse("%s", "the plan's description has another size than the library's");
  memcpy(&a.plan, info, sizeof(a.plan));
  if (a.plan.table_ints > plan.numel()) refuse("%s", "the plan's table is shorter than its description says");
  a.sm_scale = (float)PyFloat_AsDouble(x[7]);
  a.logit_cap = (float)PyFloat_AsDouble(x[8]);
  a.path = (int32_t)PyLong_AsLong(x[10]);
  if (PyErr_Occurred()) throw Refused();
  if (x[9] != Py_None) {
    const at::Tensor& t = on_device_of("o_lse", tensor("o_lse", x[9]), q);
    if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.dim() != 2 || t.size(0) != q.size(0) || t.size(1) != q.size(1))
      refuse("%s", "o_lse must be a contiguous float32 tensor with the rows and heads of q");
    a.o_lse = static_cast<float*>(t.data_ptr());
  }
  a.q = q.data_ptr(), a.k_buffer = k.data_ptr(), a.v_buffer = v.data_ptr(), a.o = o.data_ptr();
  a.num_qo_heads = (int32_t)q.size(1), a.num_kv_heads = (int32_t)k.size(1), a.head_dim = (int32_t)q.size(2);
  a.q_rows = q.size(0), a.kv_rows = k.size(0);
  a.q_stride0 = q.stride(0), a.q_stride1 = q.stride(1), a.k_stride0 = k.stride(0), a.k_stride1 = k.stride(1);
  a.v_stride0 = v.stride(0), a.v_stride1 = v.stride(1), a.o_stride0 = o.stride(0), a.o_stride1 = o.stride(1);
  a.kv_entries = static_cast<const int32_t*>(entries.data_ptr()), a.kv_entries_len = entries.numel();
  a.plan_table = static_cast<const int32_t*>(plan.data_ptr());
  if (a.plan.partial_rows > 0) {
    const int64_t lse = (int64_t)a.plan.partial_rows * a.num_qo_heads;
    hold = at::empty({lse * (a.head_dim + 1)}, q.options().dtype(at::kFloat));
    a.mid_o = static_cast<float*>(hold.data_ptr());
    a.mid_lse = a.mid_o + lse * a.head_dim;
  }
}

// extend_args(...as extend()) -> bytes of the filled ft_extend_args; its scratch is gone when the call returns
PyObject* py_extend_args(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 11) return PyErr_Format(PyExc_TypeError, "extend_args() takes 11 arguments");
  try {
    ft_extend_args a;
    at::Tensor hold;
    fill_extend(x, a, hold);
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&a), sizeof(a));
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

PyObject* py_extend(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 11) return PyErr_Format(PyExc_TypeError, "extend() takes 11 arguments");
  try {
    ft_extend_args a;
    at::Tensor hold;
    fill_extend(x, a, hold);
    return launch_on(THPVariable_Unpack(x[0]), a, g_extend);
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    return PyErr_Format(PyExc_RuntimeError, "%s", e.what());
  }
}

// bind(addresses of ft_decode, ft_stage1, ft_stage2, ft_append, ft_extend, sizes of their argument blocks in the library)
PyObject* py_bind(PyObject*, PyObject* const* x, Py_ssize_t n) {
  if (n != 8) return PyErr_Format(PyExc_TypeError, "bind() takes 8 arguments");
  if (PyLong_AsLong(x[5]) != (long)sizeof(ft_decode_args) || PyLong_AsLong(x[6]) != (long)sizeof(ft_append_args) ||
      PyLong_AsLong(x[7]) != (long)sizeof(ft_extend_args))
    return PyErr_Format(PyExc_RuntimeError, "the library's argument blocks differ from those this module was built with");
  for (int i = 0; i < 3; ++i) g_entry[i] = reinterpret_cast<DecodeFn>(PyLong_AsVoidPtr(x[i]));
  g_append = reinterpret_cast<int (*)(const ft_append_args*)>(PyLong_AsVoidPtr(x[3]));
  g_extend = reinterpret_cast<int (*)(const ft_extend_args*)>(PyLong_AsVoidPtr(x[4]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"args", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_args)), METH_FASTCALL, "filled ft_decode_args as bytes"},
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_call)), METH_FASTCALL, "check, fill and launch"},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_append)), METH_FASTCALL, "check, fill and launch ft_append"},
    {"extend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_extend)), METH_FASTCALL, "check, fill and launch ft_extend"},
    {"extend_args", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_extend_args)), METH_FASTCALL, "filled ft_extend_args as bytes"},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_bind)), METH_FASTCALL, "addresses of the C ABI"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "ft_call", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_ft_call(void) { return PyModule_Create(&module); }
