// The eager calls of the 4-bit and 8-bit caches, and of copies of blocks, from Python: arguments checked and read, outputs
// made and the C ABI called in one step.  A small batch's eager call is bound by the host: a launch costs it some 3.6 us,
// and checking 5 to 15 tensors attribute by attribute from Python another 4 to 5, with 1 for ctypes (decode of 4 x U[1,
// 512] through the layer: 12.7 us, so 8.1; a row written and read back 18.5, 9.0; a block copied in 28 layers 9.8, 5.1).
//
// Every function answers
//   its result   the call was made;
//   an int       the C ABI refused it or the launch failed: its status;
//   None         an argument is not plainly as it should be.  Nothing was done; the checks in _C.py then name it.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "nvamd.h"

namespace {

constexpr int64_t kHeadDim = 128;
constexpr int64_t kFp4RowBytes = 64, kFp4RowScales = 4, kFp8Tile = 16;

// The entry points of a kind of pages; those of the 8-bit cache have the same signatures.
struct Kind {
  PyTypeObject *pages;  // _C.Fp4Pages, _C.Fp8Pages
  decltype(&nvamd_kv_cache_write_fp4) write;
  decltype(&nvamd_kv_cache_read_fp4) read;
  decltype(&nvamd_qk_norm_rope_fp4) rope;
  decltype(&nvamd_paged_decode_fp4) decode;
  decltype(&nvamd_paged_decode_fused_fp4) fused;
  decltype(&nvamd_paged_prefill_fp4) prefill;
  decltype(&nvamd_paged_prefill_fp4_workspace_size) prefill_space;
};
constexpr int kFp4 = 0, kFp8 = 1;
Kind kinds[2];
decltype(&nvamd_copy_blocks) f_copy;
constexpr Py_ssize_t kMaxPools = 8;

struct Irregular {};  // thrown: answer None

void need(bool ok) {
  if (!ok) throw Irregular();
}

// A plain strided tensor (no subclass) on a GPU: on `device`, or on any, which it then names.
const at::Tensor &tensor(PyObject *o, int &device) {
  need(THPVariable_CheckExact(o));
  const at::Tensor &t = THPVariable_Unpack(o);
  need(t.is_cuda() && t.layout() == at::kStrided);
  if (device < 0) device = t.get_device();
  need(t.get_device() == device);
  return t;
}
const at::Tensor &dense(PyObject *o, int &device, at::ScalarType type) {
  const at::Tensor &t = tensor(o, device);
  need(t.scalar_type() == type && t.is_contiguous());
  return t;
}

struct Pages {
  void *kc, *ks, *vc, *vs;
  int64_t nb, bs, hkv;
  const Kind &kind;
};

int narrow(int64_t v) {
  need(v >= 0 && v <= 0x7fffffff);
  return (int)v;
}

Pages pages(PyObject *keys, PyObject *values, int &device) {
  const int is = Py_TYPE(keys) == kinds[kFp4].pages ? kFp4 : kFp8;
  need(Py_TYPE(keys) == kinds[is].pages && Py_TYPE(values) == kinds[is].pages);
  const at::Tensor &kc = dense(PyTuple_GET_ITEM(keys, 0), device, at::kByte);
  const at::Tensor &ks = dense(PyTuple_GET_ITEM(keys, 1), device, at::kByte);
  const at::Tensor &vc = dense(PyTuple_GET_ITEM(values, 0), device, at::kByte);
  const at::Tensor &vs = dense(PyTuple_GET_ITEM(values, 1), device, at::kByte);
  need(kc.dim() == 4 && kc.size(3) == (is == kFp4 ? kFp4RowBytes : kHeadDim) && vc.sizes() == kc.sizes());
  need(ks.dim() == (is == kFp4 ? 4 : 3) && ks.size(0) == kc.size(0) && ks.size(1) == kc.size(1) &&
       vs.sizes() == ks.sizes());
  need(is == kFp4 ? ks.size(2) == kc.size(2) && ks.size(3) == kFp4RowScales : ks.size(2) * kFp8Tile == kc.size(2));
  return {kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), kc.size(0), kc.size(2), kc.size(1), kinds[is]};
}

struct Rows {
  void *p;
  int64_t stride, rows, heads;
};
// [rows, heads, 128] of bf16, dense but for the stride between rows; -1: any number.
Rows rows_of(PyObject *o, int &device, int64_t rows, int64_t heads) {
  const at::Tensor &t = tensor(o, device);
  need(t.scalar_type() == at::kBFloat16 && t.dim() == 3 && t.size(2) == kHeadDim);
  need((rows < 0 || t.size(0) == rows) && (heads < 0 || t.size(1) == heads) && t.size(0) > 0 && t.size(1) > 0);
  need(t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == kHeadDim));
  const int64_t dense_row = t.size(1) * kHeadDim;
  // a single row's stride says nothing
  return {t.data_ptr(), t.size(0) > 1 || t.stride(0) > dense_row ? t.stride(0) : dense_row, t.size(0), t.size(1)};
}
const int64_t *indices(PyObject *o, int &device, int64_t rows) {
  const at::Tensor &t = dense(o, device, at::kLong);
  need(t.dim() == 1 && (rows < 0 || t.size(0) == rows));
  return t.data_ptr<int64_t>();
}
const int32_t *lengths(PyObject *o, int &device, int64_t least, bool exact) {
  const at::Tensor &t = dense(o, device, at::kInt);
  need(t.dim() == 1 && (exact ? t.size(0) == least : t.size(0) >= least));
  return t.data_ptr<int32_t>();
}

struct Table {
  const int32_t *p;
  int stride, width;
};
Table table_of(PyObject *o, int &device, int64_t least, bool exact) {
  const at::Tensor &t = tensor(o, device);
  need(t.scalar_type() == at::kInt && t.dim() == 2 && (exact ? t.size(0) == least : t.size(0) >= least));
  need(t.size(1) > 0 && (t.stride(1) == 1 || t.size(1) == 1));
  need(t.size(0) <= 1 || t.stride(0) >= t.size(1));
  // a single row's stride says nothing
  return {t.data_ptr<int32_t>(), narrow(t.stride(0) > t.size(1) ? t.stride(0) : t.size(1)), narrow(t.size(1))};
}

int integer(PyObject *o) {
  need(PyLong_CheckExact(o));
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  need(overflow == 0);
  return narrow(v);
}
float number(PyObject *o) {
  need(PyFloat_CheckExact(o));
  return (float)PyFloat_AS_DOUBLE(o);
}

// The current stream, on whose device the tensors have to be.
hipStream_t stream_on(int device) {
  need(c10::hip::current_device() == device);
  return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream();
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)device));
}

// The rows given for a result, or new ones like q's.
Rows result(PyObject *o, int device, const Rows &q, at::Tensor &made) {
  if (o != Py_None) return rows_of(o, device, q.rows, q.heads);
  made = empty({q.rows, q.heads, kHeadDim}, at::kBFloat16, device);
  return {made.data_ptr(), q.heads * kHeadDim, q.rows, q.heads};
}

struct Rope {
  const void *qw, *kw;
  const int64_t *positions;
  const float *table;
  int rows;
  float eps;
};
// q_weight, k_weight, positions, cos_sin, eps
Rope rope_of(PyObject *const *a, int &device, int64_t rows) {
  const at::Tensor &qw = dense(a[0], device, at::kBFloat16), &kw = dense(a[1], device, at::kBFloat16);
  need(qw.dim() == 1 && qw.size(0) == kHeadDim && kw.dim() == 1 && kw.size(0) == kHeadDim);
  const int64_t *positions = indices(a[2], device, rows);
  const at::Tensor &table = dense(a[3], device, at::kFloat);
  need(table.dim() == 2 && table.size(1) == kHeadDim);
  return {qw.data_ptr(), kw.data_ptr(), positions, table.data_ptr<float>(), narrow(table.size(0)), number(a[4])};
}

template <typename F>
int call(F &&f) {  // other threads run meanwhile: a full queue makes a launch wait
  PyThreadState *state = PyEval_SaveThread();
  const int status = f();
  PyEval_RestoreThread(state);
  return status;
}

PyObject *same(PyObject *o) {
  Py_INCREF(o);
  return o;
}

// (key_states, value_states, key_pages, value_pages, slot_mapping) -> True
PyObject *write(PyObject *const *a) {
  int dev = -1;
  const Pages c = pages(a[2], a[3], dev);
  const Rows k = rows_of(a[0], dev, -1, c.hkv), v = rows_of(a[1], dev, k.rows, c.hkv);
  const int64_t *slots = indices(a[4], dev, k.rows);
  const int nb = narrow(c.nb), bs = narrow(c.bs), t = narrow(k.rows), hkv = narrow(c.hkv);
  hipStream_t s = stream_on(dev);
  const int status = call([&] {
    return c.kind.write(k.p, k.stride, v.p, v.stride, c.kc, c.ks, c.vc, c.vs, nb, bs, slots, t, hkv, kHeadDim, s);
  });
  return status ? PyLong_FromLong(status) : same(Py_True);
}

// (key_pages, value_pages, slot_mapping) -> (keys, values)
PyObject *read(PyObject *const *a) {
  int dev = -1;
  const Pages c = pages(a[0], a[1], dev);
  const int64_t *slots = indices(a[2], dev, -1);
  const int64_t t = THPVariable_Unpack(a[2]).size(0);
  const int nb = narrow(c.nb), bs = narrow(c.bs), n = narrow(t), hkv = narrow(c.hkv);
  hipStream_t s = stream_on(dev);
  at::Tensor k = empty({t, c.hkv, kHeadDim}, at::kBFloat16, dev), v = empty({t, c.hkv, kHeadDim}, at::kBFloat16, dev);
  const int64_t stride = c.hkv * kHeadDim;
  const int status = call([&] {
    return c.kind.read(k.data_ptr(), stride, v.data_ptr(), stride, c.kc, c.ks, c.vc, c.vs, nb, bs, slots, n, hkv, kHeadDim, s);
  });
  if (status) return PyLong_FromLong(status);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
}

// (q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages, slot_mapping, q_out, k_out) -> q_out;
// q_out None: a new one, k_out None: none
PyObject *rope(PyObject *const *a) {
  int dev = -1;
  const Pages c = pages(a[8], a[9], dev);
  const Rows q = rows_of(a[0], dev, -1, -1), k = rows_of(a[1], dev, q.rows, c.hkv), v = rows_of(a[2], dev, q.rows, c.hkv);
  const Rope r = rope_of(a + 3, dev, q.rows);
  const int64_t *slots = indices(a[10], dev, q.rows);
  Rows ko = {nullptr, 0, 0, 0};
  if (a[12] != Py_None) {
    ko = rows_of(a[12], dev, q.rows, c.hkv);
    need(ko.p != k.p || ko.stride == k.stride);
  }
  const int nb = narrow(c.nb), bs = narrow(c.bs), t = narrow(q.rows), hq = narrow(q.heads), hkv = narrow(c.hkv);
  hipStream_t s = stream_on(dev);
  at::Tensor made;
  const Rows qo = result(a[11], dev, q, made);
  need(qo.p != q.p || qo.stride == q.stride);
  const int status = call([&] {
    return c.kind.rope(qo.p, qo.stride, ko.p, ko.stride, q.p, q.stride, k.p, k.stride, v.p, v.stride, r.qw, r.kw,
                  r.positions, r.table, r.rows, c.kc, c.ks, c.vc, c.vs, nb, bs, slots, t, hq, hkv, kHeadDim, r.eps, s);
  });
  if (status) return PyLong_FromLong(status);
  return made.defined() ? THPVariable_Wrap(std::move(made)) : same(a[11]);
}

// (out, q, key_pages, value_pages, block_tables, context_lens, scale, max_context_len, workspace) -> out; out None: a
// new one
PyObject *decode(PyObject *const *a) {
  int dev = -1;
  const Pages c = pages(a[2], a[3], dev);
  const Rows q = rows_of(a[1], dev, -1, -1);
  const Table bt = table_of(a[4], dev, q.rows, true);
  const int32_t *lens = lengths(a[5], dev, q.rows, true);
  const float scale = number(a[6]);
  const int most = integer(a[7]);
  const at::Tensor &space = tensor(a[8], dev);
  need(space.is_contiguous());
  const int nb = narrow(c.nb), bs = narrow(c.bs), t = narrow(q.rows), hq = narrow(q.heads), hkv = narrow(c.hkv);
  hipStream_t s = stream_on(dev);
  at::Tensor made;
  const Rows out = result(a[0], dev, q, made);
  const int status = call([&] {
    return c.kind.decode(out.p, out.stride, q.p, q.stride, c.kc, c.ks, c.vc, c.vs, nb, bs, bt.p, bt.stride, bt.width, lens, t,
                    hq, hkv, kHeadDim, scale, most, space.data_ptr(), space.nbytes(), s);
  });
  if (status) return PyLong_FromLong(status);
  return made.defined() ? THPVariable_Wrap(std::move(made)) : same(a[0]);
}

// (out, q, k, v, q_weight, k_weight, positions, cos_sin, eps, key_pages, value_pages, slot_mapping, block_tables,
// context_lens, scale, max_context_len, workspace) -> out; out None: a new one
PyObject *decode_fused(PyObject *const *a) {
  int dev = -1;
  const Pages c = pages(a[9], a[10], dev);
  const Rows q = rows_of(a[1], dev, -1, -1), k = rows_of(a[2], dev, q.rows, c.hkv), v = rows_of(a[3], dev, q.rows, c.hkv);
  const Rope r = rope_of(a + 4, dev, q.rows);
  const int64_t *slots = indices(a[11], dev, q.rows);
  const Table bt = table_of(a[12], dev, q.rows, true);
  const int32_t *lens = lengths(a[13], dev, q.rows, true);
  const float scale = number(a[14]);
  const int most = integer(a[15]);
  const at::Tensor &space = tensor(a[16], dev);
  need(space.is_contiguous());
  const int nb = narrow(c.nb), bs = narrow(c.bs), t = narrow(q.rows), hq = narrow(q.heads), hkv = narrow(c.hkv);
  hipStream_t s = stream_on(dev);
  at::Tensor made;
  const Rows out = result(a[0], dev, q, made);
  const int status = call([&] {
    return c.kind.fused(out.p, out.stride, q.p, q.stride, k.p, k.stride, v.p, v.stride, r.qw, r.kw, r.positions, r.table, r.rows,
                   r.eps, c.kc, c.ks, c.vc, c.vs, nb, bs, slots, bt.p, bt.stride, bt.width, lens, t, hq, hkv, kHeadDim,
                   scale, most, space.data_ptr(), space.nbytes(), s);
  });
  if (status) return PyLong_FromLong(status);
  return made.defined() ? THPVariable_Wrap(std::move(made)) : same(a[0]);
}

// (out, q, key_pages, value_pages, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale) -> out
PyObject *prefill(PyObject *const *a) {
  int dev = -1;
  const Pages c = pages(a[2], a[3], dev);
  const Rows q = rows_of(a[1], dev, -1, -1), out = rows_of(a[0], dev, q.rows, q.heads);
  const int32_t *cu = lengths(a[5], dev, 1, false);
  const int n = narrow(THPVariable_Unpack(a[5]).size(0) - 1);
  const Table bt = table_of(a[4], dev, n, false);
  const int32_t *lens = lengths(a[6], dev, n, false);
  const int most = integer(a[7]);
  const float scale = number(a[8]);
  const int nb = narrow(c.nb), bs = narrow(c.bs), t = narrow(q.rows), hq = narrow(q.heads), hkv = narrow(c.hkv);
  hipStream_t s = stream_on(dev);
  const size_t bytes = c.kind.prefill_space(n, most, hq, hkv, bs, bt.width);
  at::Tensor space;
  if (bytes) space = empty({(int64_t)bytes}, at::kByte, dev);  // freed behind the call on its stream
  void *p = bytes ? space.data_ptr() : nullptr;
  const int status = call([&] {
    return c.kind.prefill(out.p, out.stride, q.p, q.stride, c.kc, c.ks, c.vc, c.vs, nb, bs, bt.p, bt.stride, bt.width, cu, lens,
                     n, t, most, hq, hkv, kHeadDim, scale, p, bytes, s);
  });
  return status ? PyLong_FromLong(status) : same(a[0]);
}

// (pools, sources, targets) -> True; pools a list or a tuple
PyObject *copy(PyObject *const *a) {
  need(PyList_CheckExact(a[0]) || PyTuple_CheckExact(a[0]));
  PyObject *const *pools = PySequence_Fast_ITEMS(a[0]);
  const Py_ssize_t n_pools = PySequence_Fast_GET_SIZE(a[0]);
  need(n_pools > 0 && n_pools <= kMaxPools);
  int dev = -1;
  void *at[kMaxPools];
  int64_t bytes[kMaxPools], layers = 0, blocks = 0;
  for (Py_ssize_t i = 0; i < n_pools; ++i) {
    const at::Tensor &t = tensor(pools[i], dev);
    need(t.dim() >= 3 && t.is_contiguous() && t.numel() > 0);
    if (i == 0) layers = t.size(0), blocks = t.size(1);
    need(t.size(0) == layers && t.size(1) == blocks);
    at[i] = t.data_ptr();
    bytes[i] = (int64_t)t.nbytes() / (layers * blocks);  // a single block's stride says nothing
  }
  const int32_t *sources = lengths(a[1], dev, 0, false);
  const int64_t n = THPVariable_Unpack(a[1]).size(0);
  const int32_t *targets = lengths(a[2], dev, n, true);
  const int l = narrow(layers), nb = narrow(blocks), count = narrow(n);
  hipStream_t s = stream_on(dev);
  const int status = call([&] { return f_copy(at, bytes, (int)n_pools, l, nb, sources, targets, count, s); });
  return status ? PyLong_FromLong(status) : same(Py_True);
}

template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) Py_RETURN_NONE;
  try {
    return F(args);
  } catch (const Irregular &) {
    Py_RETURN_NONE;
  } catch (const std::exception &) {  // of an allocation or a device query: raised as torch raises it
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// (address of nvamd_copy_blocks)
PyObject *bind_copy(PyObject *, PyObject *arg) {
  const unsigned long long p = PyLong_AsUnsignedLongLong(arg);
  if (PyErr_Occurred()) return nullptr;
  f_copy = reinterpret_cast<decltype(f_copy)>(p);
  Py_RETURN_NONE;
}

// (index, type of the pages, addresses of its entry points)
PyObject *bind(PyObject *, PyObject *args) {
  int index;
  PyObject *type;
  unsigned long long p[7];
  if (!PyArg_ParseTuple(args, "iO!KKKKKKK", &index, &PyType_Type, &type, &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6]))
    return nullptr;
  if (index != kFp4 && index != kFp8) {
    PyErr_SetString(PyExc_ValueError, "no such kind of pages");
    return nullptr;
  }
  Kind &k = kinds[index];
  k.write = reinterpret_cast<decltype(k.write)>(p[0]);
  k.read = reinterpret_cast<decltype(k.read)>(p[1]);
  k.rope = reinterpret_cast<decltype(k.rope)>(p[2]);
  k.decode = reinterpret_cast<decltype(k.decode)>(p[3]);
  k.fused = reinterpret_cast<decltype(k.fused)>(p[4]);
  k.prefill = reinterpret_cast<decltype(k.prefill)>(p[5]);
  k.prefill_space = reinterpret_cast<decltype(k.prefill_space)>(p[6]);
  Py_INCREF(type);
  Py_XDECREF(reinterpret_cast<PyObject *>(k.pages));
  k.pages = reinterpret_cast<PyTypeObject *>(type);
  Py_RETURN_NONE;
}

#define ENTRY(name, args) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name, args>)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"bind_copy", bind_copy, METH_O, nullptr},
    ENTRY(write, 5), ENTRY(read, 3), ENTRY(rope, 13), ENTRY(decode, 9), ENTRY(decode_fused, 17),
    ENTRY(prefill, 9), ENTRY(copy, 3),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject *m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddIntConstant(m, "ABI_VERSION", NVAMD_ABI_VERSION) < 0) Py_CLEAR(m);
  return m;
}
