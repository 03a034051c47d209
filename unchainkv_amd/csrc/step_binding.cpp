// The step calls' arguments, from Python tensors to the C entries: what splitzip_cuda's rotate_write_kv_paged,
// cross_attention_paged, cross_attention, beam_select and reorder_beams_paged check, allocate and pass on. A
// small call is bound by its host time, of which tensors' attributes read one by one from Python took more than
// the launch: us a call with them and with this, rotate_write_kv_paged 13.2 and 6, beam_select (two launches) 17.3
// and 12, reorder_beams_paged of 16 layers (two launches) 26.5 and 14.5. Each function takes the entries' addresses
// first and the stream last, and gives the results, None where the call is declined, or -1 where the entry failed;
// an argument that is no tensor raises TypeError.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <Python.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <vector>

namespace {

typedef unsigned long long u64;

constexpr u64 kDeclined = 0;

const at::Tensor& tensor_of(PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), "a tensor is wanted, not ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

at::Tensor maybe_tensor(PyObject* o) { return o == Py_None ? at::Tensor() : tensor_of(o); }

u64 number_of(PyObject* o) {
  const u64 v = PyLong_AsUnsignedLongLong(o);
  if (v == ~0ull && PyErr_Occurred() != nullptr) throw python_error();
  return v;
}

u64 address(const at::Tensor& t) { return t.defined() ? reinterpret_cast<u64>(t.data_ptr()) : 0; }

template <typename Entry, typename... Args>
long long enter(u64 entry, Args... args) {
  long long got;
  Py_BEGIN_ALLOW_THREADS
  got = reinterpret_cast<Entry>(entry)(args...);
  Py_END_ALLOW_THREADS
  return got;
}

// bf16 0, fp16 1; -1 for other types
int row_dtype(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : -1;
}

bool alike(const at::Tensor& t, const at::Tensor& q) {
  return t.scalar_type() == q.scalar_type() && t.device() == q.device();
}

// (rows, heads, head_dim) with whole head rows
bool rows_ok(const at::Tensor& t, const at::Tensor& q) {
  return alike(t, q) && t.dim() == 3 && (t.size(2) == 1 || t.stride(2) == 1);
}

// a contiguous (2, num_blocks, block_tokens, kv_heads, head_dim) layer
bool layer_ok(const at::Tensor& t, at::ScalarType dtype, at::Device device) {
  return t.scalar_type() == dtype && t.device() == device && t.dim() == 5 && t.size(0) == 2 && t.numel() > 0 &&
         t.is_contiguous();
}

// a contiguous vector of at least `count` values
bool vector_ok(const at::Tensor& t, at::Device device, int64_t count, at::ScalarType dtype) {
  return t.scalar_type() == dtype && t.dim() == 1 && t.is_contiguous() && t.device() == device && t.numel() >= count;
}

bool matrix_ok(const at::Tensor& t, at::IntArrayRef sizes, at::Device device, at::ScalarType dtype) {
  return t.scalar_type() == dtype && t.sizes() == sizes && t.device() == device && t.is_contiguous();
}

// Whether autograd follows any of them: a gradient is required while gradients are recorded, or there is a
// forward-mode tangent.
bool tracked(const at::Tensor& t) {
  return t.defined() && ((t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined());
}
bool tracked(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (tracked(*t)) return true;
  return false;
}

// A kernel's write into a caller's tensor, counted as torch's in-place operations are. (An inference tensor, for
// which nothing can have been saved, has no count.)
void wrote(const at::Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// `given`, if it is a workspace of `need` bytes, or a new one.
at::Tensor workspace_of(const at::Tensor& given, u64 need, at::Device device) {
  if (given.defined() && given.scalar_type() == at::kByte && given.is_contiguous() && given.device() == device &&
      (u64)given.numel() >= need)
    return given;
  return at::empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte).device(device));
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* got = PyTuple_New((Py_ssize_t)tensors.size());
  if (got == nullptr) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(got, i++, THPVariable_Wrap(t));
  return got;
}

// declined: None; failed: -1; done: `make()`
template <typename Make>
PyObject* answer(long long got, Make make) {
  if (got < 0) return PyLong_FromLong(-1);
  return got == 0 ? none() : make();
}

bool count_ok(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, got);
  return false;
}

// entry, q, k, v, kv_layer, slots, positions, rotation, interleaved, out, stream
PyObject* rotate_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count_ok(n, 11)) return nullptr;
  const u64 entry = number_of(args[0]), stream = number_of(args[10]);
  const at::Tensor &q = tensor_of(args[1]), &k = tensor_of(args[2]), &v = tensor_of(args[3]),
                   &kv = tensor_of(args[4]), &slots = tensor_of(args[5]), &positions = tensor_of(args[6]),
                   &rotation = tensor_of(args[7]);
  const int adjacent = PyObject_IsTrue(args[8]);
  if (adjacent < 0) throw python_error();
  at::Tensor out = maybe_tensor(args[9]);
  const bool given = out.defined();
  const int dtype = row_dtype(q);
  const at::Device device = q.device();
  if (dtype < 0 || !rows_ok(q, q) || !rows_ok(k, q) || !rows_ok(v, q) || !layer_ok(kv, q.scalar_type(), device))
    return none();
  const int64_t tokens = q.size(0), q_heads = q.size(1), dim = q.size(2), heads = kv.size(3);
  const std::array<int64_t, 3> rows = {tokens, heads, dim};
  if (k.sizes() != at::IntArrayRef(rows) || v.sizes() != at::IntArrayRef(rows) || kv.size(4) != dim ||
      !vector_ok(slots, device, tokens, at::kLong) || !vector_ok(positions, device, tokens, at::kLong) ||
      rotation.scalar_type() != at::kFloat || rotation.dim() != 2 || rotation.device() != device ||
      !rotation.is_contiguous() || tracked({&q, &k, &v, &kv, &rotation, &out}) ||
      (given && !matrix_ok(out, q.sizes(), device, q.scalar_type())))
    return none();
  if (!given) out = at::empty(q.sizes(), q.options());
  if (tokens == 0) return THPVariable_Wrap(out);
  const u64 places = (u64)(kv.size(1) * kv.size(2));
  typedef long long (*Entry)(u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64,
                             u64, u64, u64, u64, u64, u64, u64);
  const long long got = enter<Entry>(
      entry, address(q), (u64)(2 * q.stride(0)), (u64)(2 * q.stride(1)), (u64)q_heads, address(k),
      (u64)(2 * k.stride(0)), (u64)(2 * k.stride(1)), address(v), (u64)(2 * v.stride(0)), (u64)(2 * v.stride(1)),
      (u64)tokens, (u64)heads, (u64)dim, (u64)dtype, address(kv), 2 * places * (u64)(heads * dim), places,
      address(slots), address(positions), address(rotation), (u64)rotation.size(0), (u64)rotation.size(1),
      (u64)adjacent, address(out), stream);
  return answer(got, [&] {
    wrote(kv);
    if (given) wrote(out);
    return THPVariable_Wrap(out);
  });
  END_HANDLE_TH_ERRORS
}

int64_t count_of(PyObject* o, int64_t otherwise) {
  if (o == Py_None) return otherwise;
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred() != nullptr) throw python_error();
  return std::min<int64_t>(v, otherwise);
}

// An attention call's scale, head_dim ** -0.5 where none is given.
float scale_of(PyObject* o, int64_t dim) {
  if (o == Py_None) return (float)(1. / std::sqrt((double)dim));
  const double v = PyFloat_AsDouble(o);
  if (v == -1. && PyErr_Occurred() != nullptr) throw python_error();
  return (float)v;
}

// An attention call's results: as q, and f32 for its rows and heads.
bool results_ok(const at::Tensor& q, const at::Tensor& out, const at::Tensor& lse) {
  const std::array<int64_t, 2> rows = {q.size(0), q.size(1)};
  return (!out.defined() || matrix_ok(out, q.sizes(), q.device(), q.scalar_type())) &&
         (!lse.defined() || matrix_ok(lse, rows, q.device(), at::kFloat));
}

typedef u64 (*AttentionSize)(u64, u64, u64, u64, u64, u64, u64);

// entry, its workspace's size, q, kv_layer, tables, query_starts, source_tokens, max_query, scale, out, lse,
// workspace, stream
PyObject* cross_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count_ok(n, 13)) return nullptr;
  const u64 entry = number_of(args[0]), size = number_of(args[1]), stream = number_of(args[12]);
  const at::Tensor &q = tensor_of(args[2]), &kv = tensor_of(args[3]), &tables = tensor_of(args[4]),
                   &starts = tensor_of(args[5]), &source = tensor_of(args[6]);
  at::Tensor out = maybe_tensor(args[9]);
  const at::Tensor lse = maybe_tensor(args[10]), workspace = maybe_tensor(args[11]);
  const bool given = out.defined();
  const int dtype = row_dtype(q);
  const at::Device device = q.device();
  if (dtype < 0 || !rows_ok(q, q) || !layer_ok(kv, q.scalar_type(), device) || tracked({&q, &kv, &out, &lse}) ||
      tables.scalar_type() != at::kInt || tables.dim() != 2 || tables.device() != device)
    return none();
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  const int64_t requests = tables.size(0), width = tables.size(1);
  if (kv.size(4) != dim || (width != 1 && tables.stride(1) != 1) ||
      !vector_ok(starts, device, requests + 1, at::kInt) || !vector_ok(source, device, requests, at::kInt) ||
      !results_ok(q, out, lse))
    return none();
  const int64_t max_query = count_of(args[7], tokens);
  const float scale = scale_of(args[8], dim);
  if (!given) out = at::empty(q.sizes(), q.options());
  if (tokens == 0 || requests == 0) return THPVariable_Wrap(out);
  if (max_query <= 0 || width == 0) return none();
  const u64 need = reinterpret_cast<AttentionSize>(size)((u64)tokens, (u64)requests, (u64)heads, (u64)kv.size(3),
                                                         (u64)dim, (u64)(width * kv.size(2)), (u64)max_query);
  const at::Tensor space = need != 0 ? workspace_of(workspace, need, device) : at::Tensor();
  typedef long long (*Entry)(u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64,
                             u64, u64, u64, u64, float, u64);
  const long long got = enter<Entry>(
      entry, address(q), (u64)(2 * q.stride(0)), (u64)(2 * q.stride(1)), (u64)tokens, (u64)heads, (u64)kv.size(3),
      (u64)dim, (u64)dtype, address(kv), (u64)kv.size(1), (u64)kv.size(2), address(tables),
      (u64)(requests > 1 ? tables.stride(0) : width), (u64)width, address(starts), address(source), (u64)requests,
      (u64)max_query, address(out), address(lse), address(space), need, scale, stream);
  return answer(got, [&] {
    if (given) wrote(out);
    wrote(lse);
    return THPVariable_Wrap(out);
  });
  END_HANDLE_TH_ERRORS
}

// entry, its workspace's size, q, k, v, query_starts, source_starts, source_tokens, max_query, max_source, scale,
// out, lse, workspace, stream
PyObject* cross_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count_ok(n, 15)) return nullptr;
  const u64 entry = number_of(args[0]), size = number_of(args[1]), stream = number_of(args[14]);
  const at::Tensor &q = tensor_of(args[2]), &k = tensor_of(args[3]), &v = tensor_of(args[4]),
                   &starts = tensor_of(args[5]), &first = tensor_of(args[6]), &source = tensor_of(args[7]);
  at::Tensor out = maybe_tensor(args[11]);
  const at::Tensor lse = maybe_tensor(args[12]), workspace = maybe_tensor(args[13]);
  const bool given = out.defined();
  const int dtype = row_dtype(q);
  const at::Device device = q.device();
  if (dtype < 0 || !rows_ok(q, q) || !rows_ok(k, q) || !rows_ok(v, q) || tracked({&q, &k, &v, &out, &lse}))
    return none();
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2), rows = k.size(0), kv_heads = k.size(1);
  const int64_t requests = source.numel();
  if (k.sizes() != v.sizes() || k.size(2) != dim || dim == 0 || !vector_ok(source, device, 0, at::kInt) ||
      !vector_ok(first, device, requests, at::kInt) || !vector_ok(starts, device, requests + 1, at::kInt) ||
      !results_ok(q, out, lse))
    return none();
  const int64_t max_query = count_of(args[8], tokens), max_source = count_of(args[9], rows);
  const float scale = scale_of(args[10], dim);
  if (!given) out = at::empty(q.sizes(), q.options());
  if (tokens == 0 || requests == 0) return THPVariable_Wrap(out);
  if (max_query <= 0 || max_source < 0 || rows == 0) return none();
  const u64 need = reinterpret_cast<AttentionSize>(size)((u64)tokens, (u64)requests, (u64)heads, (u64)kv_heads,
                                                         (u64)dim, (u64)max_source, (u64)max_query);
  const at::Tensor space = need != 0 ? workspace_of(workspace, need, device) : at::Tensor();
  typedef long long (*Entry)(u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64,
                             u64, u64, u64, u64, u64, u64, u64, float, u64);
  const long long got = enter<Entry>(
      entry, address(q), (u64)(2 * q.stride(0)), (u64)(2 * q.stride(1)), address(k), (u64)(2 * k.stride(0)),
      (u64)(2 * k.stride(1)), address(v), (u64)(2 * v.stride(0)), (u64)(2 * v.stride(1)), (u64)rows, (u64)tokens,
      (u64)heads, (u64)kv_heads, (u64)dim, (u64)dtype, address(starts), address(first), address(source),
      (u64)requests, (u64)max_query, (u64)max_source, address(out), address(lse), address(space), need, scale,
      stream);
  return answer(got, [&] {
    if (given) wrote(out);
    wrote(lse);
    return THPVariable_Wrap(out);
  });
  END_HANDLE_TH_ERRORS
}

// entry, its workspace's size, logits, scores, candidates, ended, end_token, three results or None each,
// workspace, stream
PyObject* beam_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count_ok(n, 12)) return nullptr;
  const u64 entry = number_of(args[0]), size = number_of(args[1]), stream = number_of(args[11]);
  const at::Tensor &logits = tensor_of(args[2]), &scores = tensor_of(args[3]);
  const u64 candidates = number_of(args[4]);
  const at::Tensor ended = maybe_tensor(args[5]);
  const u64 end_token = number_of(args[6]);
  at::Tensor best = maybe_tensor(args[7]), parents = maybe_tensor(args[8]), tokens = maybe_tensor(args[9]);
  const at::Tensor workspace = maybe_tensor(args[10]);
  const int dtype = logits.scalar_type() == at::kFloat ? 2 : row_dtype(logits);
  if (dtype < 0 || logits.dim() != 3) return none();
  const at::Device device = logits.device();
  const int64_t requests = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  const std::array<int64_t, 2> rows = {requests, beams}, picked = {requests, (int64_t)candidates};
  const bool given = best.defined() || parents.defined() || tokens.defined();  // (all three, or it is declined)
  if ((vocab != 1 && logits.stride(2) != 1) || !matrix_ok(scores, rows, device, at::kFloat) ||
      (ended.defined() && (!matrix_ok(ended, rows, device, at::kBool) || end_token >= (u64)vocab)) ||
      tracked({&logits, &scores, &best}) ||
      (given && !(matrix_ok(best, picked, device, at::kFloat) && matrix_ok(parents, picked, device, at::kInt) &&
                  matrix_ok(tokens, picked, device, at::kLong))))
    return none();
  if (!given) {
    const at::TensorOptions on = at::TensorOptions().device(device);
    best = at::empty(picked, on.dtype(at::kFloat));
    parents = at::empty(picked, on.dtype(at::kInt));
    tokens = at::empty(picked, on.dtype(at::kLong));
  }
  if (requests == 0) return tuple_of({best, parents, tokens});
  const u64 need = reinterpret_cast<u64 (*)(u64, u64, u64)>(size)((u64)requests, (u64)beams, (u64)vocab);
  if (need == kDeclined) return none();
  const at::Tensor space = workspace_of(workspace, need, device);
  typedef long long (*Entry)(u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64);
  const long long got =
      enter<Entry>(entry, address(logits), (u64)dtype, (u64)logits.stride(0), (u64)logits.stride(1), address(scores),
                   address(ended), (u64)requests, (u64)beams, (u64)vocab, candidates, end_token, address(best),
                   address(parents), address(tokens), address(space), need, stream);
  return answer(got, [&] {
    if (given)
      for (const at::Tensor* t : {&best, &parents, &tokens}) wrote(*t);
    return tuple_of({best, parents, tokens});
  });
  END_HANDLE_TH_ERRORS
}

// entry, its workspace's size, layers (a tuple), tables, parents, context_tokens, free_blocks, free_start,
// block_tokens, five results or None each, workspace, stream
PyObject* reorder_beams(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count_ok(n, 16)) return nullptr;
  const u64 entry = number_of(args[0]), size = number_of(args[1]), stream = number_of(args[15]);
  TORCH_CHECK_TYPE(PyTuple_Check(args[2]), "the layers are a tuple");
  const at::Tensor &tables = tensor_of(args[3]), &parents = tensor_of(args[4]), &contexts = tensor_of(args[5]),
                   &free_blocks = tensor_of(args[6]), &free_start = tensor_of(args[7]);
  const u64 block_tokens = number_of(args[8]);
  std::array<at::Tensor, 5> order;
  for (int i = 0; i < 5; ++i) order[i] = maybe_tensor(args[9 + i]);
  const at::Tensor workspace = maybe_tensor(args[14]);
  const at::Device device = tables.device();
  if (tables.scalar_type() != at::kInt || tables.dim() != 2 || parents.scalar_type() != at::kInt ||
      parents.dim() != 2 || parents.device() != device || !parents.is_contiguous() || block_tokens == 0)
    return none();
  const int64_t requests = parents.size(0), beams = parents.size(1), rows = tables.size(0), width = tables.size(1);
  if (rows != requests * beams || (width != 1 && tables.stride(1) != 1) ||
      !vector_ok(contexts, device, rows, at::kInt) || !vector_ok(free_blocks, device, 0, at::kInt) ||
      !vector_ok(free_start, device, 1, at::kInt))
    return none();
  const Py_ssize_t count = PyTuple_GET_SIZE(args[2]);
  auto layer_of = [&](Py_ssize_t i) -> const at::Tensor& { return tensor_of(PyTuple_GET_ITEM(args[2], i)); };
  std::vector<u64> layers((size_t)count + 1);  // (one more: there is an address without layers too)
  u64 blocks = 1, row_bytes = 2;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor &layer = layer_of(i), &first = layer_of(0);
    if (row_dtype(layer) < 0 || !layer_ok(layer, first.scalar_type(), device) || layer.sizes() != first.sizes() ||
        (u64)layer.size(2) != block_tokens || tracked(layer))
      return none();
    layers[(size_t)i] = address(layer);
    blocks = (u64)layer.size(1);
    row_bytes = 2 * (u64)(layer.size(3) * layer.size(4));
  }
  const bool given = std::any_of(order.begin(), order.end(), [](const at::Tensor& t) { return t.defined(); });
  const at::TensorOptions ints = at::TensorOptions().dtype(at::kInt).device(device);
  if (!given) {
    order[0] = at::empty({rows, width}, ints);
    order[1] = at::empty({rows}, ints);
    for (int i = 2; i < 5; ++i) order[i] = at::empty({1}, ints);
  } else if (order[0].scalar_type() != at::kInt || order[0].sizes() != tables.sizes() ||
             order[0].device() != device || (width != 1 && order[0].stride(1) != 1) ||
             !vector_ok(order[1], device, rows, at::kInt) || !vector_ok(order[2], device, 1, at::kInt) ||
             !vector_ok(order[3], device, 1, at::kInt) || !vector_ok(order[4], device, 1, at::kInt)) {
    return none();
  }
  auto results = [&] { return tuple_of({order[0], order[1], order[2], order[3], order[4]}); };
  if (rows == 0) {  // nothing is released
    order[2].narrow(0, 0, 1).copy_(free_start.narrow(0, 0, 1).clamp(0, free_blocks.numel()));
    order[3].narrow(0, 0, 1).zero_();
    order[4].narrow(0, 0, 1).zero_();
    return results();
  }
  const u64 need = reinterpret_cast<u64 (*)(u64, u64, u64)>(size)((u64)requests, (u64)beams, (u64)width);
  if (need == kDeclined) return none();
  const at::Tensor space = workspace_of(workspace, need, device);
  const u64 stride = (u64)(rows > 1 ? tables.stride(0) : width), to = (u64)(rows > 1 ? order[0].stride(0) : width);
  typedef long long (*Entry)(const u64*, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64, u64,
                             u64, u64, u64, u64, u64, u64, u64, u64);
  const long long got = enter<Entry>(
      entry, (const u64*)layers.data(), (u64)count, blocks, block_tokens, row_bytes, address(tables), stride,
      (u64)width, address(order[0]), to, address(parents), address(contexts), (u64)requests, (u64)beams,
      address(free_blocks), (u64)free_blocks.numel(), address(free_start), address(order[1]), address(order[2]),
      address(order[3]), address(order[4]), address(space), need, stream);
  return answer(got, [&] {
    wrote(free_blocks);
    for (Py_ssize_t i = 0; i < count; ++i) wrote(layer_of(i));
    if (given)
      for (const at::Tensor& t : order) wrote(t);
    return results();
  });
  END_HANDLE_TH_ERRORS
}

typedef PyObject* (*Call)(PyObject*, PyObject* const*, Py_ssize_t);

PyMethodDef method(const char* name, Call call) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call)), METH_FASTCALL, nullptr};
}

PyMethodDef kMethods[] = {method("rotate_write", rotate_write), method("cross_paged", cross_paged),
                          method("cross_rows", cross_rows),     method("beam_select", beam_select),
                          method("reorder_beams", reorder_beams), {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_step_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr,
                       nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step_binding() { return PyModule_Create(&kModule); }
