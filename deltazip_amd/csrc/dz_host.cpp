// The host's half of the operators on a paged cache, as a Python extension: the calls that every layer of a decode step
// makes, of tensors that need no more than looking at.  A call takes the host 15 to 21 us where Python checks the arguments, allocates
// the output and packs the C structure, and 4 to 5 here, of which the launch is 2.6, beside 3 to 10 us of the kernels of a small step.
//
// Every function returns None for what is not the ordinary case, and has then done nothing: the caller's Python form
// takes the call, checks each argument by itself and says what is wrong with it.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <map>
#include <utility>
#include <vector>

#include "../../include/dz_amd.h"

namespace {

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
const void* pointer(PyObject* o) { return PyLong_AsVoidPtr(o); }
inline int64_t step(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }   // (of a size of one it means nothing)

// [n, heads, dim] on device `dev`, values of a head side by side
bool heads_on(const at::Tensor& t, at::ScalarType type, int dev) {
  return t.dim() == 3 && t.scalar_type() == type && t.is_cuda() && t.get_device() == dev && t.stride(2) == 1;
}
bool pages_on(const at::Tensor& t, const at::Tensor& q, int dev) {
  if (t.dim() != 4 || t.scalar_type() != q.scalar_type() || !t.is_cuda() || t.get_device() != dev || t.stride(3) != 1 || t.size(3) != q.size(2))
    return false;
  const int64_t ps = t.size(2);
  return ps >= 8 && ps <= 1024 && (ps & (ps - 1)) == 0 && t.size(0) >= 1 && t.size(0) < (1ll << 31) && t.size(1) >= 1;
}
bool index_on(const at::Tensor& t, int64_t n, at::ScalarType type, int dev) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == type && t.is_cuda() && t.get_device() == dev && (n < 2 || t.stride(0) == 1);
}
// int32 [rows, pages], pages of a row side by side
bool tables_on(const at::Tensor& t, int dev) {
  return t.dim() == 2 && t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == dev && t.size(0) >= 1 && t.size(0) <= (1 << 20) && t.size(1) >= 1 &&
         t.size(1) <= (1 << 27) && (t.size(1) == 1 || t.stride(1) == 1);
}
bool floats(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// Whether [n, heads, dim] tensors of one type share nothing: by their ends, or, with rows of one stride (slices of a
// projection), by those of a row.
int64_t reach(const at::Tensor& t, int from) {
  int64_t n = 1;
  for (int d = from; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
  return n;
}
bool ends_apart(const at::Tensor& a, const at::Tensor& b) {
  const int64_t at = ((const char*)b.data_ptr() - (const char*)a.data_ptr()) / (int64_t)a.element_size();
  return at >= reach(a, 0) || -at >= reach(b, 0);
}
bool rows_apart(const at::Tensor& a, const at::Tensor& b) {
  if (ends_apart(a, b)) return true;
  const int64_t row = a.stride(0);
  if (a.size(0) < 2 || b.stride(0) != row || row < 1) return false;
  int64_t at = ((const char*)b.data_ptr() - (const char*)a.data_ptr()) / (int64_t)a.element_size() % row;
  if (at < 0) at += row;
  return at >= reach(a, 1) && at + reach(b, 1) <= row;
}

// Where a call goes: the current device and stream, and the device's status word once Python has taken note of it.
uint32_t* status_at[64];
struct Place {
  int dev;
  void* stream;
  uint32_t* status;
  Place() : dev(c10::hip::current_device()), stream(c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream()),
            status(dev >= 0 && dev < 64 ? status_at[dev] : nullptr) {}
};

// Counters, all zero between calls, and room for the sums of parts, of a stream: calls on it follow each other.  A call holds
// what it is given until it has launched: meanwhile a call of another thread may put larger room in its place, and room that
// nothing holds is given to that thread's next tensor, whose kernels may be ahead of the first call's.  (The map is never freed: it may
// outlive the runtime's own end.)
struct Space {
  at::Tensor counters, work;
};
Space space_of(const Place& p, size_t need, const at::Tensor& like) {
  static auto* spaces = new std::map<std::pair<int, void*>, Space>;
  Space& s = (*spaces)[{p.dev, p.stream}];
  if (!s.counters.defined()) s.counters = at::zeros({DZ_ATTENTION_COUNTERS}, like.options().dtype(at::kInt));
  if (!s.work.defined() || (size_t)s.work.numel() < need)
    s.work = at::empty({(int64_t)(need > (1 << 20) ? need : 1 << 20)}, like.options().dtype(at::kByte));
  return s;
}

// arm(device, address of its status word)
PyObject* arm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const long dev = n == 2 ? PyLong_AsLong(a[0]) : -1;
  void* at = n == 2 ? PyLong_AsVoidPtr(a[1]) : nullptr;
  if (PyErr_Occurred()) return nullptr;
  if (dev >= 0 && dev < 64) status_at[dev] = (uint32_t*)at;
  Py_RETURN_NONE;
}

// attend(q, k_pages, v_pages, tables, lengths, scale or None, window, shared)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *tables = tensor(a[3]), *lengths = tensor(a[4]);
  if (!q || !k || !v || !tables || !lengths || !PyLong_CheckExact(a[6]) || !(a[5] == Py_None || PyFloat_CheckExact(a[5]))) Py_RETURN_NONE;
  if (!q->is_cuda()) Py_RETURN_NONE;
  const Place here;
  const int dev = here.dev;
  if (!here.status) Py_RETURN_NONE;
  int overflow = 0;
  const long window = PyLong_AsLongAndOverflow(a[6], &overflow);
  if (overflow || window < 0 || window > 0x7fffffff) Py_RETURN_NONE;
  if (!floats(q->scalar_type()) || !heads_on(*q, q->scalar_type(), dev) || !pages_on(*k, *q, dev) || !pages_on(*v, *q, dev)) Py_RETURN_NONE;
  const int64_t rows = q->size(0), heads = q->size(1), dim = q->size(2), kv_heads = k->size(1), ps = k->size(2);
  if (rows < 1 || rows > (1 << 20) || heads < 1 || heads > 4096 || heads % kv_heads || dim % 8 || dim > 256 || v->sizes() != k->sizes()) Py_RETURN_NONE;
  if (!tables_on(*tables, dev) || tables->size(0) != rows || tables->size(1) * ps > (1ll << 30)) Py_RETURN_NONE;
  if (!index_on(*lengths, rows, at::kInt, dev)) Py_RETURN_NONE;
  const int width = (int)tables->size(1);
  const size_t need = dz_paged_attention_bytes((int)rows, (int)heads, (int)kv_heads, (int)dim, (int)ps, width);
  Space space;
  if (need) {
    if (dz_capture_id(here.stream)) Py_RETURN_NONE;    // (a graph has its own)
    space = space_of(here, need, *q);
  }
  at::Tensor out = at::empty({rows, heads, dim}, q->options());
  dz_attention_args c{};
  c.bytes = sizeof(c);
  c.q = q->data_ptr(), c.k_pages = k->data_ptr(), c.v_pages = v->data_ptr();
  c.tables = (const int32_t*)tables->data_ptr(), c.lengths = (const int32_t*)lengths->data_ptr();
  c.out = out.data_ptr();
  if (need) c.work = space.work.data_ptr(), c.counters = (uint32_t*)space.counters.data_ptr();
  c.status = here.status;
  c.work_bytes = (int64_t)need, c.num_pages = k->size(0);
  c.q_row = step(*q, 0), c.q_head = step(*q, 1);
  c.k_page = step(*k, 0), c.k_head = step(*k, 1), c.k_token = k->stride(2);
  c.v_page = step(*v, 0), c.v_head = step(*v, 1), c.v_token = v->stride(2);
  c.out_row = heads * dim, c.out_head = dim, c.table_row = step(*tables, 0);
  c.rows = (int)rows, c.heads = (int)heads, c.kv_heads = (int)kv_heads, c.dim = (int)dim, c.page_size = (int)ps;
  c.pages_per_row = width, c.window = (int)window, c.shared = PyObject_IsTrue(a[7]) == 1, c.dtype = q->scalar_type() == at::kBFloat16 ? DZ_BF16 : DZ_F16;
  c.scale = a[5] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)PyFloat_AS_DOUBLE(a[5]);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = dz_paged_attention(&c, here.stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// prefix(q, k_pages, v_pages, tables, lengths, starts, groups, prefixes (None: there are none), scale or None, bytes of tables up to which rows of one
// token go one by one)
PyObject* prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !PyLong_CheckExact(a[9])) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *tables = tensor(a[3]), *lengths = tensor(a[4]);
  if (!q || !k || !v || !tables || !lengths || !(a[8] == Py_None || PyFloat_CheckExact(a[8])) || !q->is_cuda()) Py_RETURN_NONE;
  const at::Tensor *starts = tensor(a[5]), *groups = tensor(a[6]), *prefixes = tensor(a[7]);
  if ((!starts && a[5] != Py_None) || (!groups && a[6] != Py_None) || (!prefixes && a[7] != Py_None) || !groups != !prefixes) Py_RETURN_NONE;
  const Place here;
  const int dev = here.dev;
  if (!here.status) Py_RETURN_NONE;
  if (!floats(q->scalar_type()) || !heads_on(*q, q->scalar_type(), dev) || !pages_on(*k, *q, dev) || !pages_on(*v, *q, dev) || v->sizes() != k->sizes()) Py_RETURN_NONE;
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), kv_heads = k->size(1), ps = k->size(2);
  if (!tables_on(*tables, dev)) Py_RETURN_NONE;
  const int64_t rows = tables->size(0), width = tables->size(1), ngroups = prefixes ? prefixes->numel() : 0;
  if (tokens < 1 || heads < 1 || heads > 4096 || heads % kv_heads || tokens * heads >= (1ll << 31) || dim % 8 || dim > 256 || width * ps > (1ll << 30) ||
      (!starts && tokens != rows) || ngroups > DZ_PREFIX_GROUPS)
    Py_RETURN_NONE;
  if (!index_on(*lengths, rows, at::kInt, dev) || (starts && !index_on(*starts, rows + 1, at::kInt, dev)) ||
      (prefixes && (!index_on(*prefixes, ngroups, at::kInt, dev) || !index_on(*groups, ngroups + 1, at::kInt, dev))))
    Py_RETURN_NONE;
  if (!starts && (!ngroups || rows * width * ps * kv_heads * dim * 4 <= PyLong_AsLongLong(a[9]))) {
    PyObject* const zero = PyLong_FromLong(0);
    if (!zero) return nullptr;
    PyObject* const as[] = {a[0], a[1], a[2], a[3], a[4], a[8], zero, ngroups ? Py_True : Py_False};
    PyObject* const made = attend(nullptr, as, 8);
    Py_DECREF(zero);
    return made;
  }
  const size_t need = dz_prefix_attention_bytes((int)tokens, (int)rows, (int)ngroups, (int)heads, (int)kv_heads, (int)dim);
  if (!need || dz_capture_id(here.stream)) Py_RETURN_NONE;       // (a graph has its own room)
  const Space space = space_of(here, need, *q);
  at::Tensor out = at::empty({tokens, heads, dim}, q->options());
  dz_prefix_args c{};
  c.bytes = sizeof(c);
  c.q = q->data_ptr(), c.k_pages = k->data_ptr(), c.v_pages = v->data_ptr();
  c.tables = (const int32_t*)tables->data_ptr(), c.lengths = (const int32_t*)lengths->data_ptr();
  c.starts = starts ? (const int32_t*)starts->data_ptr() : nullptr;
  if (ngroups) c.groups = (const int32_t*)groups->data_ptr(), c.prefixes = (const int32_t*)prefixes->data_ptr();
  c.out = out.data_ptr(), c.work = space.work.data_ptr(), c.status = here.status;
  c.work_bytes = (int64_t)need, c.num_pages = k->size(0);
  c.q_row = step(*q, 0), c.q_head = step(*q, 1);
  c.k_page = step(*k, 0), c.k_head = step(*k, 1), c.k_token = k->stride(2);
  c.v_page = step(*v, 0), c.v_head = step(*v, 1), c.v_token = v->stride(2);
  c.out_row = heads * dim, c.out_head = dim, c.table_row = step(*tables, 0);
  c.tokens = (int)tokens, c.rows = (int)rows, c.groups_n = (int)ngroups, c.heads = (int)heads, c.kv_heads = (int)kv_heads, c.dim = (int)dim;
  c.page_size = (int)ps, c.pages_per_row = (int)width, c.dtype = q->scalar_type() == at::kBFloat16 ? DZ_BF16 : DZ_F16;
  c.scale = a[8] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)PyFloat_AS_DOUBLE(a[8]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = dz_prefix_attention(&c, here.stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A piece of a tensor's memory as a tensor, from and n in its elements.
at::Tensor piece_of(const at::Tensor& t, int64_t from, int64_t n, at::ScalarType type) {
  at::Tensor y = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(t.storage()), t.key_set(), c10::scalarTypeToTypeMeta(type));
  y.unsafeGetTensorImpl()->set_storage_offset(from);
  y.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return y;
}

// extend(tables, lengths, counts, free_pages, taken, page_size, tokens or None): (lengths, taken, starts, positions, slots)
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *tables = tensor(a[0]), *lengths = tensor(a[1]), *counts = tensor(a[2]), *free = tensor(a[3]), *taken = tensor(a[4]);
  if (!tables || !lengths || !counts || !free || !taken || !PyLong_CheckExact(a[5]) || !(a[6] == Py_None || PyLong_CheckExact(a[6])) || !tables->is_cuda()) Py_RETURN_NONE;
  const Place here;
  const int dev = here.dev;
  if (!here.status || !tables_on(*tables, dev)) Py_RETURN_NONE;
  int overflow = 0;
  const long ps = PyLong_AsLongAndOverflow(a[5], &overflow);
  if (overflow || ps < 8 || ps > 1024 || (ps & (ps - 1))) Py_RETURN_NONE;
  const int64_t rows = tables->size(0), width = tables->size(1), pages = free->numel();
  const long tokens = a[6] == Py_None ? rows : PyLong_AsLongAndOverflow(a[6], &overflow);
  if (overflow || tokens < 0 || tokens > (1 << 24) || width * ps > (1ll << 30) || (rows > 1 && tables->stride(0) < width)) Py_RETURN_NONE;
  if (!index_on(*lengths, rows, at::kInt, dev) || !index_on(*counts, rows, at::kInt, dev) || pages > 0x7fffffff || !index_on(*free, pages, at::kInt, dev) ||
      !index_on(*taken, 1, at::kInt, dev))
    Py_RETURN_NONE;
  if (!ends_apart(*tables, *lengths) || !ends_apart(*tables, *counts) || !ends_apart(*tables, *free) || !ends_apart(*tables, *taken)) Py_RETURN_NONE;
  const at::Tensor room = at::empty({4 * tokens + 2 * rows + 2}, tables->options());      // positions, slots; lengths, pages taken, starts
  dz_extend_args c{};
  c.bytes = sizeof(c);
  c.tables = (int32_t*)tables->data_ptr(), c.lengths = (const int32_t*)lengths->data_ptr(), c.counts = (const int32_t*)counts->data_ptr();
  c.free_pages = (const int32_t*)free->data_ptr(), c.taken = (const int32_t*)taken->data_ptr();
  c.positions = (int64_t*)room.data_ptr(), c.slots = c.positions + tokens, c.status = here.status;
  c.lengths_out = (int32_t*)(c.slots + tokens), c.taken_out = c.lengths_out + rows, c.starts = c.taken_out + 1;
  c.table_row = step(*tables, 0);
  c.rows = (int)rows, c.pages_per_row = (int)width, c.page_size = (int)ps, c.free_n = (int)pages, c.tokens = (int)tokens, c.packed = a[6] != Py_None;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = dz_extend_tables(&c, here.stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  PyObject* made = PyTuple_New(5);
  if (!made) return nullptr;
  const int64_t at = 4 * tokens;
  PyTuple_SET_ITEM(made, 0, THPVariable_Wrap(piece_of(room, at, rows, at::kInt)));
  PyTuple_SET_ITEM(made, 1, THPVariable_Wrap(piece_of(room, at + rows, 1, at::kInt)));
  PyTuple_SET_ITEM(made, 2, THPVariable_Wrap(piece_of(room, at + rows + 1, rows + 1, at::kInt)));
  PyTuple_SET_ITEM(made, 3, THPVariable_Wrap(piece_of(room, 0, tokens, at::kLong)));
  PyTuple_SET_ITEM(made, 4, THPVariable_Wrap(piece_of(room, tokens, tokens, at::kLong)));
  return made;
  END_HANDLE_TH_ERRORS
}

// rotate(q, k, v, positions, slots, (turns, rot, neighbours, factor, head_dim) or None, k_pages, v_pages, q in place):
// q turned (append_kv); without pages, v and slots None: (q turned, k turned or None) (rotary)
PyObject* rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) Py_RETURN_NONE;
  const bool paged = a[4] != Py_None;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *positions = tensor(a[3]);
  if (!q || !q->is_cuda()) Py_RETURN_NONE;
  const Place here;
  const int dev = here.dev;
  if (!positions || (paged && !here.status) || (!k && (paged || a[1] != Py_None))) Py_RETURN_NONE;
  const at::ScalarType type = q->scalar_type();
  if (!floats(type) || !heads_on(*q, type, dev) || q->size(0) < 1 || q->size(0) > 0x7fffffff || q->size(1) < 1 || q->size(1) > 4096) Py_RETURN_NONE;
  const int64_t tokens = q->size(0), dim = q->size(2);
  if (k && (!heads_on(*k, type, dev) || k->size(0) != tokens || k->size(2) != dim || k->size(1) < 1 || k->size(1) > 4096)) Py_RETURN_NONE;
  if (!index_on(*positions, tokens, at::kLong, dev)) Py_RETURN_NONE;
  dz_rotary_args c{};
  c.bytes = sizeof(c);
  c.factor = 1.0f;
  if (a[5] != Py_None) {
    if (!PyTuple_CheckExact(a[5]) || PyTuple_GET_SIZE(a[5]) != 5) Py_RETURN_NONE;
    c.turns = (const double*)pointer(PyTuple_GET_ITEM(a[5], 0));
    c.rot = (int)PyLong_AsLong(PyTuple_GET_ITEM(a[5], 1)), c.neighbours = (int)PyLong_AsLong(PyTuple_GET_ITEM(a[5], 2));
    c.factor = (float)PyFloat_AsDouble(PyTuple_GET_ITEM(a[5], 3));
    if (PyLong_AsLong(PyTuple_GET_ITEM(a[5], 4)) != dim) Py_RETURN_NONE;
  } else if (!paged) {
    Py_RETURN_NONE;
  }
  const bool in_place = a[8] == Py_True;
  const at::Tensor *v = nullptr, *kp = nullptr, *vp = nullptr, *slots = nullptr;
  at::Tensor q_out, k_out;
  if (paged) {
    v = tensor(a[2]), slots = tensor(a[4]), kp = tensor(a[6]), vp = tensor(a[7]);
    if (!v || !slots || !kp || !vp || !heads_on(*v, type, dev) || v->sizes() != k->sizes() || !index_on(*slots, tokens, at::kLong, dev) ||
        !pages_on(*kp, *q, dev) || !pages_on(*vp, *q, dev) || kp->sizes() != vp->sizes() || kp->size(1) != k->size(1) ||
        !kp->is_contiguous() || !vp->is_contiguous())
      Py_RETURN_NONE;
    if (!ends_apart(*kp, *vp) || !ends_apart(*kp, *k) || !ends_apart(*kp, *v) || !ends_apart(*vp, *k) || !ends_apart(*vp, *v)) Py_RETURN_NONE;
    if (c.rot && (!ends_apart(*kp, *q) || !ends_apart(*vp, *q))) Py_RETURN_NONE;
    c.v = v->data_ptr(), c.v_row = step(*v, 0), c.v_head = step(*v, 1);
    c.slots = (const int64_t*)slots->data_ptr(), c.status = here.status;
    c.num_pages = kp->size(0), c.page_size = (int)kp->size(2);
    c.k_out = kp->data_ptr(), c.k_out_page = step(*kp, 0), c.k_out_head = step(*kp, 1), c.k_out_token = kp->stride(2);
    c.v_out = vp->data_ptr(), c.v_out_page = step(*vp, 0), c.v_out_head = step(*vp, 1), c.v_out_token = vp->stride(2);
  } else if (in_place) {
    Py_RETURN_NONE;
  }
  if (in_place) {
    c.q_out = q->data_ptr(), c.q_out_row = step(*q, 0), c.q_out_head = step(*q, 1);
    if ((tokens > 1 && q->stride(0) < q->size(1) * q->stride(1)) || (q->size(1) > 1 && q->stride(1) < dim)) Py_RETURN_NONE;
    if (c.rot && (!rows_apart(*q, *k) || !rows_apart(*q, *v))) Py_RETURN_NONE;
  } else {
    q_out = at::empty(q->sizes(), q->options());
    c.q_out = q_out.data_ptr(), c.q_out_row = q->size(1) * dim, c.q_out_head = dim;
  }
  c.q = q->data_ptr(), c.q_row = step(*q, 0), c.q_head = step(*q, 1);
  if (k) {
    c.k = k->data_ptr(), c.k_row = step(*k, 0), c.k_head = step(*k, 1), c.kv_heads = (int)k->size(1);
    if (!paged) {
      k_out = at::empty(k->sizes(), k->options());
      c.k_out = k_out.data_ptr(), c.k_out_token = k->size(1) * dim, c.k_out_head = dim;
    }
  }
  c.positions = (const int64_t*)positions->data_ptr();
  c.tokens = (int)tokens, c.heads = in_place && !c.rot ? 0 : (int)q->size(1), c.dim = (int)dim, c.dtype = type == at::kBFloat16 ? DZ_BF16 : DZ_F16;
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = dz_rotary(&c, here.stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  if (in_place) {
    Py_INCREF(a[0]);
    return a[0];
  }
  if (paged) return THPVariable_Wrap(std::move(q_out));
  PyObject* both = PyTuple_New(2);
  if (!both) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(q_out)));
  if (k) {
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(k_out)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(both, 1, Py_None);
  }
  return both;
  END_HANDLE_TH_ERRORS
}

// copy(pools [n, pages, ...], pairs [m, 2] on the host): True where the copies were launched
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) Py_RETURN_NONE;
  const at::Tensor *pools = tensor(a[0]), *pairs = tensor(a[1]);
  if (!pools || !pairs || !pools->is_cuda()) Py_RETURN_NONE;
  const Place here;
  const int dev = here.dev;
  if (pools->get_device() != dev || pools->dim() < 2 || !pools->is_contiguous() || pools->numel() == 0 ||
      pools->size(1) >= (1ll << 31) || pools->size(0) > (1 << 20))
    Py_RETURN_NONE;
  if (!pairs->is_cpu() || pairs->scalar_type() != at::kLong || pairs->dim() != 2 || pairs->size(1) != 2 || !pairs->is_contiguous() ||
      pairs->size(0) < 1 || pairs->size(0) > (1 << 24))
    Py_RETURN_NONE;
  const int64_t pages = pools->size(1), m = pairs->size(0), npools = pools->size(0);
  const int64_t bytes = pools->numel() / npools / pages * (int64_t)pools->element_size();
  // pages that the call writes: a mark for each, taken back below
  static thread_local std::vector<unsigned char> written;
  if ((int64_t)written.size() < pages) written.resize(pages, 0);
  std::vector<int32_t> list(2 * m);
  const int64_t* from = (const int64_t*)pairs->data_ptr();
  bool fits = true;
  int64_t marked = 0;
  for (; marked < m && fits; ++marked) {
    const int64_t x = from[2 * marked], y = from[2 * marked + 1];
    if (x < 0 || x >= pages || y < 0 || y >= pages || written[y]) {
      fits = false;
      break;
    }
    written[y] = 1;
    list[2 * marked] = (int32_t)x, list[2 * marked + 1] = (int32_t)y;
  }
  for (int64_t i = 0; i < m && fits; ++i) fits = !written[list[2 * i]];
  for (int64_t i = 0; i < marked; ++i) written[list[2 * i + 1]] = 0;
  if (!fits) Py_RETURN_NONE;
  std::vector<void*> at(npools);
  for (int64_t i = 0; i < npools; ++i) at[i] = (char*)pools->data_ptr() + i * pages * bytes;
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = dz_copy_pages(at.data(), (int)npools, bytes, bytes, (int)pages, list.data(), (int)m, here.stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"arm", (PyCFunction)(void (*)(void))arm, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
                         {"prefix", (PyCFunction)(void (*)(void))prefix, METH_FASTCALL, nullptr},
                         {"extend", (PyCFunction)(void (*)(void))extend, METH_FASTCALL, nullptr},
                         {"rotate", (PyCFunction)(void (*)(void))rotate, METH_FASTCALL, nullptr},
                         {"copy", (PyCFunction)(void (*)(void))copy, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
