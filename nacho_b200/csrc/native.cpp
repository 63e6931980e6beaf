// Python operators over the C ABI (module nacho_b200._native). A call on small operands computes for a few
// microseconds, so what surrounds it counts: this module reads the tensors of the operand objects, takes the
// result arrays from torch's caching allocator, runs one C-ABI entry point without the interpreter lock and
// hands back an object of the caller's class -- about 4 us where the same steps in Python with ctypes took
// 35. It computes nothing itself. Classes, slots and error texts are those of nacho/nacho_ext.py, which
// hands them over with bind().
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "nacho_b200.h"

namespace {

// ---- what nacho_ext.py binds ---------------------------------------------------------------

enum Kind { CSR = 0, COO = 1, DCSR = 2, COO3 = 3, CSF3 = 4, SCALAR = 5, KINDS = 6, ORDER = 6, FP8 = 7, INT8 = 8, ALL_KINDS = 9 };
PyTypeObject *g_class[ALL_KINDS] = {};  // the first KINDS from nacho_ext.py, the others from experts.py and layers.py
PyObject *g_check = nullptr;  // check(status, where): raises on a non-zero status
enum Name { N_offsets, N_indices, N_values, N_dims, N_i, N_j, N_k, N_jp, N_kp, N_rows, N_slots, N_token_offsets, N_scales, N_tiled, NAMES };
PyObject *g_name[NAMES] = {};  // interned slot names
const char *const NAME_TEXT[NAMES] = {"_offsets", "_indices", "_values", "_dims", "_i", "_j", "_k", "_jp", "_kp", "_rows", "_slots", "_token_offsets", "_scales", "_tiled"};

struct PyFailure {};  // a Python exception is set

struct Ref {  // owned reference
    PyObject *p;
    explicit Ref(PyObject *o) : p(o) { if (!o) throw PyFailure(); }
    ~Ref() { Py_XDECREF(p); }
    Ref(const Ref &) = delete;
    PyObject *release() { PyObject *r = p; p = nullptr; return r; }
};

const at::Tensor &tensor_of(PyObject *obj, Name slot) {
    Ref t(PyObject_GetAttr(obj, g_name[slot]));
    if (!THPVariable_Check(t.p)) {
        PyErr_SetString(PyExc_TypeError, "operand slot does not hold a tensor");
        throw PyFailure();
    }
    return THPVariable_Unpack(t.p);  // the operand object keeps it alive while the interpreter lock is held
}

template <int N>
void dims_of(PyObject *obj, int32_t *out) {
    Ref d(PyObject_GetAttr(obj, g_name[N_dims]));
    if (!PyTuple_Check(d.p) || PyTuple_GET_SIZE(d.p) != N) {
        PyErr_SetString(PyExc_TypeError, "operand has no extents");
        throw PyFailure();
    }
    for (int k = 0; k < N; ++k) out[k] = (int32_t)PyLong_AsLong(PyTuple_GET_ITEM(d.p, k));
}

void need_kind(PyObject *obj, Kind kind, const char *where, const char *what) {
    if (Py_TYPE(obj) == g_class[kind]) return;
    const int is = PyObject_IsInstance(obj, reinterpret_cast<PyObject *>(g_class[kind]));
    if (is < 0) throw PyFailure();
    if (!is) {
        PyErr_Format(PyExc_TypeError, "%s: operands must be %s", where, what);
        throw PyFailure();
    }
}

// ---- operand views -------------------------------------------------------------------------

int32_t *ints(const at::Tensor &t) { return static_cast<int32_t *>(t.data_ptr()); }
float *floats(const at::Tensor &t) { return static_cast<float *>(t.data_ptr()); }

struct View {  // device and arrays of one operand, for what all kinds share
    c10::Device device = c10::Device(c10::kCPU);
    at::Tensor arrays[6];  // references of their own: another thread may give the operand new arrays meanwhile
    int n = 0;

    const at::Tensor &array(PyObject *o, Name slot) {
        arrays[n] = tensor_of(o, slot);
        return arrays[n++];
    }
    int32_t *index(PyObject *o, Name slot) { return ints(array(o, slot)); }
};

nb200_csr view_csr(PyObject *o, View &v) {
    const at::Tensor &val = v.array(o, N_values);
    int32_t d[2];
    dims_of<2>(o, d);
    v.device = val.device();
    return nb200_csr{d[0], d[1], (int32_t)val.numel(), v.index(o, N_offsets), v.index(o, N_indices), floats(val)};
}

nb200_coo view_coo(PyObject *o, View &v) {
    const at::Tensor &val = v.array(o, N_values);
    int32_t d[2];
    dims_of<2>(o, d);
    v.device = val.device();
    return nb200_coo{d[0], d[1], (int32_t)val.numel(), v.index(o, N_i), v.index(o, N_j), floats(val)};
}

nb200_dcsr view_dcsr(PyObject *o, View &v) {
    const at::Tensor &val = v.array(o, N_values), &i = v.array(o, N_i);
    int32_t d[2];
    dims_of<2>(o, d);
    v.device = val.device();
    return nb200_dcsr{d[0], d[1], (int32_t)i.numel(), (int32_t)val.numel(), ints(i), v.index(o, N_jp), v.index(o, N_j), floats(val)};
}

nb200_coo3 view_coo3(PyObject *o, View &v) {
    const at::Tensor &val = v.array(o, N_values);
    nb200_coo3 s{};
    dims_of<3>(o, s.dims);
    v.device = val.device();
    s.nnz = (int32_t)val.numel();
    s.i = v.index(o, N_i), s.j = v.index(o, N_j), s.k = v.index(o, N_k), s.val = floats(val);
    return s;
}

nb200_csf3 view_csf3(PyObject *o, View &v) {
    const at::Tensor &val = v.array(o, N_values), &i = v.array(o, N_i), &j = v.array(o, N_j), &k = v.array(o, N_k);
    nb200_csf3 s{};
    dims_of<3>(o, s.dims);
    v.device = val.device();
    s.n_i = (int32_t)i.numel(), s.n_j = (int32_t)j.numel(), s.n_k = (int32_t)k.numel();
    s.i_idx = ints(i), s.j_ptr = v.index(o, N_jp), s.j_idx = ints(j), s.k_ptr = v.index(o, N_kp), s.k_idx = ints(k), s.val = floats(val);
    return s;
}

void same_device(const View &a, const View &b) {
    if (a.device != b.device) {
        PyErr_SetString(PyExc_ValueError, "operands live on different devices");
        throw PyFailure();
    }
}

// ---- results -------------------------------------------------------------------------------

at::Tensor array(int64_t n, at::ScalarType type, c10::Device dev) {
    return at::Tensor(at::detail::empty_cuda({std::max<int64_t>(n, 1)}, type, dev, std::nullopt));
}
at::Tensor int_array(int64_t n, c10::Device dev) { return array(n, at::kInt, dev); }
at::Tensor float_array(int64_t n, c10::Device dev) { return array(n, at::kFloat, dev); }

// A result array was taken at its worst-case length; its tensor covers the part in use.
void used(at::Tensor &t, int64_t n) {
    t.unsafeGetTensorImpl()->set_sizes_contiguous(c10::IntArrayRef(&n, 1));
}

struct Result {
    Ref obj;
    explicit Result(Kind kind) : obj(g_class[kind]->tp_alloc(g_class[kind], 0)) {}
    void set(Name slot, at::Tensor &t) {
        Ref v(THPVariable_Wrap(t));
        if (PyObject_SetAttr(obj.p, g_name[slot], v.p) < 0) throw PyFailure();
    }
    template <int N>
    void dims(const int32_t *d) {
        Ref t(PyTuple_New(N));
        for (int k = 0; k < N; ++k) PyTuple_SET_ITEM(t.p, k, PyLong_FromLong(d[k]));
        if (PyObject_SetAttr(obj.p, g_name[N_dims], t.p) < 0) throw PyFailure();
    }
};

void check(int status, const char *where) {
    if (status == NB200_OK) return;
    Ref r(PyObject_CallFunction(g_check, "is", status, where));
    PyErr_Format(PyExc_RuntimeError, "%s: status %d", where, status);  // only if check() did not raise
    throw PyFailure();
}

struct NoLock {  // releases the interpreter lock
    PyThreadState *state = PyEval_SaveThread();
    ~NoLock() { PyEval_RestoreThread(state); }
};

// Calls of several host threads on one stream take turns at issuing their kernels: they share the stream's scratch
// arrays and result words. The lock's key is the pool's, device and stream: the default stream has the same handle
// on every device, and a lock is held while its call waits for a length. (Locks stay, as the pool's entries do.)
std::mutex &stream_lock(int device, void *stream) {
    static std::mutex guard;
    static std::map<std::pair<int, void *>, std::mutex> locks;
    thread_local std::pair<int, void *> last{-1, nullptr};
    thread_local std::mutex *last_lock = nullptr;
    const std::pair<int, void *> key{device, stream};
    if (!last_lock || last != key) {
        std::lock_guard<std::mutex> g(guard);
        last_lock = &locks[key];
        last = key;
    }
    return *last_lock;
}

// Runs a C-ABI call on the operands' device and the current stream of the caller, without the interpreter lock. A call
// returns when the result's length is known, with kernels still running: the allocator is told that the
// operands' arrays are in use on this stream, which matters when they came from another one.
template <size_t N, typename F>
int run(const View *const (&operands)[N], F call) {
    const c10::Device device = operands[0]->device;
    c10::cuda::CUDAGuard guard(device);
    const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream(device.index());
    void *stream = current.stream();
    int status;
    {
        NoLock unlocked;
        std::lock_guard<std::mutex> turn(stream_lock(device.index(), stream));
        status = call(stream);
    }
    for (const View *operand : operands)
        for (int k = 0; k < operand->n; ++k) c10::cuda::CUDACachingAllocator::recordStream(operand->arrays[k].storage().data_ptr(), current);
    return status;
}

template <size_t N, typename F>
void launch(const View *const (&operands)[N], const char *where, F call) {
    check(run(operands, call), where);
}

// ---- operators -----------------------------------------------------------------------------

typedef int (*csr2_fn)(const nb200_csr *, const nb200_csr *, nb200_csr *, int64_t, void *);
typedef int (*coo2_fn)(const nb200_coo *, const nb200_coo *, nb200_coo *, int64_t, void *);
typedef int (*dcsr2_fn)(const nb200_dcsr *, const nb200_dcsr *, nb200_dcsr *, int64_t, int64_t, void *);

// A CSR result of up to `capacity` entries, filled by `call(z, stream)`.
template <size_t N, typename F>
PyObject *csr_result(const View *const (&operands)[N], const char *where, int32_t rows, int32_t cols, int64_t capacity, F call) {
    const c10::Device device = operands[0]->device;
    at::Tensor rp = int_array((int64_t)rows + 1, device), col = int_array(capacity, device), val = float_array(capacity, device);
    nb200_csr z{rows, cols, 0, ints(rp), ints(col), floats(val)};
    launch(operands, where, [&](void *stream) { return call(&z, stream); });
    used(col, z.nnz);
    used(val, z.nnz);
    Result r(CSR);
    r.set(N_offsets, rp), r.set(N_indices, col), r.set(N_values, val);
    const int32_t d[2] = {z.rows, z.cols};
    r.dims<2>(d);
    return r.obj.release();
}

PyObject *csr_binary(csr2_fn fn, bool is_union, const char *where, PyObject *const *args) {
    for (int k = 0; k < 2; ++k) need_kind(args[k], CSR, where, "CSR_gpu");
    View va, vb;
    const nb200_csr a = view_csr(args[0], va), b = view_csr(args[1], vb);
    same_device(va, vb);
    const int64_t capacity = is_union ? (int64_t)a.nnz + b.nnz : std::min(a.nnz, b.nnz);
    return csr_result({&va, &vb}, where, a.rows, a.cols, capacity, [&](nb200_csr *z, void *stream) { return fn(&a, &b, z, capacity, stream); });
}

PyObject *csr_add(PyObject *const *args) { return csr_binary(nb200_csr_add_f32_into, true, "gpu_csr_add_f32", args); }
PyObject *csr_mul(PyObject *const *args) { return csr_binary(nb200_csr_mul_f32_into, false, "gpu_csr_mul_f32", args); }

constexpr int64_t ADD3_POOL_BYTES = 8 << 20;

PyObject *csr_add_3(PyObject *const *args) {
    const char *where = "gpu_csr_add_3_f32";
    for (int k = 0; k < 3; ++k) need_kind(args[k], CSR, where, "CSR_gpu");
    View va, vb, vc;
    const nb200_csr a = view_csr(args[0], va), b = view_csr(args[1], vb), c = view_csr(args[2], vc);
    same_device(va, vb);
    same_device(va, vc);
    const int64_t capacity = (int64_t)a.nnz + b.nnz + c.nnz;
    // The intermediate sum is as large as the operands: it lies in an array of this call. Only a small one stays in the
    // library's pool (the array costs half a microsecond).
    const int64_t scratch_bytes = nb200_csr_add_3_f32_scratch(&a, &b, &c);
    if (scratch_bytes <= ADD3_POOL_BYTES)
        return csr_result({&va, &vb, &vc}, where, a.rows, a.cols, capacity,
                          [&](nb200_csr *z, void *stream) { return nb200_csr_add_3_f32_into(&a, &b, &c, z, capacity, stream); });
    at::Tensor scratch = array(scratch_bytes, at::kByte, va.device);
    return csr_result({&va, &vb, &vc}, where, a.rows, a.cols, capacity,
                      [&](nb200_csr *z, void *stream) { return nb200_csr_add_3_f32_lent(&a, &b, &c, z, capacity, scratch.data_ptr(), scratch_bytes, stream); });
}

PyObject *sssmm(PyObject *const *args) {
    const char *where = "gpu_sssmm_f32";
    for (int k = 0; k < 3; ++k) need_kind(args[k], CSR, where, "CSR_gpu");
    View va, vb, vc;
    const nb200_csr a = view_csr(args[0], va), b = view_csr(args[1], vb), c = view_csr(args[2], vc);
    same_device(va, vb);
    same_device(va, vc);
    return csr_result({&va, &vb, &vc}, where, a.rows, b.cols, c.nnz, [&](nb200_csr *z, void *stream) { return nb200_sssmm_f32_into(&a, &b, &c, z, c.nnz, stream); });
}

PyObject *coo_csr_add(PyObject *const *args) {
    const char *where = "gpu_coo_csr_add_f32";
    need_kind(args[0], CSR, where, "(CSR_gpu, COO_gpu)");
    need_kind(args[1], COO, where, "(CSR_gpu, COO_gpu)");
    View va, vb;
    const nb200_csr a = view_csr(args[0], va);
    const nb200_coo b = view_coo(args[1], vb);
    same_device(va, vb);
    const int64_t capacity = (int64_t)a.nnz + b.nnz;
    return csr_result({&va, &vb}, where, a.rows, a.cols, capacity, [&](nb200_csr *z, void *stream) { return nb200_coo_csr_add_f32_into(&a, &b, z, capacity, stream); });
}

PyObject *spgemm(PyObject *const *args) {
    const char *where = "gpu_spgemm_f32";
    for (int k = 0; k < 2; ++k) need_kind(args[k], CSR, where, "CSR_gpu");
    View va, vb;
    const nb200_csr a = view_csr(args[0], va), b = view_csr(args[1], vb);
    same_device(va, vb);
    at::Tensor rp = int_array((int64_t)a.rows + 1, va.device);
    nb200_csr c{a.rows, b.cols, 0, ints(rp), nullptr, nullptr};
    struct Taken {  // the result's arrays, taken when their length is known, and those it moved out of
        c10::Device device;
        at::Tensor col, val, earlier_col, earlier_val;
        std::exception_ptr failure;
    } taken{va.device};
    auto take = [](void *ctx, int64_t entries, int32_t **col, float **val) noexcept -> int {
        Taken &t = *static_cast<Taken *>(ctx);
        try {
            at::Tensor c = int_array(entries, t.device), v = float_array(entries, t.device);
            t.earlier_col = std::move(t.col), t.earlier_val = std::move(t.val);
            t.col = std::move(c), t.val = std::move(v);
            *col = ints(t.col), *val = floats(t.val);
            return NB200_OK;
        } catch (...) {
            t.failure = std::current_exception();
            return NB200_E_NOMEM;
        }
    };
    const int status = run({&va, &vb}, [&](void *stream) { return nb200_spgemm_f32_with(&a, &b, &c, take, &taken, stream); });
    if (status == NB200_E_NOMEM && taken.failure) std::rethrow_exception(taken.failure);
    check(status, where);
    at::Tensor &col = taken.col, &val = taken.val;
    if (!col.defined()) col = int_array(0, va.device), val = float_array(0, va.device);
    used(col, c.nnz);
    used(val, c.nnz);
    Result r(CSR);
    r.set(N_offsets, rp), r.set(N_indices, col), r.set(N_values, val);
    const int32_t d[2] = {c.rows, c.cols};
    r.dims<2>(d);
    return r.obj.release();
}

PyObject *coo_binary(coo2_fn fn, bool is_union, const char *where, PyObject *const *args) {
    for (int k = 0; k < 2; ++k) need_kind(args[k], COO, where, "COO_gpu");
    View va, vb;
    const nb200_coo a = view_coo(args[0], va), b = view_coo(args[1], vb);
    same_device(va, vb);
    const int64_t capacity = is_union ? (int64_t)a.nnz + b.nnz : std::min(a.nnz, b.nnz);
    at::Tensor i = int_array(capacity, va.device), j = int_array(capacity, va.device), val = float_array(capacity, va.device);
    nb200_coo z{a.rows, a.cols, 0, ints(i), ints(j), floats(val)};
    launch({&va, &vb}, where, [&](void *stream) { return fn(&a, &b, &z, capacity, stream); });
    used(i, z.nnz), used(j, z.nnz), used(val, z.nnz);
    Result r(COO);
    r.set(N_i, i), r.set(N_j, j), r.set(N_values, val);
    const int32_t d[2] = {z.rows, z.cols};
    r.dims<2>(d);
    return r.obj.release();
}

PyObject *coo_add(PyObject *const *args) { return coo_binary(nb200_coo_add_f32_into, true, "gpu_coo_add_f32", args); }
PyObject *coo_mul(PyObject *const *args) { return coo_binary(nb200_coo_mul_f32_into, false, "gpu_coo_mul_f32", args); }

PyObject *dcsr_binary(dcsr2_fn fn, bool is_union, const char *where, PyObject *const *args) {
    for (int k = 0; k < 2; ++k) need_kind(args[k], DCSR, where, "DCSR_gpu");
    View va, vb;
    const nb200_dcsr a = view_dcsr(args[0], va), b = view_dcsr(args[1], vb);
    same_device(va, vb);
    const int64_t cap_i = is_union ? std::min<int64_t>((int64_t)a.n_i + b.n_i, a.rows) : std::min(a.n_i, b.n_i);
    const int64_t capacity = is_union ? (int64_t)a.nnz + b.nnz : std::min(a.nnz, b.nnz);
    at::Tensor i = int_array(cap_i, va.device), jp = int_array(cap_i + 1, va.device), j = int_array(capacity, va.device), val = float_array(capacity, va.device);
    nb200_dcsr z{a.rows, a.cols, 0, 0, ints(i), ints(jp), ints(j), floats(val)};
    launch({&va, &vb}, where, [&](void *stream) { return fn(&a, &b, &z, cap_i, capacity, stream); });
    used(i, z.n_i), used(jp, (int64_t)z.n_i + 1), used(j, z.nnz), used(val, z.nnz);
    Result r(DCSR);
    r.set(N_i, i), r.set(N_jp, jp), r.set(N_j, j), r.set(N_values, val);
    const int32_t d[2] = {z.rows, z.cols};
    r.dims<2>(d);
    return r.obj.release();
}

PyObject *dcsr_add(PyObject *const *args) { return dcsr_binary(nb200_dcsr_add_f32_into, true, "gpu_dcsr_add_f32", args); }
PyObject *dcsr_mul(PyObject *const *args) { return dcsr_binary(nb200_dcsr_mul_f32_into, false, "gpu_dcsr_mul_f32", args); }

PyObject *coo3d_add(PyObject *const *args) {
    const char *where = "gpu_coo3d_add_f32";
    for (int k = 0; k < 2; ++k) need_kind(args[k], COO3, where, "COO3_gpu");
    View va, vb;
    const nb200_coo3 a = view_coo3(args[0], va), b = view_coo3(args[1], vb);
    same_device(va, vb);
    const int64_t capacity = (int64_t)a.nnz + b.nnz;
    at::Tensor i = int_array(capacity, va.device), j = int_array(capacity, va.device), k = int_array(capacity, va.device), val = float_array(capacity, va.device);
    nb200_coo3 z{};
    z.i = ints(i), z.j = ints(j), z.k = ints(k), z.val = floats(val);
    launch({&va, &vb}, where, [&](void *stream) { return nb200_coo3d_add_f32_into(&a, &b, &z, capacity, stream); });
    used(i, z.nnz), used(j, z.nnz), used(k, z.nnz), used(val, z.nnz);
    Result r(COO3);
    r.set(N_i, i), r.set(N_j, j), r.set(N_k, k), r.set(N_values, val);
    r.dims<3>(z.dims);
    return r.obj.release();
}

PyObject *csf_add(PyObject *const *args) {
    const char *where = "gpu_csf_add_f32";
    for (int k = 0; k < 2; ++k) need_kind(args[k], CSF3, where, "CSF3_gpu");
    View va, vb;
    const nb200_csf3 a = view_csf3(args[0], va), b = view_csf3(args[1], vb);
    same_device(va, vb);
    const int64_t cap_i = (int64_t)a.n_i + b.n_i, cap_j = (int64_t)a.n_j + b.n_j, cap_k = (int64_t)a.n_k + b.n_k;
    at::Tensor i = int_array(cap_i, va.device), jp = int_array(cap_i + 1, va.device), j = int_array(cap_j, va.device);
    at::Tensor kp = int_array(cap_j + 1, va.device), k = int_array(cap_k, va.device), val = float_array(cap_k, va.device);
    nb200_csf3 z{};
    z.i_idx = ints(i), z.j_ptr = ints(jp), z.j_idx = ints(j), z.k_ptr = ints(kp), z.k_idx = ints(k), z.val = floats(val);
    launch({&va, &vb}, where, [&](void *stream) { return nb200_csf_add_f32_into(&a, &b, &z, cap_i, cap_j, cap_k, stream); });
    used(i, z.n_i), used(jp, (int64_t)z.n_i + 1), used(j, z.n_j), used(kp, (int64_t)z.n_j + 1), used(k, z.n_k), used(val, z.n_k);
    Result r(CSF3);
    r.set(N_i, i), r.set(N_jp, jp), r.set(N_j, j), r.set(N_kp, kp), r.set(N_k, k), r.set(N_values, val);
    r.dims<3>(z.dims);
    return r.obj.release();
}

template <typename S, typename F>
PyObject *inner(Kind kind, const char *what, const char *where, PyObject *const *args, S (*view)(PyObject *, View &), F fn) {
    for (int k = 0; k < 2; ++k) need_kind(args[k], kind, where, what);
    View va, vb;
    const S a = view(args[0], va), b = view(args[1], vb);
    same_device(va, vb);
    at::Tensor z = float_array(1, va.device);
    launch({&va, &vb}, where, [&](void *stream) { return fn(&a, &b, floats(z), stream); });
    Result r(SCALAR);
    r.set(N_values, z);
    return r.obj.release();
}

PyObject *inner_prod(PyObject *const *args) { return inner(CSF3, "CSF3_gpu", "gpu_inner_prod_f32", args, view_csf3, nb200_inner_prod_f32); }
PyObject *inner_prod_coo(PyObject *const *args) { return inner(COO3, "COO3_gpu", "gpu_inner_prod_coo_f32", args, view_coo3, nb200_inner_prod_coo_f32); }

// ---- around a router -------------------------------------------------------------------------

int type_of(const at::Tensor &t) { return t.scalar_type() == at::kFloat ? NB200_F32 : t.scalar_type() == at::kHalf ? NB200_F16 : t.scalar_type() == at::kBFloat16 ? NB200_BF16 : -1; }
at::ScalarType scalar_of(int type) { return type == NB200_F32 ? at::kFloat : type == NB200_F16 ? at::kHalf : at::kBFloat16; }

void refuse(PyObject *kind, const char *text, const char *where, const char *name) {
    PyErr_Format(kind, text, where, name);
    throw PyFailure();
}

// A 2-D CUDA tensor of floats whose rows are contiguous; any distance between rows. With `groups`, also a 3-D one whose groups follow one
// another at that distance: it is seen as their rows.
nb200_dense view_dense(PyObject *o, View &v, const char *where, const char *name, int64_t *groups = nullptr) {
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s: %s must be a torch tensor", where, name);
    v.arrays[v.n] = THPVariable_Unpack(o);
    const at::Tensor &t = v.arrays[v.n++];
    const int type = type_of(t);
    const bool three = groups && t.dim() == 3;
    if (!t.is_cuda() || type < 0 || !(t.dim() == 2 || three)) refuse(PyExc_TypeError, "%s: %s must be a CUDA tensor of rows of float32, float16 or bfloat16", where, name);
    const int64_t rows = t.size(-2), cols = t.size(-1);
    if (rows > INT32_MAX || cols > INT32_MAX || (three && t.size(0) > INT32_MAX)) refuse(PyExc_ValueError, "%s: %s has an extent beyond int32", where, name);
    if (cols > 1 && rows > 0 && t.stride(-1) != 1) refuse(PyExc_TypeError, "%s: the rows of %s must be contiguous", where, name);
    int64_t all = rows, stride = rows > 1 ? t.stride(-2) : cols;
    if (three) {
        all = t.size(0) * rows;
        if (rows == 1) stride = t.size(0) > 1 ? t.stride(0) : cols;
        else if (t.size(0) > 1 && t.numel() > 0 && t.stride(0) != rows * stride) refuse(PyExc_TypeError, "%s: the groups of %s must follow one another", where, name);
    }
    if (groups) *groups = three ? t.size(0) : 1;
    v.device = t.device();
    return nb200_dense{all, cols, stride, type, t.data_ptr()};
}

nb200_expert_order view_order(PyObject *o, View &v) {
    const at::Tensor &slots = v.array(o, N_slots);
    int32_t d[2];
    dims_of<2>(o, d);
    v.device = slots.device();
    return nb200_expert_order{d[0], d[1], (int32_t)slots.numel(), v.index(o, N_token_offsets), v.index(o, N_offsets), v.index(o, N_rows), ints(slots)};
}

nb200_fp8 view_fp8(PyObject *o, View &v) {
    const at::Tensor &values = v.array(o, N_values), &scales = v.array(o, N_scales);
    int32_t d[3];
    dims_of<3>(o, d);
    Ref tiled(PyObject_GetAttr(o, g_name[N_tiled]));
    v.device = values.device();
    return nb200_fp8{d[0], d[1], d[2], tiled.p == Py_True, static_cast<uint8_t *>(values.data_ptr()), floats(scales)};
}

at::Tensor matrix(int64_t rows, int64_t cols, int type, c10::Device dev) { return at::Tensor(at::detail::empty_cuda({rows, cols}, scalar_of(type), dev, std::nullopt)); }
nb200_dense dense(const at::Tensor &t, int type) { return nb200_dense{t.size(0), t.size(1), t.size(1), type, t.data_ptr()}; }

struct OrderResult {  // the arrays of an order of R, and the object that holds them
    at::Tensor row_ptr, offsets, rows, slots;
    nb200_expert_order order{};
    int64_t entries;

    OrderResult(PyObject *r, const nb200_csr &a, c10::Device dev)
        : row_ptr(tensor_of(r, N_offsets)), offsets(int_array((int64_t)a.cols + 1, dev)), rows(int_array(a.nnz, dev)), slots(int_array(a.nnz, dev)), entries(a.nnz) {
        order.offsets = ints(offsets), order.rows = ints(rows), order.slots = ints(slots);
    }
    PyObject *object() {
        used(rows, entries), used(slots, entries);
        Result r(ORDER);
        r.set(N_offsets, offsets), r.set(N_rows, rows), r.set(N_slots, slots), r.set(N_token_offsets, row_ptr);
        const int32_t d[2] = {order.tokens, order.experts};
        r.dims<2>(d);
        return r.obj.release();
    }
};

struct Fp8Result {
    at::Tensor values, scales;
    nb200_fp8 m{};

    Fp8Result(int64_t groups, int64_t rows, int64_t cols, bool tiled, c10::Device dev) {
        m = nb200_fp8{(int32_t)groups, (int32_t)rows, (int32_t)cols, tiled, nullptr, nullptr};
        const int64_t n = nb200_fp8_value_count(&m), s = nb200_fp8_scale_count(&m);
        values = array(n, at::kByte, dev), scales = float_array(s, dev);
        m.values = static_cast<uint8_t *>(values.data_ptr()), m.scales = floats(scales);
        used(values, n), used(scales, s);
    }
    PyObject *object() {
        Result r(FP8);
        r.set(N_values, values), r.set(N_scales, scales);
        if (PyObject_SetAttr(r.obj.p, g_name[N_tiled], m.tiled ? Py_True : Py_False) < 0) throw PyFailure();
        const int32_t d[3] = {m.groups, m.rows, m.cols};
        r.dims<3>(d);
        return r.obj.release();
    }
};

PyObject *two(PyObject *a, PyObject *b) {
    Ref first(a), second(b);
    return PyTuple_Pack(2, first.p, second.p);
}
PyObject *wrap(const at::Tensor &t) { return THPVariable_Wrap(t); }

void extent(int64_t is, int64_t wanted, const char *where, const char *name, const char *what) {
    if (is == wanted) return;
    PyErr_Format(PyExc_ValueError, "%s: %s has %lld %s, %lld expected", where, name, (long long)is, what, (long long)wanted);
    throw PyFailure();
}
void same_type(int a, int b, const char *where) {
    if (a != b) refuse(PyExc_TypeError, "%s: operands differ in %s", where, "type");
}

PyObject *expert_order(PyObject *const *args) {
    const char *where = "gpu_expert_order";
    need_kind(args[0], CSR, where, "CSR_gpu");
    View vr;
    const nb200_csr r = view_csr(args[0], vr);
    OrderResult z(args[0], r, vr.device);
    launch({&vr}, where, [&](void *stream) { return nb200_expert_sort(&r, nullptr, &z.order, nullptr, stream); });
    return z.object();
}

PyObject *expert_sort(PyObject *const *args) {
    const char *where = "gpu_expert_sort";
    need_kind(args[0], CSR, where, "(CSR_gpu, tensor)");
    View vr, vx;
    const nb200_csr r = view_csr(args[0], vr);
    const nb200_dense x = view_dense(args[1], vx, where, "x");
    same_device(vr, vx);
    extent(x.rows, r.rows, where, "x", "rows");
    OrderResult z(args[0], r, vr.device);
    at::Tensor xs = matrix(r.nnz, x.cols, x.type, vr.device);
    nb200_dense out = dense(xs, x.type);
    launch({&vr, &vx}, where, [&](void *stream) { return nb200_expert_sort(&r, &x, &z.order, &out, stream); });
    return two(z.object(), wrap(xs));
}

PyObject *expert_sort_fp8(PyObject *const *args) {
    const char *where = "gpu_expert_sort_fp8";
    need_kind(args[0], CSR, where, "(CSR_gpu, tensor)");
    View vr, vx;
    const nb200_csr r = view_csr(args[0], vr);
    const nb200_dense x = view_dense(args[1], vx, where, "x");
    same_device(vr, vx);
    extent(x.rows, r.rows, where, "x", "rows");
    OrderResult z(args[0], r, vr.device);
    Fp8Result xs(1, r.nnz, x.cols, false, vr.device);
    launch({&vr, &vx}, where, [&](void *stream) { return nb200_expert_sort_fp8(&r, &x, &z.order, &xs.m, stream); });
    return two(z.object(), xs.object());
}

PyObject *expert_sort_grad(PyObject *const *args) {
    const char *where = "gpu_expert_sort_grad";
    need_kind(args[0], ORDER, where, "(ExpertOrder_gpu, tensor)");
    View vo, vz;
    const nb200_expert_order o = view_order(args[0], vo);
    const nb200_dense z = view_dense(args[1], vz, where, "dxs");
    same_device(vo, vz);
    extent(z.rows, o.entries, where, "dxs", "rows");
    at::Tensor y = matrix(o.tokens, z.cols, z.type, vo.device);
    nb200_dense out = dense(y, z.type);
    launch({&vo, &vz}, where, [&](void *stream) { return nb200_expert_unsort(&o, nullptr, &z, &out, stream); });
    return wrap(y);
}

// R is read for its values only.
nb200_csr routing_of(PyObject *r, PyObject *order, View &vr, View &vo, nb200_expert_order *o, const char *where) {
    need_kind(r, CSR, where, "(CSR_gpu, ExpertOrder_gpu, tensors)");
    need_kind(order, ORDER, where, "(CSR_gpu, ExpertOrder_gpu, tensors)");
    const nb200_csr a = view_csr(r, vr);
    *o = view_order(order, vo);
    same_device(vr, vo);
    extent(a.nnz, o->entries, where, "the routing", "entries");
    extent(a.rows, o->tokens, where, "the routing", "rows");
    return a;
}

PyObject *expert_unsort(PyObject *const *args) {
    const char *where = "gpu_expert_unsort";
    View vr, vo, vz;
    nb200_expert_order o;
    const nb200_csr r = routing_of(args[0], args[1], vr, vo, &o, where);
    const nb200_dense z = view_dense(args[2], vz, where, "z");
    same_device(vo, vz);
    extent(z.rows, o.entries, where, "z", "rows");
    at::Tensor y = matrix(o.tokens, z.cols, z.type, vo.device);
    nb200_dense out = dense(y, z.type);
    launch({&vr, &vo, &vz}, where, [&](void *stream) { return nb200_expert_unsort(&o, r.val, &z, &out, stream); });
    return wrap(y);
}

PyObject *expert_unsort_grad(PyObject *const *args) {
    const char *where = "gpu_expert_unsort_grad";
    View vr, vo, vz, vd;
    nb200_expert_order o;
    const nb200_csr r = routing_of(args[0], args[1], vr, vo, &o, where);
    const nb200_dense z = view_dense(args[2], vz, where, "z"), dy = view_dense(args[3], vd, where, "dy");
    same_device(vo, vz);
    same_device(vo, vd);
    extent(z.rows, o.entries, where, "z", "rows");
    extent(dy.rows, o.tokens, where, "dy", "rows");
    extent(dy.cols, z.cols, where, "dy", "columns");
    same_type(dy.type, z.type, where);
    at::Tensor dz = matrix(o.entries, z.cols, z.type, vo.device), dw = float_array(o.entries, vo.device);
    nb200_dense out = dense(dz, z.type);
    launch({&vr, &vo, &vz, &vd}, where, [&](void *stream) { return nb200_expert_unsort_grad(&o, r.val, &z, &dy, &out, floats(dw), stream); });
    used(dw, o.entries);
    return two(wrap(dz), wrap(dw));
}

PyObject *fp8_quantised(PyObject *x, bool tiled, const char *where) {
    View vx;
    int64_t groups = 1;
    const nb200_dense a = view_dense(x, vx, where, "x", tiled ? &groups : nullptr);
    Fp8Result z(groups, vx.arrays[0].size(-2), a.cols, tiled, vx.device);
    launch({&vx}, where, [&](void *stream) { return nb200_fp8_quantise(&a, &z.m, stream); });
    return z.object();
}
PyObject *fp8_rows(PyObject *const *args) { return fp8_quantised(args[0], false, "to_fp8_rows"); }
PyObject *fp8_tiles(PyObject *const *args) { return fp8_quantised(args[0], true, "to_fp8_tiles"); }

// fp8_pack(codes as bytes, scales, tiled): codes of 2 dimensions, or 3 where tiled; both contiguous (the caller has checked)
PyObject *fp8_pack(PyObject *const *args) {
    const char *where = "to_fp8";
    if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) refuse(PyExc_TypeError, "%s: %s must be torch tensors", where, "codes and scales");
    View vc;
    vc.arrays[vc.n++] = THPVariable_Unpack(args[0]);
    vc.arrays[vc.n++] = THPVariable_Unpack(args[1]);
    const at::Tensor &codes = vc.arrays[0], &scales = vc.arrays[1];
    vc.device = codes.device();
    const bool tiled = args[2] == Py_True;
    const int64_t groups = codes.dim() == 3 ? codes.size(0) : 1;
    Fp8Result z(groups, codes.size(-2), codes.size(-1), tiled, vc.device);
    launch({&vc}, where, [&](void *stream) { return nb200_fp8_pack(static_cast<const uint8_t *>(codes.data_ptr()), floats(scales), &z.m, stream); });
    return z.object();
}

PyObject *fp8_unpack(PyObject *const *args) {
    const char *where = "to_dense";
    need_kind(args[0], FP8, where, "FP8_gpu");
    View va;
    const nb200_fp8 a = view_fp8(args[0], va);
    at::Tensor z = matrix((int64_t)a.groups * a.rows, a.cols, NB200_F32, va.device);
    launch({&va}, where, [&](void *stream) { return nb200_fp8_unpack(&a, floats(z), stream); });
    return wrap(z);
}

PyObject *fp8_transpose(PyObject *const *args) {
    const char *where = "transposed";
    need_kind(args[0], FP8, where, "FP8_gpu");
    View va;
    const nb200_fp8 a = view_fp8(args[0], va);
    Fp8Result z(a.groups, a.cols, a.rows, true, va.device);
    launch({&va}, where, [&](void *stream) { return nb200_fp8_transpose(&a, &z.m, stream); });
    return z.object();
}

// Row ranges of the groups: an order's, or none for a single matrix.
const int32_t *ranges_of(PyObject *order, View &vo, int64_t rows, int64_t groups, const char *where) {
    if (order == Py_None) {
        extent(groups, 1, where, "w without an order", "groups");
        return nullptr;
    }
    need_kind(order, ORDER, where, "ExpertOrder_gpu (or None)");
    const nb200_expert_order o = view_order(order, vo);
    extent(rows, o.entries, where, "the left operand", "rows");
    extent(groups, o.experts, where, "w", "groups");
    return o.offsets;
}

// fp8_product(a, w, order or None, type)
PyObject *fp8_product(PyObject *const *args) {
    const char *where = "gpu_fp8_product";
    for (int k = 0; k < 2; ++k) need_kind(args[k], FP8, where, "FP8_gpu");
    View va, vw, vo;
    const nb200_fp8 a = view_fp8(args[0], va), w = view_fp8(args[1], vw);
    same_device(va, vw);
    vo.device = va.device;
    const int32_t *offsets = ranges_of(args[2], vo, a.rows, w.groups, where);
    same_device(va, vo);
    if (a.tiled || !w.tiled) refuse(PyExc_ValueError, "%s: %s", where, "the left operand has a scale per row (to_fp8_rows), the right one per tile (to_fp8_tiles)");
    extent(a.cols, w.cols, where, "the left operand", "columns");
    const int type = (int)PyLong_AsLong(args[3]);
    at::Tensor y = matrix(a.rows, w.rows, type, va.device);
    nb200_dense out = dense(y, type);
    launch({&va, &vw, &vo}, where, [&](void *stream) { return nb200_fp8_product(&a, &w, offsets, &out, stream); });
    return wrap(y);
}

// fp8_grad_w(dy, x, order or None, groups): the weights' gradient and dy quantised by rows
PyObject *fp8_grad_w(PyObject *const *args) {
    const char *where = "gpu_fp8_product_grad";
    View vd, vx, vo;
    const nb200_dense dy = view_dense(args[0], vd, where, "dy"), x = view_dense(args[1], vx, where, "x");
    same_device(vd, vx);
    same_type(dy.type, x.type, where);
    extent(x.rows, dy.rows, where, "x", "rows");
    const int64_t groups = PyLong_AsLongLong(args[3]);
    vo.device = vd.device;
    const int32_t *offsets = ranges_of(args[2], vo, dy.rows, groups, where);
    same_device(vd, vo);
    const int64_t bytes = nb200_fp8_product_grad_w_scratch(&dy, &x, (int32_t)groups);
    if (bytes < 0) check(NB200_E_BADARG, where);
    at::Tensor scratch = array(bytes, at::kByte, vd.device), z = at::Tensor(at::detail::empty_cuda({groups, dy.cols, x.cols}, at::kFloat, vd.device, std::nullopt));
    Fp8Result rows(1, dy.rows, dy.cols, false, vd.device);
    launch({&vd, &vx, &vo}, where,
           [&](void *stream) { return nb200_fp8_product_grad_w(&dy, &x, (int32_t)groups, offsets, floats(z), &rows.m, scratch.data_ptr(), bytes, stream); });
    return two(wrap(z), rows.object());
}

// ---- layers ----------------------------------------------------------------------------------

// A dense operand of a gated layer: 16-bit.
nb200_dense view_half(PyObject *o, View &v, const char *where, const char *name, int64_t *groups = nullptr) {
    const nb200_dense x = view_dense(o, v, where, name, groups);
    if (x.type == NB200_F32) refuse(PyExc_TypeError, "%s: %s must be float16 or bfloat16", where, name);
    return x;
}

// w: [2 hidden][width] or one per expert; hidden
int64_t hidden_of(const View &vw, const char *where) {
    const int64_t rows = vw.arrays[0].size(-2);
    if (rows % 2) refuse(PyExc_ValueError, "%s: %s must hold as many rows of gates as of values", where, "w");
    return rows / 2;
}

int64_t with_scratch(int64_t bytes, const char *where) {
    if (bytes < 0) check(NB200_E_BADARG, where);
    return bytes;
}

// gated_product(x, w, order or None, activation, keep): h, or (h, both)
PyObject *gated_product(PyObject *const *args) {
    const char *where = "gpu_gated_product";
    View vx, vw, vo;
    int64_t groups = 1;
    const nb200_dense x = view_half(args[0], vx, where, "x"), w = view_half(args[1], vw, where, "w", &groups);
    same_device(vx, vw);
    same_type(x.type, w.type, where);
    extent(x.cols, w.cols, where, "x", "columns");
    const int64_t hidden = hidden_of(vw, where);
    vo.device = vx.device;
    const int32_t *offsets = ranges_of(args[2], vo, x.rows, groups, where);
    same_device(vx, vo);
    const int activation = (int)PyLong_AsLong(args[3]);
    const bool keep = args[4] == Py_True;
    at::Tensor h = matrix(x.rows, hidden, x.type, vx.device), both;
    nb200_dense out = dense(h, x.type), sums{};
    if (keep) both = matrix(x.rows, 2 * hidden, x.type, vx.device), sums = dense(both, x.type);
    const int64_t bytes = with_scratch(nb200_gated_product_scratch(&x, &w, (int32_t)groups), where);
    at::Tensor scratch;
    if (bytes) scratch = array(bytes, at::kByte, vx.device);
    launch({&vx, &vw, &vo}, where, [&](void *stream) {
        return nb200_gated_product(&x, &w, (int32_t)groups, offsets, activation, &out, keep ? &sums : nullptr, bytes ? scratch.data_ptr() : nullptr, bytes, stream);
    });
    return keep ? two(wrap(h), wrap(both)) : wrap(h);
}

// gated_product_grad(dh, both, x, w, order or None, activation): (dx, dw)
PyObject *gated_product_grad(PyObject *const *args) {
    const char *where = "gpu_gated_product_grad";
    View vd, vb, vx, vw, vo;
    int64_t groups = 1;
    const nb200_dense dh = view_half(args[0], vd, where, "dh"), both = view_half(args[1], vb, where, "both"), x = view_half(args[2], vx, where, "x");
    const nb200_dense w = view_half(args[3], vw, where, "w", &groups);
    for (const View *v : {&vb, &vx, &vw}) same_device(vd, *v);
    for (const nb200_dense *o : {&both, &x, &w}) same_type(dh.type, o->type, where);
    const int64_t hidden = hidden_of(vw, where);
    extent(x.cols, w.cols, where, "x", "columns");
    extent(dh.cols, hidden, where, "dh", "columns");
    extent(both.cols, 2 * hidden, where, "both", "columns");
    extent(dh.rows, x.rows, where, "dh", "rows");
    extent(both.rows, x.rows, where, "both", "rows");
    vo.device = vx.device;
    const int32_t *offsets = ranges_of(args[4], vo, x.rows, groups, where);
    same_device(vx, vo);
    const int activation = (int)PyLong_AsLong(args[5]);
    at::Tensor dx = matrix(x.rows, x.cols, x.type, vx.device), dw = at::Tensor(at::detail::empty_cuda(vw.arrays[0].sizes(), scalar_of(x.type), vx.device, std::nullopt));
    nb200_dense out_x = dense(dx, x.type), out_w{w.rows, w.cols, w.cols, x.type, dw.data_ptr()};
    const int64_t bytes = with_scratch(nb200_gated_product_grad_scratch(&x, &w, (int32_t)groups), where);
    at::Tensor scratch = array(bytes, at::kByte, vx.device);
    launch({&vd, &vb, &vx, &vw, &vo}, where, [&](void *stream) {
        return nb200_gated_product_grad(&dh, &both, &x, &w, (int32_t)groups, offsets, activation, &out_x, &out_w, scratch.data_ptr(), bytes, stream);
    });
    return two(wrap(dx), wrap(dw));
}

nb200_int8 view_int8(PyObject *o, View &v) {
    const at::Tensor &values = v.array(o, N_values), &scales = v.array(o, N_scales);
    int32_t d[3];
    dims_of<3>(o, d);
    v.device = values.device();
    return nb200_int8{d[0], d[1], d[2], static_cast<int8_t *>(values.data_ptr()), floats(scales)};
}

struct Int8Result {
    at::Tensor values, scales;
    nb200_int8 m{};

    Int8Result(int64_t groups, int64_t rows, int64_t cols, c10::Device dev, const char *where) {
        m = nb200_int8{(int32_t)groups, (int32_t)rows, (int32_t)cols, nullptr, nullptr};
        const int64_t n = with_scratch(nb200_int8_value_count(&m), where), s = groups * rows;
        values = array(n, at::kChar, dev), scales = float_array(s, dev);
        m.values = static_cast<int8_t *>(values.data_ptr()), m.scales = floats(scales);
        used(values, n), used(scales, s);
    }
    PyObject *object() {
        Result r(INT8);
        r.set(N_values, values), r.set(N_scales, scales);
        const int32_t d[3] = {m.groups, m.rows, m.cols};
        r.dims<3>(d);
        return r.obj.release();
    }
};

PyObject *int8_rows(PyObject *const *args) {
    const char *where = "to_int8_rows";
    View vx;
    int64_t groups = 1;
    const nb200_dense a = view_dense(args[0], vx, where, "x", &groups);
    Int8Result z(groups, vx.arrays[0].size(-2), a.cols, vx.device, where);
    launch({&vx}, where, [&](void *stream) { return nb200_int8_quantise(&a, &z.m, stream); });
    return z.object();
}

// int8_pack(codes, scales): int8 codes of 2 or 3 dimensions, a scale per row; both contiguous (the caller has checked)
PyObject *int8_pack(PyObject *const *args) {
    const char *where = "to_int8_rows";
    if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) refuse(PyExc_TypeError, "%s: %s must be torch tensors", where, "codes and scales");
    View vc;
    vc.arrays[vc.n++] = THPVariable_Unpack(args[0]);
    vc.arrays[vc.n++] = THPVariable_Unpack(args[1]);
    const at::Tensor &codes = vc.arrays[0], &scales = vc.arrays[1];
    vc.device = codes.device();
    Int8Result z(codes.dim() == 3 ? codes.size(0) : 1, codes.size(-2), codes.size(-1), vc.device, where);
    launch({&vc}, where, [&](void *stream) { return nb200_int8_pack(static_cast<const int8_t *>(codes.data_ptr()), floats(scales), &z.m, stream); });
    return z.object();
}

PyObject *int8_unpack(PyObject *const *args) {
    const char *where = "to_dense";
    need_kind(args[0], INT8, where, "INT8_gpu");
    View va;
    const nb200_int8 a = view_int8(args[0], va);
    at::Tensor z = matrix((int64_t)a.groups * a.rows, a.cols, NB200_F32, va.device);
    launch({&va}, where, [&](void *stream) { return nb200_int8_unpack(&a, floats(z), stream); });
    return wrap(z);
}

// int8_product(a, w, order or None, type)
PyObject *int8_product(PyObject *const *args) {
    const char *where = "gpu_int8_product";
    for (int k = 0; k < 2; ++k) need_kind(args[k], INT8, where, "INT8_gpu");
    View va, vw, vo;
    const nb200_int8 a = view_int8(args[0], va), w = view_int8(args[1], vw);
    same_device(va, vw);
    extent(a.groups, 1, where, "the left operand", "groups");
    extent(a.cols, w.cols, where, "the left operand", "columns");
    vo.device = va.device;
    const int32_t *offsets = ranges_of(args[2], vo, a.rows, w.groups, where);
    same_device(va, vo);
    const int type = (int)PyLong_AsLong(args[3]);
    at::Tensor y = matrix(a.rows, w.rows, type, va.device);
    nb200_dense out = dense(y, type);
    launch({&va, &vw, &vo}, where, [&](void *stream) { return nb200_int8_product(&a, &w, offsets, &out, stream); });
    return wrap(y);
}

// Tensors in a row, as a list or a tuple.
std::vector<at::Tensor> tensors_of(PyObject *o, const char *where, const char *name) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) refuse(PyExc_TypeError, "%s: %s must be a list or a tuple of CUDA tensors", where, name);
    std::vector<at::Tensor> all;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
    all.reserve((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject *t = PySequence_Fast_GET_ITEM(o, i);
        if (!THPVariable_Check(t)) refuse(PyExc_TypeError, "%s: %s must be a list or a tuple of CUDA tensors", where, name);
        all.push_back(THPVariable_Unpack(t));
        const at::Tensor &x = all.back();
        if (!x.is_cuda() || x.layout() != at::kStrided || type_of(x) < 0) refuse(PyExc_TypeError, "%s: %s must hold CUDA tensors of float32, float16 or bfloat16", where, name);
        if (!x.is_non_overlapping_and_dense()) refuse(PyExc_ValueError, "%s: the elements of each of %s must lie one after another", where, name);
        if (x.device() != all.front().device()) refuse(PyExc_ValueError, "%s: %s live on different devices", where, name);
    }
    return all;
}

// clip(tensors, results or None, max_norm): the norm
PyObject *clip(PyObject *const *args) {
    const char *where = "gpu_clip_gradients";
    const std::vector<at::Tensor> from = tensors_of(args[0], where, "gradients");
    const bool in_place = args[1] == Py_None;
    const std::vector<at::Tensor> others = in_place ? std::vector<at::Tensor>() : tensors_of(args[1], where, "out"), &to = in_place ? from : others;
    if (from.empty()) refuse(PyExc_ValueError, "%s: %s are none", where, "gradients");
    if (from.size() != to.size() || to.empty()) refuse(PyExc_ValueError, "%s: %s must hold as many tensors as there are gradients", where, "out");
    const double max_norm = PyFloat_AsDouble(args[2]);
    const c10::Device device = from[0].device();
    if (to[0].device() != device) refuse(PyExc_ValueError, "%s: gradients and %s live on different devices", where, "out");
    std::vector<nb200_span> spans;
    typedef std::pair<uintptr_t, uintptr_t> Range;
    std::vector<Range> read, written;  // what is both is written
    spans.reserve(from.size()), written.reserve(from.size());
    if (!in_place) read.reserve(from.size());
    for (size_t i = 0; i < from.size(); ++i) {
        const at::Tensor &x = from[i], &z = to[i];
        if (!in_place && (x.sizes() != z.sizes() || !(x.strides() == z.strides() || (x.is_contiguous() && z.is_contiguous()))))
            refuse(PyExc_ValueError, "%s: a tensor of %s differs from its gradient in shape or layout", where, "out");
        const int64_t n = x.numel();
        if (n == 0) continue;
        const int type = type_of(x), to_type = in_place ? type : type_of(z);
        const nb200_span s{x.data_ptr(), in_place ? x.data_ptr() : z.data_ptr(), n, type, to_type};
        spans.push_back(s);
        const uintptr_t a = reinterpret_cast<uintptr_t>(s.from), b = reinterpret_cast<uintptr_t>(s.to);
        if (a != b || type != to_type) read.emplace_back(a, a + (size_t)n * (type == NB200_F32 ? 4 : 2));
        written.emplace_back(b, b + (size_t)n * (to_type == NB200_F32 ? 4 : 2));
    }
    for (std::vector<Range> *r : {&read, &written})
        if (!std::is_sorted(r->begin(), r->end())) std::sort(r->begin(), r->end());
    const char *what = in_place ? "gradients" : "gradients and out";
    uintptr_t end = 0;
    size_t next = 0;
    for (const Range &w : written) {
        if (w.first < end) refuse(PyExc_ValueError, "%s: %s overlap one another in memory", where, what);
        end = w.second;
        while (next < read.size() && read[next].second <= w.first) ++next;
        if (next < read.size() && read[next].first < w.second) refuse(PyExc_ValueError, "%s: %s overlap one another in memory", where, what);
    }
    const int64_t bytes = with_scratch(nb200_clip_scratch(spans.data(), (int64_t)spans.size()), where);
    at::Tensor scratch = array(bytes, at::kByte, device), norm = at::Tensor(at::detail::empty_cuda({}, at::kFloat, device, std::nullopt));
    // A tensor that must not be written here is refused before any of them counts as changed.
    if (!c10::InferenceMode::is_enabled())
        for (const at::Tensor &z : to)
            if (z.is_inference()) refuse(PyExc_RuntimeError, "%s: %s of inference mode cannot be changed outside of it", where, in_place ? "gradients" : "out");
    for (const at::Tensor &z : to) z.unsafeGetTensorImpl()->bump_version();
    View v;
    v.device = device;
    const int status = run({&v}, [&](void *stream) { return nb200_clip(spans.data(), (int64_t)spans.size(), (float)max_norm, floats(norm), scratch.data_ptr(), bytes, stream); });
    const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream(device.index());
    const void *last = nullptr;  // parts of one long buffer follow one another
    auto record = [&](const at::Tensor &t) {
        const c10::DataPtr &p = t.storage().data_ptr();
        if (p.get() != last) c10::cuda::CUDACachingAllocator::recordStream(p, current);
        last = p.get();
    };
    for (const at::Tensor &x : from) record(x);
    if (!in_place)
        for (const at::Tensor &z : to) record(z);
    check(status, where);  // behind that: of several launches the first may be under way
    return wrap(norm);
}

// ---- module --------------------------------------------------------------------------------

template <PyObject *(*OP)(PyObject *const *), int ARGS>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != ARGS) {
        PyErr_Format(PyExc_TypeError, "%d operands expected, %zd given", ARGS, n);
        return nullptr;
    }
    try {
        return OP(args);
    } catch (const PyFailure &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// bind((CSR_gpu, COO_gpu, DCSR_gpu, COO3_gpu, CSF3_gpu, Scalar_gpu), check)
PyObject *bind(PyObject *, PyObject *args) {
    PyObject *classes, *check_fn;
    if (!PyArg_ParseTuple(args, "O!O", &PyTuple_Type, &classes, &check_fn)) return nullptr;
    if (PyTuple_GET_SIZE(classes) != KINDS) return PyErr_Format(PyExc_TypeError, "bind: %d classes expected", (int)KINDS);
    for (int k = 0; k < KINDS; ++k) {
        PyObject *c = PyTuple_GET_ITEM(classes, k);
        if (!PyType_Check(c)) return PyErr_Format(PyExc_TypeError, "bind: not a class");
        Py_INCREF(c);
        g_class[k] = reinterpret_cast<PyTypeObject *>(c);
    }
    Py_INCREF(check_fn);
    g_check = check_fn;
    Py_RETURN_NONE;
}

// bind_experts((ExpertOrder_gpu, FP8_gpu))
PyObject *bind_experts(PyObject *, PyObject *args) {
    PyObject *classes[2];
    if (!PyArg_ParseTuple(args, "(O!O!)", &PyType_Type, &classes[0], &PyType_Type, &classes[1])) return nullptr;
    for (int k = 0; k < 2; ++k) {
        Py_INCREF(classes[k]);
        g_class[ORDER + k] = reinterpret_cast<PyTypeObject *>(classes[k]);
    }
    Py_RETURN_NONE;
}

// bind_layers(INT8_gpu)
PyObject *bind_layers(PyObject *, PyObject *args) {
    PyObject *c;
    if (!PyArg_ParseTuple(args, "O!", &PyType_Type, &c)) return nullptr;
    Py_INCREF(c);
    g_class[INT8] = reinterpret_cast<PyTypeObject *>(c);
    Py_RETURN_NONE;
}

// turn_of(device, stream handle): identity of the lock by which calls there take turns (for tests)
PyObject *turn_of(PyObject *, PyObject *args) {
    int device;
    unsigned long long stream;
    if (!PyArg_ParseTuple(args, "iK", &device, &stream)) return nullptr;
    return PyLong_FromVoidPtr(&stream_lock(device, reinterpret_cast<void *>(stream)));
}

template <PyObject *(*OP)(PyObject *const *), int ARGS>
PyMethodDef op(const char *name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<OP, ARGS>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr}, {"turn_of", turn_of, METH_VARARGS, nullptr},
    op<csr_add, 2>("csr_add"), op<csr_mul, 2>("csr_mul"), op<csr_add_3, 3>("csr_add_3"), op<spgemm, 2>("spgemm"),
    op<sssmm, 3>("sssmm"), op<coo3d_add, 2>("coo3d_add"), op<csf_add, 2>("csf_add"), op<coo_add, 2>("coo_add"),
    op<coo_mul, 2>("coo_mul"), op<coo_csr_add, 2>("coo_csr_add"), op<dcsr_add, 2>("dcsr_add"), op<dcsr_mul, 2>("dcsr_mul"),
    op<inner_prod, 2>("inner_prod"), op<inner_prod_coo, 2>("inner_prod_coo"),
    {"bind_experts", bind_experts, METH_VARARGS, nullptr},
    op<expert_order, 1>("expert_order"), op<expert_sort, 2>("expert_sort"), op<expert_sort_fp8, 2>("expert_sort_fp8"),
    op<expert_sort_grad, 2>("expert_sort_grad"), op<expert_unsort, 3>("expert_unsort"), op<expert_unsort_grad, 4>("expert_unsort_grad"),
    op<fp8_rows, 1>("fp8_rows"), op<fp8_tiles, 1>("fp8_tiles"), op<fp8_pack, 3>("fp8_pack"), op<fp8_unpack, 1>("fp8_unpack"),
    op<fp8_transpose, 1>("fp8_transpose"), op<fp8_product, 4>("fp8_product"), op<fp8_grad_w, 4>("fp8_grad_w"),
    {"bind_layers", bind_layers, METH_VARARGS, nullptr},
    op<gated_product, 5>("gated_product"), op<gated_product_grad, 6>("gated_product_grad"), op<int8_rows, 1>("int8_rows"), op<int8_pack, 2>("int8_pack"),
    op<int8_unpack, 1>("int8_unpack"), op<int8_product, 4>("int8_product"), op<clip, 3>("clip"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() {
    for (int k = 0; k < NAMES; ++k)
        if (!(g_name[k] = PyUnicode_InternFromString(NAME_TEXT[k]))) return nullptr;
    return PyModule_Create(&g_module);
}
