// Python calls of the paged cache's entries (include/wtalign.h, wt_kv_*): the argument checks of kvcache.PagedKVCache, the
// results' tensors and the launch in one step.  A decoder makes two such calls per layer and token, and their kernels take 3
// to 6 us; checks written in Python and a ctypes call took 8 us of the host, these take 4.
// The library itself knows no tensors: its entries come in as addresses.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cmath>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "wt_overlap.h"
#include "wtalign.h"

namespace {

PyObject *g_error = nullptr;   // _lib.WtError
decltype(&wt_kv_append) g_append = nullptr;
decltype(&wt_kv_gather) g_gather = nullptr;
decltype(&wt_kv_attend) g_attend = nullptr;
decltype(&wt_kv_attend_workspace) g_workspace = nullptr;
decltype(&wt_last_error) g_last_error = nullptr;

struct Cache {
    wt_kv_cache desc;
    int device;   // -1: host memory, whose every call is refused
    at::ScalarType type;
    at::Storage kept[5];   // what desc points into lives as long as it
    const void *start[5];  // ... and has to be where it was
    size_t bytes[5];
    wt::Strided3 memory[4];   // k, v and their exponents
    c10::VariableVersion version[4];
};
constexpr const char *PARTS[4] = {"k", "v", "k_exp", "v_exp"};
constexpr const char *CACHE = "wt_kv_cache";

struct Refused {};   // the Python error is set

template <typename... A>
[[noreturn]] void refuse(const char *format, A... args) {
    PyErr_Format(g_error, format, args...);
    throw Refused();
}
void check(int64_t rc, const char *what) {
    if (rc < 0) refuse("%s failed (rc=%d): %s", what, (int)rc, g_last_error());
}

Cache *cache_of(PyObject *o) {
    Cache *c = static_cast<Cache *>(PyCapsule_GetPointer(o, CACHE));
    if (!c) throw Refused();
    for (int i = 0; i < 5; ++i)
        if (c->kept[i] && (c->kept[i].data() != c->start[i] || c->kept[i].nbytes() < c->bytes[i]))
            refuse("the cache's memory has been resized or moved since it was made");
    return c;
}
// A tensor that means what its memory holds and nothing else, and whose memory is there: a storage may have been resized under it
void plain(const at::Tensor &t, const char *name) {
    if (t.numel() > 0) {
        int64_t last = t.storage_offset();
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        if (!t.has_storage() || !t.storage().data() || (uint64_t)(last + 1) * t.element_size() > t.storage().nbytes())
            refuse("%s: not all of it has memory", name);
    }
    if (t.is_neg()) refuse("%s: a view that is negated when it is read: call resolve_neg()", name);
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        refuse("%s has a tangent (forward-mode differentiation), which the cache's calls do not have", name);
}
const at::Tensor &tensor(PyObject *o, const Cache *c, const char *name, int64_t dim) {
    if (!THPVariable_Check(o)) refuse("%s: not a tensor", name);
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.layout() != at::kStrided || (t.is_cuda() ? (int)t.get_device() : t.is_cpu() ? -1 : -2) != c->device)
        refuse("%s: not a tensor of the cache's device", name);
    if (t.dim() != dim) refuse("%s: %d dimensions, not %d", name, (int)t.dim(), (int)dim);
    plain(t, name);
    return t;
}
bool is_none(PyObject *o) { return o == Py_None; }

// what a call has written: autograd's saved tensors in the same memory are out of date (inference tensors have no versions)
void written(c10::VariableVersion version) {
    if (version.enabled()) version.bump();
}
c10::VariableVersion version_of(const at::Tensor &t) { return t.unsafeGetTensorImpl()->version_counter(); }

// Nothing here has a gradient; a call that autograd would have to record is refused rather than left out of the graph.
void no_gradient(const at::Tensor &t, const char *name) {
    if (t.requires_grad() && at::GradMode::is_enabled()) refuse("%s requires a gradient, which the cache's calls do not have: call them under torch.no_grad()", name);
}

int dtype_of(at::ScalarType s, const Cache *c, const char *name) {   // an 8-bit cache takes and gives any of three types, another its own
    const int dt = s == at::kFloat ? WT_DTYPE_F32 : s == at::kHalf ? WT_DTYPE_F16 : s == at::kBFloat16 ? WT_DTYPE_BF16 : -1;
    if (dt < 0 || (c->desc.dtype != WT_DTYPE_E4M3 && s != c->type))
        refuse("%s: %s with a cache of %s", name, c10::toString(s), c10::toString(c->type));
    return dt;
}

struct Table {
    const int32_t *p;
    int64_t stride;
    int n, width;
};
Table table_of(PyObject *o, const Cache *c) {
    const at::Tensor &t = tensor(o, c, "page table", 2);
    const int64_t n = t.size(0), width = t.size(1);
    if (t.scalar_type() != at::kInt) refuse("page table: not int32");
    if (width < 1 || (width > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < width))
        refuse("page table: the pages of a sequence stand side by side, its rows apart (strides %ld, %ld)", (long)t.stride(0), (long)t.stride(1));
    if (n > INT32_MAX || width > WT_KV_MAX_POSITIONS / c->desc.page_size)
        refuse("page table: %ld pages of %d are more than %d positions", (long)width, c->desc.page_size, WT_KV_MAX_POSITIONS);
    return {static_cast<const int32_t *>(t.const_data_ptr()), n > 1 ? t.stride(0) : width, (int)n, (int)width};
}
const int32_t *int32s(PyObject *o, const Cache *c, const char *name, int64_t n) {
    const at::Tensor &t = tensor(o, c, name, 1);
    if (t.scalar_type() != at::kInt || t.size(0) != n || (n > 1 && t.stride(0) != 1)) refuse("%s: %ld int32, side by side", name, (long)n);
    return static_cast<const int32_t *>(t.const_data_ptr());
}

struct Rows {
    Table table;
    const int32_t *sequences, *positions;
    int n;
};
Rows rows_of(PyObject *table, PyObject *positions, PyObject *sequences, const Cache *c) {
    Rows r;
    r.table = table_of(table, c);
    const int64_t n = tensor(positions, c, "positions", 1).size(0);
    if (n > INT32_MAX) refuse("positions: %ld rows", (long)n);
    r.n = (int)n;
    r.positions = int32s(positions, c, "positions", n);
    r.sequences = is_none(sequences) ? nullptr : int32s(sequences, c, "sequences", n);
    if (!r.sequences && n > r.table.n) refuse("%ld rows for %d sequences: say whose they are (sequences=)", (long)n, r.table.n);
    return r;
}

struct Strided {
    void *p;
    int64_t row, head;
};
// (rows, heads, head_dim); a dimension of size one has no stride to speak of
Strided strided(const at::Tensor &t, const Cache *c, const char *name, int64_t n, int64_t heads, bool whole16) {
    if (t.size(0) != n || t.size(1) != heads || t.size(2) != c->desc.head_dim)
        refuse("%s: (%ld, %ld, %ld), not (%ld, %ld, %d)", name, (long)t.size(0), (long)t.size(1), (long)t.size(2), (long)n, (long)heads, c->desc.head_dim);
    Strided s = {t.data_ptr(), n > 1 ? t.stride(0) : 0, heads > 1 ? t.stride(1) : 0};
    const int64_t item = t.element_size();
    if (n > 0 && (t.stride(2) != 1 || (whole16 && (((uintptr_t)s.p | (uint64_t)(s.row * item) | (uint64_t)(s.head * item)) & 15))))
        refuse("%s: a head's values stand side by side%s (strides %ld, %ld, %ld)", name, whole16 ? ", heads and rows start on 16-byte steps" : "",
               (long)t.stride(0), (long)t.stride(1), (long)t.stride(2));
    return s;
}

wt::Strided3 memory_of(const at::Tensor &t, int rows) {   // `rows` dimensions of rows of adjacent values
    int64_t row = t.element_size(), stride[3];
    for (int i = rows; i < t.dim(); ++i) row *= t.size(i);
    for (int i = 0; i < rows; ++i) stride[i] = t.stride(i) * t.element_size();
    return wt::Strided3(t.const_data_ptr(), row, rows, t.sizes().data(), stride);
}

void not_the_caches(const wt::Strided3 &m, const Cache *c, const char *name) {
    for (const wt::Strided3 &part : c->memory)
        if (wt::overlap(m, part)) refuse("%s: the cache's own memory", name);
}

// the cache's device is the current one, and its current stream the launch's
struct On {
    int before = -1;
    void *stream = nullptr;
    explicit On(const Cache *c) {
        if (c->device < 0) refuse("the cache's kernels only run on the GPU");
        const int now = c10::hip::current_device();
        if (now != c->device) {
            c10::hip::set_device((c10::DeviceIndex)c->device);
            before = now;
        }
        stream = c10::hip::getCurrentHIPStream((c10::DeviceIndex)c->device).stream();
    }
    ~On() {
        if (before >= 0) try {
                c10::hip::set_device((c10::DeviceIndex)before);
            } catch (...) {   // (it was the current one: nothing left to say in a destructor)
            }
    }
};

void arguments(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) refuse("%d arguments, not %d", (int)got, (int)want);
}

PyObject *setup(PyObject *, PyObject *args) {   // error class, addresses of the entries
    unsigned long long a[5];
    PyObject *error;
    if (!PyArg_ParseTuple(args, "OKKKKK", &error, &a[0], &a[1], &a[2], &a[3], &a[4])) return nullptr;
    Py_INCREF(error);
    Py_XDECREF(g_error);
    g_error = error;
    g_append = reinterpret_cast<decltype(g_append)>(a[0]);
    g_gather = reinterpret_cast<decltype(g_gather)>(a[1]);
    g_attend = reinterpret_cast<decltype(g_attend)>(a[2]);
    g_workspace = reinterpret_cast<decltype(g_workspace)>(a[3]);
    g_last_error = reinterpret_cast<decltype(g_last_error)>(a[4]);
    Py_RETURN_NONE;
}

// (pages, heads, slots, head_dim): values of a row side by side, 16-byte steps, no two rows in one place
const at::Tensor &pages(PyObject *o, const char *name, int *dtype) {
    if (!THPVariable_Check(o)) refuse("%s: not a tensor", name);
    const at::Tensor &t = THPVariable_Unpack(o);
    const at::ScalarType s = t.scalar_type();
    *dtype = s == at::kFloat ? WT_DTYPE_F32 : s == at::kHalf ? WT_DTYPE_F16 : s == at::kBFloat16 ? WT_DTYPE_BF16 : s == at::kFloat8_e4m3fn ? WT_DTYPE_E4M3 : -1;
    if (t.layout() != at::kStrided || t.dim() != 4 || *dtype < 0)
        refuse("%s: a 4-dimensional tensor (pages, heads, slots, head_dim) of float32, float16, bfloat16 or float8_e4m3fn", name);
    plain(t, name);
    t.mutable_data_ptr();   // (a lazy clone gets its memory now, before addresses are compared and kept)
    const int64_t d = t.size(3);
    if (t.numel() == 0 || (d != 32 && d != 64 && d != 96 && d != 128 && d != 256))
        refuse("%s: (%ld, %ld, %ld, %ld); head_dim is 32, 64, 96, 128 or 256, nothing is empty", name, (long)t.size(0), (long)t.size(1), (long)t.size(2), (long)d);
    if (t.size(0) > INT32_MAX || t.size(1) > 65535 || t.size(2) > INT32_MAX)
        refuse("%s: (%ld, %ld, %ld, %ld) is beyond 32-bit page and slot numbers or 65535 heads", name, (long)t.size(0), (long)t.size(1), (long)t.size(2), (long)d);
    bool steps = t.stride(3) == 1 && ((uintptr_t)t.const_data_ptr() & 15) == 0;
    int order[3], n = 0;   // dimensions that have a stride to speak of, the nearest rows first
    for (int i = 0; i < 3; ++i)
        if (t.size(i) > 1) {
            steps = steps && t.stride(i) * t.element_size() % 16 == 0;
            int j = n++;
            for (; j > 0 && t.stride(order[j - 1]) > t.stride(i); --j) order[j] = order[j - 1];
            order[j] = i;
        }
    if (!steps) refuse("%s: rows must be contiguous and start on 16-byte steps (strides %ld, %ld, %ld, %ld)", name, (long)t.stride(0), (long)t.stride(1), (long)t.stride(2), (long)t.stride(3));
    int64_t extent = d;
    for (int i = 0; i < n; ++i) {
        if (t.stride(order[i]) < extent) refuse("%s: rows overlap (strides %ld, %ld, %ld, %ld)", name, (long)t.stride(0), (long)t.stride(1), (long)t.stride(2), (long)t.stride(3));
        extent += t.stride(order[i]) * (t.size(order[i]) - 1);
    }
    return t;
}

// k, v, k_exp or None, v_exp or None, host (tensors of the host's memory are taken, for calls that are refused in the end) ->
// (handle, error word)
PyObject *make(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        arguments(n, 5);
        int dtype, v_dtype;
        const at::Tensor &k = pages(args[0], "k", &dtype), &v = pages(args[1], "v", &v_dtype);
        if (k.requires_grad() || v.requires_grad()) refuse("k, v: pages have no gradient");
        if (k.sizes() != v.sizes() || dtype != v_dtype) refuse("k and v differ in shape or type");
        if (k.const_data_ptr() == v.const_data_ptr()) refuse("k and v are the same memory");
        uint8_t *e[2] = {nullptr, nullptr};
        at::Storage es[2];
        wt::Strided3 memory[4] = {memory_of(k, 3), memory_of(v, 3)};
        c10::VariableVersion version[4] = {version_of(k), version_of(v), version_of(k), version_of(v)};
        for (int i = 0; i < 2; ++i) {
            const char *name = i == 0 ? "k_exp" : "v_exp";
            if (is_none(args[2 + i]) == (dtype == WT_DTYPE_E4M3)) refuse("%s: a float8_e4m3fn cache has exponents, another has none", name);
            if (dtype != WT_DTYPE_E4M3) continue;
            if (!THPVariable_Check(args[2 + i])) refuse("%s: not a tensor", name);
            const at::Tensor &x = THPVariable_Unpack(args[2 + i]);
            if (x.layout() != at::kStrided || x.scalar_type() != at::kByte || x.dim() != 3 || x.size(0) != k.size(0) || x.size(1) != k.size(1) || x.size(2) != k.size(2) ||
                !x.is_contiguous() || ((uintptr_t)x.const_data_ptr() & 15) || x.device() != k.device())
                refuse("%s: contiguous uint8 (%ld, %ld, %ld) beside the pages, 16-byte aligned", name, (long)k.size(0), (long)k.size(1), (long)k.size(2));
            plain(x, name);
            e[i] = static_cast<uint8_t *>(x.data_ptr());
            es[i] = x.storage();
            memory[2 + i] = memory_of(x, 0);
            version[2 + i] = version_of(x);
        }
        if (e[0] && e[0] == e[1]) refuse("k_exp and v_exp are the same memory");
        for (int i = 0; i < 4; ++i)
            for (int j = i + 1; j < 4; ++j)
                if (k.device() == v.device() && wt::overlap(memory[i], memory[j])) refuse("%s and %s share memory", PARTS[i], PARTS[j]);
        const int host = PyObject_IsTrue(args[4]);
        if (host < 0) return nullptr;
        if (!k.is_cuda() && !(host && k.is_cpu())) refuse("k must be on the GPU: the cache's kernels only run there");
        if (k.device() != v.device()) refuse("k and v live on different devices");
        at::Tensor error = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(k.device()));
        const auto stride = [](const at::Tensor &t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
        Cache *c = new Cache{{k.data_ptr(), v.data_ptr(), e[0], e[1], stride(k, 0), stride(k, 1), stride(k, 2), stride(v, 0), stride(v, 1), stride(v, 2),
                              (int32_t)k.size(0), (int32_t)k.size(1), (int32_t)k.size(2), (int32_t)k.size(3), dtype, 0, error.data_ptr<int32_t>()},
                             k.is_cuda() ? (int)k.get_device() : -1,
                             k.scalar_type(),
                             {k.storage(), v.storage(), es[0], es[1], error.storage()},
                             {},
                             {},
                             {memory[0], memory[1], memory[2], memory[3]},
                             {version[0], version[1], version[2], version[3]}};
        for (int i = 0; i < 5; ++i)
            if (c->kept[i]) c->start[i] = c->kept[i].data(), c->bytes[i] = c->kept[i].nbytes();
        PyObject *handle = PyCapsule_New(c, CACHE, [](PyObject *o) { delete static_cast<Cache *>(PyCapsule_GetPointer(o, CACHE)); });
        if (!handle) {
            delete c;
            return nullptr;
        }
        PyObject *both = PyTuple_New(2);
        if (!both) {
            Py_DECREF(handle);
            return nullptr;
        }
        PyTuple_SET_ITEM(both, 0, handle);
        PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(error));
        return both;
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// handle, k, v, table, positions, sequences
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        arguments(n, 6);
        const Cache *c = cache_of(args[0]);
        const Rows r = rows_of(args[3], args[4], args[5], c);
        const at::Tensor &k = tensor(args[1], c, "k", 3), &v = tensor(args[2], c, "v", 3);
        if (k.scalar_type() != v.scalar_type()) refuse("k and v differ: %s, %s", c10::toString(k.scalar_type()), c10::toString(v.scalar_type()));
        no_gradient(k, "k"), no_gradient(v, "v");
        const int dt = dtype_of(k.scalar_type(), c, "k, v");
        const Strided ks = strided(k, c, "k", r.n, c->desc.n_heads, true), vs = strided(v, c, "v", r.n, c->desc.n_heads, true);
        not_the_caches(memory_of(k, 2), c, "k"), not_the_caches(memory_of(v, 2), c, "v");
        if (r.n > 0) {
            const On on(c);
            check(g_append(&c->desc, ks.p, vs.p, dt, ks.row, ks.head, vs.row, vs.head, r.n, r.table.p, r.table.stride, r.table.n, r.table.width,
                           r.sequences, r.positions, on.stream),
                  "wt_kv_append");
            for (int i = 0; i < (c->desc.dtype == WT_DTYPE_E4M3 ? 4 : 2); ++i) written(c->version[i]);
        }
        Py_RETURN_NONE;
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// handle, table, positions, sequences, a tensor of the result's type or None, (k, v) to write or None -> (k, v)
PyObject *gather(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        arguments(n, 6);
        const Cache *c = cache_of(args[0]);
        const Rows r = rows_of(args[1], args[2], args[3], c);
        at::ScalarType type = c->desc.dtype == WT_DTYPE_E4M3 ? at::kFloat : c->type;
        if (!is_none(args[4])) {
            if (!THPDtype_Check(args[4])) refuse("dtype: a torch.dtype");
            type = reinterpret_cast<THPDtype *>(args[4])->scalar_type;
        }
        at::Tensor k, v;
        if (!is_none(args[5])) {
            if (!PyTuple_Check(args[5]) || PyTuple_GET_SIZE(args[5]) != 2) refuse("out: two tensors");
            k = tensor(PyTuple_GET_ITEM(args[5], 0), c, "out[0]", 3), v = tensor(PyTuple_GET_ITEM(args[5], 1), c, "out[1]", 3);
            if (k.scalar_type() != v.scalar_type() || (!is_none(args[4]) && k.scalar_type() != type))
                refuse("out: %s and %s", c10::toString(k.scalar_type()), c10::toString(v.scalar_type()));
            type = k.scalar_type();
            no_gradient(k, "out[0]"), no_gradient(v, "out[1]");
            strided(k, c, "out[0]", r.n, c->desc.n_heads, true), strided(v, c, "out[1]", r.n, c->desc.n_heads, true);
            if (!k.is_contiguous() || !v.is_contiguous()) refuse("out: not contiguous");
            not_the_caches(memory_of(k, 0), c, "out[0]"), not_the_caches(memory_of(v, 0), c, "out[1]");
            const char *kp = static_cast<const char *>(k.const_data_ptr()), *vp = static_cast<const char *>(v.const_data_ptr());
            if (r.n > 0 && kp < vp + v.nbytes() && vp < kp + k.nbytes()) refuse("out: the same memory twice");
        }
        const int dt = dtype_of(type, c, "dtype");
        if (!k.defined()) {
            if (c->device < 0) refuse("the cache's kernels only run on the GPU");
            const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)c->device);
            k = at::empty({r.n, c->desc.n_heads, c->desc.head_dim}, options);
            v = at::empty({r.n, c->desc.n_heads, c->desc.head_dim}, options);
        }
        if (r.n > 0) {
            const On on(c);
            check(g_gather(&c->desc, k.data_ptr(), v.data_ptr(), dt, r.n, r.table.p, r.table.stride, r.table.n, r.table.width, r.sequences,
                           r.positions, on.stream),
                  "wt_kv_gather");
            written(version_of(k)), written(version_of(v));
        }
        if (!is_none(args[5])) {
            Py_INCREF(args[5]);
            return args[5];
        }
        PyObject *kv = PyTuple_New(2);
        if (!kv) return nullptr;
        PyTuple_SET_ITEM(kv, 0, THPVariable_Wrap(k));
        PyTuple_SET_ITEM(kv, 1, THPVariable_Wrap(v));
        return kv;
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

at::Tensor new_workspace(const Cache *c, int n_seqs, int n_q_heads, int width) {   // undefined: none is needed
    int64_t bytes;
    {
        const On on(c);
        bytes = g_workspace(&c->desc, n_seqs, n_q_heads, width);
    }
    check(bytes, "wt_kv_attend_workspace");
    if (bytes == 0) return {};
    at::Tensor ws = at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (c10::DeviceIndex)c->device));
    ws.narrow(0, 0, WT_KV_WORKSPACE_ZEROED).zero_();
    return ws;
}

// handle, table, query heads -> tensor or None
PyObject *workspace(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        arguments(n, 3);
        const Cache *c = cache_of(args[0]);
        const Table t = table_of(args[1], c);
        const long heads = PyLong_AsLong(args[2]);
        if (heads == -1 && PyErr_Occurred()) return nullptr;
        if (heads < 1 || heads > INT32_MAX) refuse("%ld query heads", heads);
        at::Tensor ws = new_workspace(c, t.n, (int)heads, t.width);
        if (!ws.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(ws);
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// handle, q, table, lengths, scale or None, out or None, return_lse, workspace or None -> out, or (out, lse)
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        arguments(n, 8);
        const Cache *c = cache_of(args[0]);
        const Table t = table_of(args[2], c);
        const at::Tensor &q = tensor(args[1], c, "q", 3);
        const int64_t heads = q.size(1);
        if (heads < 1 || heads % c->desc.n_heads || heads > INT32_MAX) refuse("q: %ld query heads over %d key heads", (long)heads, c->desc.n_heads);
        no_gradient(q, "q");
        const int dt = dtype_of(q.scalar_type(), c, "q");
        const Strided qs = strided(q, c, "q", t.n, heads, false);
        const int32_t *lengths = int32s(args[3], c, "lengths", t.n);
        double scale = 1.0 / std::sqrt((double)c->desc.head_dim);
        if (!is_none(args[4])) {
            scale = PyFloat_AsDouble(args[4]);
            if (scale == -1.0 && PyErr_Occurred()) return nullptr;
        }
        const int lse_wanted = PyObject_IsTrue(args[6]);
        if (lse_wanted < 0) return nullptr;
        at::Tensor out, lse, ws;
        if (!is_none(args[5])) {
            out = tensor(args[5], c, "out", 3);
            no_gradient(out, "out");
            if (out.scalar_type() != q.scalar_type()) refuse("out: %s, not %s", c10::toString(out.scalar_type()), c10::toString(q.scalar_type()));
        }
        if (!is_none(args[7])) {
            ws = tensor(args[7], c, "workspace", 1);
            if (ws.scalar_type() != at::kByte || !ws.is_contiguous()) refuse("workspace: what attend_workspace() gave");
        }
        Strided os = {nullptr, heads * c->desc.head_dim, c->desc.head_dim};
        if (out.defined()) {
            os = strided(out, c, "out", t.n, heads, false);
            const int64_t d = c->desc.head_dim;
            const bool rows_outside = os.head >= d && os.row >= (heads - 1) * os.head + d, heads_outside = os.row >= d && os.head >= (t.n - 1) * os.row + d;
            if (t.n > 1 && heads > 1 ? !rows_outside && !heads_outside : (t.n > 1 && os.row < d) || (heads > 1 && os.head < d))
                refuse("out: two heads' values in one place (strides %ld, %ld)", (long)os.row, (long)os.head);
            const wt::Strided3 result = memory_of(out, 2), query = memory_of(q, 2);
            not_the_caches(result, c, "out");
            if (!(qs.p == os.p && qs.row == os.row && qs.head == os.head) && wt::overlap(result, query))   // (a row's query is read before its result is written)
                refuse("out: shares memory with q without being q");
        }
        if (c->device < 0) refuse("the cache's kernels only run on the GPU");
        if (!out.defined()) {
            out = at::empty({t.n, heads, c->desc.head_dim}, at::TensorOptions().dtype(q.scalar_type()).device(q.device()));
            os.p = out.data_ptr();
        }
        if (lse_wanted) lse = at::empty({t.n, heads}, at::TensorOptions().dtype(at::kFloat).device(q.device()));
        if (t.n > 0) {
            const auto go = [&]() {
                const On on(c);
                return g_attend(&c->desc, qs.p, dt, qs.row, qs.head, t.n, (int)heads, (float)scale, t.p, t.stride, t.width, lengths, os.p, os.row,
                                os.head, lse.defined() ? lse.data_ptr<float>() : nullptr, ws.defined() ? ws.data_ptr() : nullptr,
                                ws.defined() ? (int64_t)ws.nbytes() : 0, on.stream);
            };
            int rc = go();
            if (rc == WT_E_CAPTURE && !ws.defined()) {   // a captured call: in its graph's own memory, cleared in every replay
                ws = new_workspace(c, t.n, (int)heads, t.width);
                rc = go();
            }
            check(rc, "wt_kv_attend");
            written(version_of(out));
        }
        PyObject *o;
        if (is_none(args[5])) o = THPVariable_Wrap(out);
        else {
            o = args[5];
            Py_INCREF(o);
        }
        if (!o || !lse_wanted) return o;
        PyObject *both = PyTuple_New(2);
        if (!both) {
            Py_DECREF(o);
            return nullptr;
        }
        PyTuple_SET_ITEM(both, 0, o);
        PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(lse));
        return both;
    } catch (const Refused &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

#define WT_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL
PyMethodDef METHODS[] = {{"setup", setup, METH_VARARGS, nullptr},           {"make", WT_FAST(make), nullptr},
                         {"append", WT_FAST(append), nullptr},              {"gather", WT_FAST(gather), nullptr},
                         {"attend", WT_FAST(attend), nullptr},              {"workspace", WT_FAST(workspace), nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_kvcalls", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__kvcalls(void) { return PyModule_Create(&MODULE); }
