// Python binding of the decode step's entry points (page plan, paged store, paged attention,
// sampling).  These calls take one to ten microseconds on the device, so checking their tensors
// and marshalling their arguments in Python (11 to 19 us a call) is what a step would wait for;
// here a call costs about as much as its launch.  The checks are the ones a caller gets from the
// other modules: ValueError for what the operators do not take, before anything is launched.
//
// The C entry points are not linked: escha_mlx_b200._lib passes their addresses to init(), so
// that another build of the library can stand in for them.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/escha_b200.h"

namespace {

// the entry points, by the types that the header declares
decltype(&escha_last_error) g_last_error;
decltype(&escha_page_plan) g_page_plan;
decltype(&escha_paged_append) g_append;
decltype(&escha_paged_attend_workspace_bytes) g_workspace;
decltype(&escha_paged_attend) g_attend;
decltype(&escha_sample) g_sample;

// What becomes a ValueError.
struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};

[[noreturn]] void refuse(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    throw Refused(buf);
}

void check(int rc) {
    if (rc == ESCHA_OK) return;
    if (rc == ESCHA_EINVAL) throw Refused(g_last_error());
    throw std::runtime_error(g_last_error());
}

std::string text(at::IntArrayRef sizes) {
    std::string s = "[";
    for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
    return s + "]";
}
const char* text(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return "torch.float16";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kFloat: return "torch.float32";
        case at::kDouble: return "torch.float64";
        case at::kInt: return "torch.int32";
        case at::kLong: return "torch.int64";
        case at::kChar: return "torch.int8";
        default: return c10::toString(t);
    }
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse("%s must be a CUDA tensor (there is no CPU path in this package)", name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse("%s must be a CUDA tensor (there is no CPU path in this package)", name);
    return t;
}

void same_device(const at::Tensor& t, const char* name, int index) {
    if (t.get_device() != index)
        refuse("%s is on cuda:%d, the other tensors on cuda:%d", name, static_cast<int>(t.get_device()), index);
}

// A dense int32 tensor of that shape on that device (extent -1: any); its address.
template <size_t N>
int32_t* ints(PyObject* o, const char* name, int index, const int64_t (&shape)[N]) {
    const at::Tensor& t = tensor(o, name);
    same_device(t, name, index);
    if (t.scalar_type() != at::kInt) refuse("%s must be torch.int32, got %s", name, text(t.scalar_type()));
    bool fits = t.dim() == static_cast<int64_t>(N);
    for (size_t i = 0; fits && i < N; ++i) fits = shape[i] < 0 || shape[i] == t.size(i);
    if (!fits) {
        std::string want = "[";
        for (size_t i = 0; i < N; ++i)
            want += (i ? ", " : "") + (shape[i] < 0 ? std::string("*") : std::to_string(shape[i]));
        refuse("%s must have shape %s], got %s", name, want.c_str(), text(t.sizes()).c_str());
    }
    if (!t.is_contiguous()) refuse("%s must be contiguous", name);
    return static_cast<int32_t*>(t.data_ptr());
}

long whole(PyObject* o, const char* name, long least, long most) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) {
        if (PyErr_ExceptionMatches(PyExc_OverflowError)) {
            PyErr_Clear();
            refuse("%s must be in [%ld, %ld]", name, least, most);
        }
        throw std::exception();       // the Python error stands
    }
    if (v < least || v > most) refuse("%s must be in [%ld, %ld], got %ld", name, least, most, v);
    return v;
}

// [rows, heads, channels] as the kernels can read it: dense channels, other strides multiples of
// 8 elements, 16-byte aligned; a dense copy where it is not so.
struct Rows {
    at::Tensor t;
    long row, head;
};
Rows rows_of(PyObject* o, const char* name, int64_t n, int64_t heads, int64_t channels, int index) {
    at::Tensor x = tensor(o, name);
    same_device(x, name, index);
    if (x.dim() != 3 || (n >= 0 && x.size(0) != n) || (heads >= 0 && x.size(1) != heads) || x.size(2) != channels)
        refuse("%s must have shape [%s, %s, %ld], got %s", name, n < 0 ? "*" : std::to_string(n).c_str(),
               heads < 0 ? "*" : std::to_string(heads).c_str(), static_cast<long>(channels),
               text(x.sizes()).c_str());
    if (x.stride(2) != 1 || ((x.stride(0) | x.stride(1)) & 7) != 0 ||
        (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) != 0)
        x = x.clone(at::MemoryFormat::Contiguous);
    return {x, static_cast<long>(x.stride(0)), static_cast<long>(x.stride(1))};
}

constexpr int kF16 = ESCHA_F16, kBF16 = ESCHA_BF16, kF32 = ESCHA_F32, kI8 = ESCHA_I8;
int type_of(at::ScalarType t) {
    return t == at::kHalf ? kF16 : t == at::kBFloat16 ? kBF16 : t == at::kFloat ? kF32 : t == at::kChar ? kI8 : -1;
}

// The tensors of a cache, checked when it was made.
struct Cache {
    const at::Tensor &k, &v;
    float *k_scale = nullptr, *v_scale = nullptr;
    int index, type, pages, heads, page_size, channels;
    explicit Cache(PyObject* const* a) : k(tensor(a[0], "k")), v(tensor(a[1], "v")) {
        if (a[2] != Py_None) {
            k_scale = static_cast<float*>(tensor(a[2], "k_scale").data_ptr());
            v_scale = static_cast<float*>(tensor(a[3], "v_scale").data_ptr());
        }
        index = k.get_device();
        type = type_of(k.scalar_type());
        pages = static_cast<int>(k.size(0));
        heads = static_cast<int>(k.size(1));
        page_size = static_cast<int>(k.size(2));
        channels = static_cast<int>(k.size(3));
    }
    int row_type(const at::Tensor& x, const char* name) const {
        const int t = type_of(x.scalar_type());
        if (type == kI8 ? (t != kF16 && t != kBF16) : t != type)
            refuse("%s must be %s for a %s cache, got %s", name,
                   type == kI8 ? "torch.float16 or torch.bfloat16" : text(k.scalar_type()),
                   text(k.scalar_type()), text(x.scalar_type()));
        return t;
    }
};

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int index) {
    return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index)),
                                  std::nullopt);
}

void* stream_of(int index) {
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream();
}

// n elements of a dense one-dimensional tensor, as a tensor over the same storage
PyObject* part(const at::Tensor& whole, int64_t at, int64_t n) {
    at::Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(),
                                                           whole.dtype());
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    t.unsafeGetTensorImpl()->set_storage_offset(at);
    return THPVariable_Wrap(t);
}

template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* kind = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (kind) PyErr_SetString(kind, e.what_without_backtrace());
        Py_XDECREF(kind);
        Py_XDECREF(torch);
    } catch (const c10::Error& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception& e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

void count(Py_ssize_t got, Py_ssize_t want, const char* name) {
    if (got != want) refuse("%s takes %zd arguments, got %zd", name, want, got);
}

// plan(table, lengths, added, free_pages, head, page_size, n_pages, rows) -> six tensors
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 8, "plan");
        const at::Tensor& table = tensor(a[0], "table");
        const int index = table.get_device();
        int32_t* tab = ints(a[0], "table", index, {-1, -1});
        const int64_t b = table.size(0), w = table.size(1);
        int32_t* lengths = ints(a[1], "lengths", index, {b});
        int32_t* added = ints(a[2], "added", index, {b});
        int32_t* free_pages = ints(a[3], "free_pages", index, {-1});
        const int64_t f = THPVariable_Unpack(a[3]).size(0);
        int32_t* head = ints(a[4], "head", index, {1});
        const long page_size = whole(a[5], "page_size", 1, 1 << 20);
        const long n_pages = whole(a[6], "n_pages", 1, 0x7fffffff);
        const long rows = whole(a[7], "rows", 0, 1 << 30);
        if (b < 1 || b > 4096) refuse("plan_pages takes 1..4096 requests, got %ld", static_cast<long>(b));
        if (w > 0x7fffffff || f > 0x7fffffff) refuse("table or free_pages is too long");
        c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
        const at::Tensor buf = empty({2 * rows + 2 * b + 3}, at::kInt, index);
        int32_t* p = buf.data_ptr<int32_t>();
        int32_t *starts = p + 2 * rows, *ends = starts + b + 1;
        check(g_page_plan(tab, lengths, added, free_pages, static_cast<int>(f), head, static_cast<int>(b),
                          static_cast<int>(w), static_cast<int>(page_size), static_cast<int>(n_pages),
                          static_cast<int>(rows), p, p + rows, starts, ends, ends + b, ends + b + 1,
                          stream_of(index)));
        const int64_t at[6] = {0, rows, 2 * rows, 2 * rows + b + 1, 2 * rows + 2 * b + 1, 2 * rows + 2 * b + 2};
        const int64_t size[6] = {rows, rows, b + 1, b, 1, 1};
        PyObject* out = PyTuple_New(6);
        if (out == nullptr) throw std::exception();
        for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(out, i, part(buf, at[i], size[i]));
        return out;
    });
}

// append(k_cache, v_cache, k_scale, v_scale, k, v, slots)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 7, "append");
        const Cache c(a);
        const Rows k = rows_of(a[4], "k", -1, c.heads, c.channels, c.index);
        const int64_t t = k.t.size(0);
        const Rows v = rows_of(a[5], "v", t, c.heads, c.channels, c.index);
        if (k.t.scalar_type() != v.t.scalar_type())
            refuse("k is %s, v is %s", text(k.t.scalar_type()), text(v.t.scalar_type()));
        const int type = c.row_type(k.t, "k");
        int32_t* slots = ints(a[6], "slots", c.index, {t});
        if (t > 0x7fffffff) refuse("append takes 2^31 - 1 rows at most");
        if (t > 0) {
            c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.index));
            check(g_append(k.t.data_ptr(), k.row, k.head, v.t.data_ptr(), v.row, v.head, type, slots,
                           static_cast<int>(t), c.heads, c.channels, c.page_size, c.pages, c.k.data_ptr(),
                           c.v.data_ptr(), c.type, c.k_scale, c.v_scale, stream_of(c.index)));
        }
        Py_RETURN_NONE;
    });
}

// attend(k_cache, v_cache, k_scale, v_scale, q, table, lengths, scale) -> [B, heads, channels]
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 8, "attend");
        const Cache c(a);
        const Rows q = rows_of(a[4], "q", -1, -1, c.channels, c.index);
        const int type = c.row_type(q.t, "q");
        const int64_t b = q.t.size(0), heads = q.t.size(1);
        if (heads < 1 || heads % c.heads != 0)
            refuse("%ld query heads do not share %d key/value heads evenly", static_cast<long>(heads), c.heads);
        int32_t* table = ints(a[5], "table", c.index, {b, -1});
        int32_t* lengths = ints(a[6], "lengths", c.index, {b});
        const int64_t w = THPVariable_Unpack(a[5]).size(1), group = heads / c.heads;
        if (w < 1) refuse("table needs at least one page per request");
        if (b > 1 << 20 || w > 0x7fffffff || group > 0x7fffffff) refuse("attend takes 2^20 requests at most");
        const double scale = PyFloat_AsDouble(a[7]);
        if (scale == -1.0 && PyErr_Occurred()) throw std::exception();
        c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.index));
        const at::Tensor out = empty({b, heads, c.channels}, q.t.scalar_type(), c.index);
        if (b > 0) {
            const size_t need = g_workspace(static_cast<int>(b), c.heads, static_cast<int>(group), c.channels,
                                            static_cast<int>(w), c.page_size);
            at::Tensor work;
            if (need) work = empty({static_cast<int64_t>(need)}, at::kByte, c.index);
            check(g_attend(q.t.data_ptr(), q.row, q.head, type, c.k.data_ptr(), c.v.data_ptr(), c.type,
                           c.k_scale, c.v_scale, table, lengths, static_cast<int>(b), c.heads,
                           static_cast<int>(group), c.channels, static_cast<int>(w), c.page_size, c.pages,
                           static_cast<float>(scale), need ? work.data_ptr() : nullptr, need, out.data_ptr(),
                           stream_of(c.index)));
        }
        return THPVariable_Wrap(out);
    });
}

// A setting of sampling: a number, or a dense tensor with one value per row.
template <class T>
struct Setting {
    T* each = nullptr;
    T one = T(0);
    Setting(PyObject* o, const char* name, int64_t rows, at::ScalarType type, int index) {
        if (THPVariable_Check(o)) {
            const at::Tensor& t = THPVariable_Unpack(o);
            if (t.scalar_type() != type || t.numel() != rows || !t.is_contiguous() || !t.is_cuda())
                refuse("%s must be a number or a contiguous %s CUDA tensor of %ld values, got %s %s", name,
                       text(type), static_cast<long>(rows), text(t.scalar_type()), text(t.sizes()).c_str());
            same_device(t, name, index);
            each = static_cast<T*>(t.data_ptr());
            return;
        }
        if constexpr (std::is_same<T, int>::value) {
            // any number past the vocabulary says the same
            int overflow = 0;
            const long v = PyLong_AsLongAndOverflow(o, &overflow);
            if (v == -1 && PyErr_Occurred()) throw std::exception();
            one = overflow > 0 || v > 0x7fffffff ? 0x7fffffff : overflow < 0 || v < 0 ? 0 : static_cast<int>(v);
        } else {
            const double v = PyFloat_AsDouble(o);
            if (v == -1.0 && PyErr_Occurred()) throw std::exception();
            one = static_cast<T>(v);
        }
    }
};

// sample(logits, uniforms, temperature, top_k, top_p, min_p) -> tokens
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 6, "sample");
        at::Tensor x = tensor(a[0], "logits");
        const int type = type_of(x.scalar_type());
        if (type != kF16 && type != kBF16 && type != kF32)
            refuse("logits must be torch.float16, torch.bfloat16 or torch.float32, got %s", text(x.scalar_type()));
        if (x.dim() < 1 || x.size(-1) < 1)
            refuse("logits must have shape [..., V], got %s", text(x.sizes()).c_str());
        const int index = x.get_device();
        const at::Tensor& u = tensor(a[1], "uniforms");
        const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
        if (u.scalar_type() != at::kFloat || u.sizes() != lead || !u.is_contiguous())
            refuse("uniforms must be a contiguous torch.float32 tensor of shape %s", text(lead).c_str());
        same_device(u, "uniforms", index);
        const int64_t b = u.numel(), v = x.size(-1);
        if (v > 0x7fffffff || b > 0x7fffffff) refuse("%ld rows of V=%ld logits are too many", b, v);
        const Setting<float> t(a[2], "temperature", b, at::kFloat, index);
        const Setting<int> k(a[3], "top_k", b, at::kInt, index);
        const Setting<float> p(a[4], "top_p", b, at::kFloat, index);
        const Setting<float> m(a[5], "min_p", b, at::kFloat, index);
        c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
        const at::Tensor tokens = empty(lead, at::kLong, index);
        if (b > 0) {
            if (x.dim() != 2) x = x.reshape({b, v});
            if (x.stride(1) != 1 && v > 1) x = x.contiguous();
            check(g_sample(x.data_ptr(), type, x.stride(0), static_cast<int>(b), static_cast<int>(v),
                           u.data_ptr<float>(),
                           t.each, t.one, k.each, k.one, p.each, p.one, m.each, m.one,
                           tokens.data_ptr<int64_t>(),
                           stream_of(index)));
        }
        return THPVariable_Wrap(tokens);
    });
}

// init(address, ...): of escha_last_error and the entry points, in the order below
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        count(n, 6, "init");
        void* at[6];
        for (int i = 0; i < 6; ++i) {
            at[i] = PyLong_AsVoidPtr(a[i]);
            if (at[i] == nullptr) throw std::runtime_error("init takes addresses");
        }
        g_last_error = reinterpret_cast<decltype(g_last_error)>(at[0]);
        g_page_plan = reinterpret_cast<decltype(g_page_plan)>(at[1]);
        g_append = reinterpret_cast<decltype(g_append)>(at[2]);
        g_workspace = reinterpret_cast<decltype(g_workspace)>(at[3]);
        g_attend = reinterpret_cast<decltype(g_attend)>(at[4]);
        g_sample = reinterpret_cast<decltype(g_sample)>(at[5]);
        Py_RETURN_NONE;
    });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init), METHOD(plan), METHOD(append), METHOD(attend), METHOD(sample),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode() { return PyModule_Create(&module); }
