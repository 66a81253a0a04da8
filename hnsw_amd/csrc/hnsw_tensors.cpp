// The token cache's calls on torch tensors (module hnsw_amd._tensors, used by hnsw_amd/cache.py): checks of types, shapes and devices,
// outputs, workspaces and the current stream, then the C entry points of include/hnsw_amd.h.  In Python these cost several times
// what a launch does, and the calls of a decoding step are a launch each.  The entry points come as addresses from the library
// that the process has loaded, which this module is not linked with.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <cmath>
#include <exception>
#include <string>

#include "../../include/hnsw_amd.h"

namespace {

decltype(&hnsw_amd_cache_plan_device) g_plan = nullptr;
decltype(&hnsw_amd_cache_append_device) g_append = nullptr;
decltype(&hnsw_amd_cache_read_device) g_read = nullptr;
decltype(&hnsw_amd_cache_attend_workspace) g_attend_workspace = nullptr;
decltype(&hnsw_amd_cache_attend_found_workspace) g_found_workspace = nullptr;
decltype(&hnsw_amd_cache_attend_device) g_attend = nullptr;
decltype(&hnsw_amd_cache_attend_found_device) g_found = nullptr;
PyObject* g_check = nullptr;                // capi.check: raises for a status that is not 0

struct Raised {};                           // a Python error is set

[[noreturn]] void refuse(const std::string& what)
{
    PyErr_SetString(PyExc_ValueError, what.c_str());
    throw Raised{};
}

template <class F> PyObject* guarded(F&& f)
{
    try {
        return f();
    } catch (const Raised&) {
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());         // (torch's own error types: out of memory is torch.OutOfMemoryError)
    }
    return nullptr;
}

void check(int rc)
{
    if (rc == HNSW_AMD_OK) return;
    PyObject* r = PyObject_CallFunction(g_check, "i", rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "hnsw_amd: a call failed");
    throw Raised{};
}

void count_args(Py_ssize_t have, Py_ssize_t want)
{
    if (have == want) return;
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    throw Raised{};
}

const at::Tensor& tensor(PyObject* o, const char* name)
{
    if (!THPVariable_Check(o)) {
        PyErr_SetString(PyExc_TypeError, (std::string(name) + " must be a tensor").c_str());
        throw Raised{};
    }
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, int64_t least, int64_t most, const char* name)
{
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw Raised{};
    if (x < least || x > most) refuse(std::string(name) + " is out of range");
    return x;
}

// A contiguous tensor of this type and shape (-1: any extent) on `device`.
void need(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, const at::Device& device)
{
    if (t.scalar_type() == type && t.device() == device && t.dim() == (int64_t)shape.size() && t.is_contiguous() && t.layout() == at::kStrided) {
        bool fits = true;
        for (size_t i = 0; i < shape.size(); i++) fits &= shape[i] < 0 || t.size(i) == shape[i];
        if (fits) return;
    }
    std::string want = "[";
    for (size_t i = 0; i < shape.size(); i++) want += (i ? ", " : "") + (shape[i] < 0 ? std::string("any") : std::to_string(shape[i]));
    refuse(std::string(name) + " must be a contiguous " + at::toString(type) + " tensor of shape " + want + "] on " + device.str());
}

uint32_t row_type(const at::Tensor& t, const char* name)
{
    switch (t.scalar_type()) {
    case at::kFloat: return HNSW_AMD_TYPE_F32;
    case at::kHalf: return HNSW_AMD_TYPE_F16;
    case at::kBFloat16: return HNSW_AMD_TYPE_BF16;
    default: refuse(std::string(name) + " must be float32, float16 or bfloat16");
    }
}

void* stream_of(const at::Device& device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream(); }

struct Cache {
    hnsw_amd_token_cache c;
    at::Tensor k, v, ks, vs;                // (kept alive)
    at::Device device;
};

const char* const kCapsule = "hnsw_amd.token_cache";

// Nothing here has a gradient, and none is lost without a word.
void no_gradient(const at::Tensor& t, const char* name)
{
    if (t.requires_grad() && at::GradMode::is_enabled()) refuse(std::string(name) + " requires a gradient: the token cache has none");
}

void no_gradient(const Cache& c)
{
    no_gradient(c.k, "k_codes");
    no_gradient(c.v, "v_codes");
    no_gradient(c.ks, "k_scale");
    no_gradient(c.vs, "v_scale");
}

const Cache& cache(PyObject* o)
{
    void* p = PyCapsule_GetPointer(o, kCapsule);
    if (!p) throw Raised{};
    const Cache& c = *static_cast<const Cache*>(p);
    no_gradient(c);
    return c;
}

// Rows [rows, heads, dim] of one of the three types, the last dimension contiguous.
uint32_t rows_of(const Cache& c, const at::Tensor& t, const char* name, int64_t heads)
{
    if (t.device() != c.device || t.layout() != at::kStrided || t.dim() != 3 || t.size(1) != heads || t.size(2) != c.c.dim)
        refuse(std::string(name) + " must be a [rows, " + std::to_string(heads) + ", " + std::to_string(c.c.dim) + "] tensor on " + c.device.str());
    if (t.stride(2) != 1) refuse(std::string(name) + ": the last dimension must be contiguous");
    if (t.size(0) >= INT64_C(1) << 31) refuse(std::string(name) + " has too many rows");
    no_gradient(t, name);
    return row_type(t, name);
}

PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        count_args(n, 8);
        void* p[7];
        for (int i = 0; i < 7; i++) {
            p[i] = PyLong_AsVoidPtr(args[i]);
            if (PyErr_Occurred()) throw Raised{};
        }
        g_plan = reinterpret_cast<decltype(g_plan)>(p[0]);
        g_append = reinterpret_cast<decltype(g_append)>(p[1]);
        g_read = reinterpret_cast<decltype(g_read)>(p[2]);
        g_attend_workspace = reinterpret_cast<decltype(g_attend_workspace)>(p[3]);
        g_found_workspace = reinterpret_cast<decltype(g_found_workspace)>(p[4]);
        g_attend = reinterpret_cast<decltype(g_attend)>(p[5]);
        g_found = reinterpret_cast<decltype(g_found)>(p[6]);
        Py_INCREF(args[7]);
        Py_XDECREF(g_check);
        g_check = args[7];
        Py_RETURN_NONE;
    });
}

PyObject* py_cache(PyObject*, PyObject* const* args, Py_ssize_t n)
{
    return guarded([&]() -> PyObject* {
        count_args(n, 4);
        const at::Tensor &k = tensor(args[0], "k_codes"), &v = tensor(args[1], "v_codes"), &ks = tensor(args[2], "k_scale"), &vs = tensor(args[3], "v_scale");
        const at::Device device = k.device();
        if (!device.is_cuda()) refuse("TokenCache: the buffers must be on a GPU");
        if (k.scalar_type() != at::kChar && k.scalar_type() != at::kFloat8_e4m3fn) refuse("TokenCache: codes must be int8 or float8_e4m3fn");
        need(k, "k_codes", k.scalar_type(), {-1, -1, -1, -1}, device);
        need(v, "v_codes", k.scalar_type(), k.sizes(), device);
        need(ks, "k_scale", at::kFloat, {k.size(0), k.size(1)}, device);
        need(vs, "v_scale", at::kFloat, {k.size(0), k.size(1)}, device);
        no_gradient(k, "k_codes");
        no_gradient(v, "v_codes");
        no_gradient(ks, "k_scale");
        no_gradient(vs, "v_scale");
        for (int i = 0; i < 4; i++)
            if (k.size(i) > 0xffffffffll) refuse("TokenCache: an extent is out of range");
        Cache* c = new Cache{{k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), (uint32_t)k.size(0), (uint32_t)k.size(1), (uint32_t)k.size(2),
                              (uint32_t)k.size(3), (uint32_t)(k.scalar_type() == at::kChar ? HNSW_AMD_CODES_I8 : HNSW_AMD_CODES_E4M3)}, k, v, ks, vs, device};
        PyObject* o = PyCapsule_New(c, kCapsule, [](PyObject* self) { delete static_cast<Cache*>(PyCapsule_GetPointer(self, kCapsule)); });
        if (!o) delete c;
        return o;
    });
}

PyObject* tuple_of(std::initializer_list<at::Tensor> ts)
{
    PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
    if (!t) throw Raised{};
    Py_ssize_t i = 0;
    for (const at::Tensor& x : ts) {
        PyObject* o = THPVariable_Wrap(x);
        if (!o) { Py_DECREF(t); throw Raised{}; }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

// Tensors that lie one behind the other in one allocation of `longs` 64-bit words (an allocation costs several times what a tensor does).
class Pieces {
public:
    Pieces(const at::TensorOptions& options, int64_t longs) : all_(at::empty({longs}, options.dtype(at::kLong))) {}
    at::Tensor next(at::ScalarType type, int64_t n)
    {
        const int64_t size = (int64_t)c10::elementSize(type);
        at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all_.storage()), all_.key_set(), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
        t.unsafeGetTensorImpl()->set_storage_offset(at_ / size);
        at_ += n * size;
        return t;
    }

private:
    at::Tensor all_;
    int64_t at_ = 0;                        // bytes (the longer types come first)
};

PyObject* py_plan(PyObject*, PyObject* const* args, Py_ssize_t n_args)
{
    return guarded([&]() -> PyObject* {
        count_args(n_args, 7);
        const at::Tensor &lens = tensor(args[0], "lens"), &grow = tensor(args[1], "grow"), &table = tensor(args[2], "table"), &ring = tensor(args[3], "ring"),
                         &state = tensor(args[4], "state");
        const int64_t block = integer(args[5], 0, 0xffffffffll, "block_tokens"), n_slots = integer(args[6], 0, 0x7fffffffll, "n_slots");
        const at::Device device = lens.device();
        if (!device.is_cuda()) refuse("cache_plan: the tensors must be on a GPU");
        need(lens, "lens", at::kInt, {-1}, device);
        const int64_t n = lens.size(0);
        need(grow, "grow", at::kInt, {n}, device);
        need(table, "table", at::kInt, {n, -1}, device);
        need(ring, "ring", at::kInt, {-1}, device);
        need(state, "state", at::kLong, {2}, device);
        if (n > 0xffffffffll || table.size(1) > 0xffffffffll || ring.size(0) > 0xffffffffll) refuse("cache_plan: an extent is out of range");
        // one allocation for the five results
        Pieces pieces(state.options(), n_slots + 2 + (n + 1 + n + 1 + 1) / 2);
        const at::Tensor slots = pieces.next(at::kLong, n_slots), state_out = pieces.next(at::kLong, 2), cu = pieces.next(at::kInt, n + 1),
                         lens_out = pieces.next(at::kInt, n), status = pieces.next(at::kInt, 1);
        check(g_plan(lens.data_ptr<int32_t>(), grow.data_ptr<int32_t>(), (uint32_t)n, table.data_ptr<int32_t>(), (uint32_t)table.size(1), ring.data_ptr<int32_t>(),
                     (uint32_t)ring.size(0), state.data_ptr<int64_t>(), (uint32_t)block, (uint32_t)n_slots, slots.data_ptr<int64_t>(), cu.data_ptr<int32_t>(),
                     lens_out.data_ptr<int32_t>(), state_out.data_ptr<int64_t>(), status.data_ptr<int32_t>(), device.index(), stream_of(device)));
        return tuple_of({slots, cu, lens_out, state_out, status});
    });
}

PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n_args)
{
    return guarded([&]() -> PyObject* {
        count_args(n_args, 4);
        const Cache& c = cache(args[0]);
        const at::Tensor &k = tensor(args[1], "k"), &v = tensor(args[2], "v"), &slots = tensor(args[3], "slots");
        const uint32_t type = rows_of(c, k, "k", c.c.n_heads);
        rows_of(c, v, "v", c.c.n_heads);
        if (v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type()) refuse("append: k and v must have the same shape and type");
        need(slots, "slots", at::kLong, {k.size(0)}, c.device);
        check(g_append(&c.c, k.data_ptr(), v.data_ptr(), (uint32_t)k.size(0), type, k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr<int64_t>(),
                       c.device.index(), stream_of(c.device)));
        Py_RETURN_NONE;
    });
}

// read(cache, slots, dtype of the outputs or None)
PyObject* py_read(PyObject*, PyObject* const* args, Py_ssize_t n_args)
{
    return guarded([&]() -> PyObject* {
        count_args(n_args, 3);
        const Cache& c = cache(args[0]);
        const at::Tensor& slots = tensor(args[1], "slots");
        if (args[2] != Py_None && !THPDtype_Check(args[2])) refuse("read: float32, float16 or bfloat16");
        const at::ScalarType dtype = args[2] == Py_None ? at::kFloat : reinterpret_cast<THPDtype*>(args[2])->scalar_type;
        if (dtype != at::kFloat && dtype != at::kHalf && dtype != at::kBFloat16) refuse("read: float32, float16 or bfloat16");
        const uint32_t type = dtype == at::kFloat ? HNSW_AMD_TYPE_F32 : dtype == at::kHalf ? HNSW_AMD_TYPE_F16 : HNSW_AMD_TYPE_BF16;
        need(slots, "slots", at::kLong, {-1}, c.device);
        if (slots.size(0) >= INT64_C(1) << 31) refuse("read: too many slots");
        const auto options = slots.options().dtype(dtype);
        at::Tensor k = at::empty({slots.size(0), c.c.n_heads, c.c.dim}, options), v = at::empty({slots.size(0), c.c.n_heads, c.c.dim}, options);
        check(g_read(&c.c, slots.data_ptr<int64_t>(), (uint32_t)slots.size(0), type, k.data_ptr(), v.data_ptr(), c.device.index(), stream_of(c.device)));
        return tuple_of({k, v});
    });
}

// attend(cache, q, table, lens, cu_q, causal, scale, max_len, ids): ids None: over all tokens
PyObject* py_attend(PyObject*, PyObject* const* args, Py_ssize_t n_args)
{
    return guarded([&]() -> PyObject* {
        count_args(n_args, 9);
        const Cache& c = cache(args[0]);
        const at::Tensor &q = tensor(args[1], "q"), &table = tensor(args[2], "table"), &lens = tensor(args[3], "lens");
        if (q.dim() != 3 || q.size(1) % c.c.n_heads || q.size(1) > 0xffffffffll) refuse("q must be [rows, heads, dim], its heads a multiple of the cache's");
        const uint32_t type = rows_of(c, q, "q", q.size(1));
        need(lens, "lens", at::kInt, {-1}, c.device);
        const int64_t n = lens.size(0), rows = q.size(0), heads = q.size(1);
        need(table, "table", at::kInt, {n, -1}, c.device);
        if (n > 0xffffffffll || table.size(1) > 0xffffffffll) refuse("lens or table: an extent is out of range");
        const int32_t* cu = nullptr;
        if (args[4] != Py_None) {
            const at::Tensor& t = tensor(args[4], "cu_q");
            need(t, "cu_q", at::kInt, {n + 1}, c.device);
            cu = t.data_ptr<int32_t>();
        }
        const int causal = PyObject_IsTrue(args[5]);
        double scale = 1.0 / std::sqrt((double)c.c.dim);
        if (args[6] != Py_None) scale = PyFloat_AsDouble(args[6]);
        if (causal < 0 || (scale == -1.0 && PyErr_Occurred())) throw Raised{};
        const uint32_t max_len = (uint32_t)integer(args[7], 0, 0xffffffffll, "max_len");
        const bool found = args[8] != Py_None;
        uint32_t lists = 0, n_ids = 0;
        const void* ids = nullptr;
        if (found) {
            const at::Tensor& t = tensor(args[8], "ids");
            need(t, "ids", at::kInt, {rows, -1, -1}, c.device);
            if (t.size(1) > 0xffffffffll || t.size(2) > 0x7fffffffll) refuse("ids: an extent is out of range");
            lists = (uint32_t)t.size(1);
            n_ids = (uint32_t)t.size(2);
            ids = t.data_ptr();
        }
        at::Tensor out = at::empty(q.sizes(), q.options()), lse = at::empty({rows, heads}, q.options().dtype(at::kFloat)), work;
        const uint64_t bytes = found ? g_found_workspace(&c.c, (uint32_t)rows, (uint32_t)heads, lists, n_ids)
                                     : g_attend_workspace(&c.c, (uint32_t)rows, (uint32_t)heads, (uint32_t)n, (uint32_t)table.size(1), max_len);
        void* at = nullptr;
        if (bytes) {
            work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
            at = work.data_ptr();
        }
        if (found)
            check(g_found(&c.c, q.data_ptr(), (uint32_t)rows, (uint32_t)heads, q.stride(0), q.stride(1), type, table.data_ptr<int32_t>(), (uint32_t)table.size(1),
                          lens.data_ptr<int32_t>(), (uint32_t)n, cu, causal, static_cast<const uint32_t*>(ids), lists, n_ids, (float)scale, out.data_ptr(),
                          lse.data_ptr<float>(), at, bytes, c.device.index(), stream_of(c.device)));
        else
            check(g_attend(&c.c, q.data_ptr(), (uint32_t)rows, (uint32_t)heads, q.stride(0), q.stride(1), type, table.data_ptr<int32_t>(), (uint32_t)table.size(1),
                           lens.data_ptr<int32_t>(), (uint32_t)n, cu, causal, (float)scale, max_len, out.data_ptr(), lse.data_ptr<float>(), at, bytes,
                           c.device.index(), stream_of(c.device)));
        return tuple_of({out, lse});
    });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {METHOD(bind), METHOD(cache), METHOD(plan), METHOD(append), METHOD(read), METHOD(attend), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&kModule); }
