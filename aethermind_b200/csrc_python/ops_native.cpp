// Native binding of the operators that a decode loop calls for single tokens:
// amcu_sample, amcu_kv4_append, amcu_kv4_gather and amcu_attn_kv4 with torch
// tensors. Their kernels run for 5 to 15 us in small calls; reading a dozen
// tensors' types, shapes and strides from Python and filling the argument
// structs through ctypes takes 20 to 40 us, here it takes about 2.
//
// Each function checks its tensors (ValueError), allocates outputs and
// workspace with torch, launches on the current stream, and returns the outputs
// or, where the C ABI refused the call, its status code for ops.py to raise.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "aethermind_b200.h"

namespace {

// The C ABI, from the library that _lib.py loaded (bind()).
decltype(&amcu_sample) f_sample;
decltype(&amcu_kv4_append) f_append;
decltype(&amcu_kv4_gather) f_gather;
decltype(&amcu_attn_kv4_workspace_bytes) f_attn_workspace;
decltype(&amcu_attn_kv4) f_attn;

struct BadArgument : std::runtime_error {
    using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const std::string& what) { throw BadArgument(what); }

// A CUDA tensor of the current device; the launch goes to its current stream.
const at::Tensor& tensor(PyObject* o, c10::DeviceIndex here, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + ": expected a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != here)
        refuse(std::string(name) + ": aethermind_b200 ops take CUDA tensors of the current device");
    return t;
}
const at::Tensor* optional(PyObject* o, c10::DeviceIndex here, const char* name) {
    return o == Py_None ? nullptr : &tensor(o, here, name);
}
int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
int32_t act_dtype(const at::Tensor& t, const char* name) {
    if (t.scalar_type() == at::kBFloat16) return AMCU_BF16;
    if (t.scalar_type() == at::kFloat) return AMCU_F32;
    refuse(std::string(name) + ": float32 or bfloat16");
}
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

at::Tensor make(at::IntArrayRef size, at::ScalarType type, c10::DeviceIndex here) {
    return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, here));
}

// Rows of `width` contiguous elements.
void rows_of(const at::Tensor& t, int64_t rows, int64_t width, at::ScalarType type, const char* name, bool written) {
    if (t.dim() != 2 || t.size(1) != width || (t.stride(1) != 1 && width > 1) || t.scalar_type() != type)
        refuse(std::string(name) + ": expected " + c10::toString(type) + " rows of " + std::to_string(width) +
               " contiguous elements");
    if (t.size(0) != rows) refuse(std::string(name) + ": expected " + std::to_string(rows) + " rows");
    if (written && rows > 1 && t.stride(0) < width) refuse(std::string(name) + ": rows overlap");
}

void plane(const at::Tensor& c, const at::Tensor& p, int64_t n_kv, int64_t d) {
    if (c.scalar_type() != at::kByte || c.dim() != 4 || c.size(1) != n_kv || c.size(3) != d / 2)
        refuse("kv4 cache: codes are uint8 [pages, n_kv, page_size, head_dim / 2]");
    const int64_t page = c.size(2), groups = d / 64;
    if (p.scalar_type() != at::kHalf || p.dim() != 5 || p.size(0) != c.size(0) || p.size(1) != n_kv ||
        p.size(2) != page || p.size(3) != groups || p.size(4) != 2)
        refuse("kv4 cache: params are float16 [pages, n_kv, page_size, head_dim / 64, 2]");
    if (c.stride(3) != 1 || c.stride(2) != d / 2 || c.stride(1) != page * d / 2 || p.stride(4) != 1 ||
        p.stride(3) != 2 || p.stride(2) != groups * 2 || p.stride(1) != page * groups * 2)
        refuse("kv4 cache: pages are contiguous inside");
    if (c.size(0) > 1 && (c.stride(0) < n_kv * page * d / 2 || p.stride(0) < n_kv * page * groups * 2))
        refuse("kv4 cache: pages overlap");
}

void kv4(PyObject* cache, PyObject* table, PyObject* start, PyObject* ctx, PyObject* status, int64_t rows, int64_t n_kv,
         int64_t d, c10::DeviceIndex here, AmcuKv4Cache* c, AmcuKv4Batch* b) {
    if (!(PyTuple_Check(cache) || PyList_Check(cache)) || PySequence_Fast_GET_SIZE(cache) != 4)
        refuse("kv4 cache: (k_codes, k_params, v_codes, v_params)");
    PyObject** it = PySequence_Fast_ITEMS(cache);
    const at::Tensor &kc = tensor(it[0], here, "k_codes"), &kp = tensor(it[1], here, "k_params"),
                     &vc = tensor(it[2], here, "v_codes"), &vp = tensor(it[3], here, "v_params");
    plane(kc, kp, n_kv, d);
    plane(vc, vp, n_kv, d);
    if (vc.size(0) != kc.size(0) || vc.size(2) != kc.size(2) || vc.stride(0) != kc.stride(0) ||
        vp.stride(0) != kp.stride(0))
        refuse("kv4 cache: K's and V's sizes and strides are the same");
    const at::Tensor &pt = tensor(table, here, "page_table"), &rs = tensor(start, here, "row_start"),
                     &cl = tensor(ctx, here, "ctx_len");
    const at::Tensor* st = optional(status, here, "status");
    const int64_t n_seq = cl.dim() == 1 ? cl.size(0) : -1;
    if (pt.scalar_type() != at::kInt || rs.scalar_type() != at::kInt || cl.scalar_type() != at::kInt || pt.dim() != 2 ||
        pt.size(0) != n_seq || rs.dim() != 1 || rs.size(0) != n_seq + 1 || (pt.stride(1) != 1 && pt.size(1) > 1) ||
        (n_seq > 1 && pt.stride(0) < pt.size(1)) || !rs.is_contiguous() || !cl.is_contiguous())
        refuse("kv4: int32 page_table [n_seq, pages], row_start [n_seq + 1] and ctx_len [n_seq]");
    if (st && (st->scalar_type() != at::kInt || st->numel() < 1)) refuse("kv4: status is one int32");
    const bool many = kc.size(0) > 1;  // a lone page's stride says nothing
    *c = AmcuKv4Cache{kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(), many ? kc.stride(0) : 0,
                      many ? 2 * kp.stride(0) : 0, kc.size(0), kc.size(2), n_kv, d};
    *b = AmcuKv4Batch{static_cast<const int32_t*>(pt.data_ptr()), n_seq > 1 ? pt.stride(0) : 0, pt.size(1),
                      static_cast<const int32_t*>(rs.data_ptr()), static_cast<const int32_t*>(cl.data_ptr()), n_seq, rows,
                      static_cast<int32_t*>(ptr(st))};
}

// A call with rows but no sequence: the C ABI touches nothing, the rows are zero and out of range.
void nowhere(const AmcuKv4Batch& b, PyObject* status, std::initializer_list<at::Tensor> outputs) {
    if (b.n_seq > 0 || b.rows == 0) return;
    for (const at::Tensor& t : outputs) t.zero_();
    if (status != Py_None) THPVariable_Unpack(status).as_strided({1}, {1}).fill_((int64_t)AM_STATUS_OUT_OF_RANGE);
}

// Runs `f`, turning refusals into ValueError and torch's errors into theirs.
template <typename F>
PyObject* call(Py_ssize_t got, Py_ssize_t want, F f) {
    HANDLE_TH_ERRORS
    if (got != want) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        at::AutoDispatchBelowADInplaceOrView guard;
        return f(c10::cuda::device_count() > 0 ? c10::cuda::current_device() : (c10::DeviceIndex)-1);
    } catch (const BadArgument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

void* stream_of(c10::DeviceIndex here) { return c10::cuda::getCurrentCUDAStream(here).stream(); }
PyObject* pair(at::Tensor a, at::Tensor b) {
    PyObject* x = THPVariable_Wrap(std::move(a));
    PyObject* y = x ? THPVariable_Wrap(std::move(b)) : nullptr;
    PyObject* r = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return r;
}

// logits, uniform, temperature, top_k, top_p, min_p, with_prob, out
PyObject* py_sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 8, [&](c10::DeviceIndex here) -> PyObject* {
        const at::Tensor& x = tensor(a[0], here, "logits");
        if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < x.size(1)))
            refuse("sample takes logits [rows, vocab] with contiguous rows that do not overlap");
        const int64_t rows = x.size(0);
        auto one = [&](const at::Tensor* t, at::ScalarType type, const char* name) {
            if (t && (t->scalar_type() != type || t->dim() != 1 || t->size(0) != rows || !t->is_contiguous()))
                refuse(std::string(name) + ": expected one contiguous " + c10::toString(type) + " per row");
            return ptr(t);
        };
        AmcuSampleArgs s = {};
        s.logits = x.data_ptr();
        s.row_stride = rows > 1 ? x.stride(0) : 0;
        s.rows = rows;
        s.vocab = x.size(1);
        s.dtype = act_dtype(x, "logits");
        s.uniform = static_cast<const float*>(one(&tensor(a[1], here, "uniform"), at::kFloat, "uniform"));
        s.temperature = static_cast<const float*>(one(optional(a[2], here, "temperature"), at::kFloat, "temperature"));
        s.top_k = static_cast<const int32_t*>(one(optional(a[3], here, "top_k"), at::kInt, "top_k"));
        s.top_p = static_cast<const float*>(one(optional(a[4], here, "top_p"), at::kFloat, "top_p"));
        s.min_p = static_cast<const float*>(one(optional(a[5], here, "min_p"), at::kFloat, "min_p"));
        const bool with_prob = a[6] == Py_True;
        const at::Tensor* given = optional(a[7], here, "out");
        one(given, at::kLong, "out");
        at::Tensor idx = given ? *given : make({rows}, at::kLong, here);
        at::Tensor prob = with_prob ? make({rows}, at::kFloat, here) : at::Tensor();
        s.out_index = static_cast<int64_t*>(idx.data_ptr());
        s.out_prob = with_prob ? static_cast<float*>(prob.data_ptr()) : nullptr;
        const am_status_code code = f_sample(&s, stream_of(here));
        if (code != AM_STATUS_OK) return PyLong_FromLong(code);
        return with_prob ? pair(std::move(idx), std::move(prob)) : THPVariable_Wrap(std::move(idx));
    });
}

// q, k, v, cache, page_table, row_start, ctx_len, cos_sin, n_q, n_kv, head_dim, q_norm, k_norm, eps, q_out, status
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 16, [&](c10::DeviceIndex here) -> PyObject* {
        const at::Tensor &q = tensor(a[0], here, "q"), &k = tensor(a[1], here, "k"), &v = tensor(a[2], here, "v"),
                         &cs = tensor(a[7], here, "cos_sin");
        const int64_t n_q = integer(a[8]), n_kv = integer(a[9]), d = integer(a[10]);
        const int64_t rows = q.dim() == 2 ? q.size(0) : -1;
        const at::ScalarType type = q.scalar_type();
        AmcuKv4AppendArgs s = {};
        s.dtype = act_dtype(q, "q");
        rows_of(q, rows, n_q * d, type, "q", false);
        rows_of(k, rows, n_kv * d, type, "k", false);
        rows_of(v, rows, n_kv * d, type, "v", false);
        if (cs.scalar_type() != at::kFloat || cs.dim() != 3 || cs.size(1) != d / 2 || cs.size(2) != 2 || !cs.is_contiguous())
            refuse("kv4_append: cos_sin is float32 [positions, head_dim / 2, 2]");
        const at::Tensor *qw = optional(a[11], here, "q_norm"), *kw = optional(a[12], here, "k_norm");
        for (const at::Tensor* w : {qw, kw})
            if (w && (w->scalar_type() != type || w->dim() != 1 || w->size(0) != d || !w->is_contiguous()))
                refuse("kv4_append: norm weights are [head_dim] of q's type");
        const at::Tensor* given = optional(a[14], here, "q_out");
        if (given) rows_of(*given, rows, n_q * d, type, "q_out", true);
        kv4(a[3], a[4], a[5], a[6], a[15], rows, n_kv, d, here, &s.cache, &s.batch);
        at::Tensor out = given ? *given : make({rows, n_q * d}, type, here);
        s.q = q.data_ptr();
        s.k = k.data_ptr();
        s.v = v.data_ptr();
        s.q_out = out.data_ptr();
        s.q_stride = rows > 1 ? q.stride(0) : n_q * d;
        s.k_stride = rows > 1 ? k.stride(0) : n_kv * d;
        s.v_stride = rows > 1 ? v.stride(0) : n_kv * d;
        s.q_out_stride = rows > 1 ? out.stride(0) : n_q * d;
        s.q_norm = ptr(qw);
        s.k_norm = ptr(kw);
        s.eps = (float)real(a[13]);
        s.cos_sin = static_cast<const float*>(cs.data_ptr());
        s.max_pos = cs.size(0);
        s.n_q_heads = n_q;
        const am_status_code code = f_append(&s, stream_of(here));
        if (code == AM_STATUS_OK) nowhere(s.batch, a[15], {out});
        return code != AM_STATUS_OK ? PyLong_FromLong(code) : THPVariable_Wrap(std::move(out));
    });
}

// cache, page_table, row_start, ctx_len, rows, n_kv, head_dim, float32 (else bfloat16), status
PyObject* py_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 9, [&](c10::DeviceIndex here) -> PyObject* {
        const int64_t rows = integer(a[4]), n_kv = integer(a[5]), d = integer(a[6]);
        if (rows < 0 || n_kv < 0 || d < 0) refuse("kv4_gather: negative size");
        AmcuKv4GatherArgs s = {};
        kv4(a[0], a[1], a[2], a[3], a[8], rows, n_kv, d, here, &s.cache, &s.batch);
        const bool f32 = a[7] == Py_True;
        s.dtype = f32 ? AMCU_F32 : AMCU_BF16;
        at::Tensor k = make({rows, n_kv * d}, f32 ? at::kFloat : at::kBFloat16, here);
        at::Tensor v = make({rows, n_kv * d}, f32 ? at::kFloat : at::kBFloat16, here);
        s.k_out = k.data_ptr();
        s.v_out = v.data_ptr();
        s.k_out_stride = s.v_out_stride = n_kv * d;
        const am_status_code code = f_gather(&s, stream_of(here));
        if (code == AM_STATUS_OK) nowhere(s.batch, a[8], {k, v});
        return code != AM_STATUS_OK ? PyLong_FromLong(code) : pair(std::move(k), std::move(v));
    });
}

// q, cache, page_table, row_start, ctx_len, n_q, n_kv, head_dim, scale, out, status
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 11, [&](c10::DeviceIndex here) -> PyObject* {
        const at::Tensor& q = tensor(a[0], here, "q");
        const int64_t n_q = integer(a[5]), n_kv = integer(a[6]), d = integer(a[7]);
        const int64_t rows = q.dim() == 2 ? q.size(0) : -1;
        AmcuKv4AttentionArgs s = {};
        s.dtype = act_dtype(q, "q");
        rows_of(q, rows, n_q * d, q.scalar_type(), "q", false);
        const at::Tensor* given = optional(a[9], here, "out");
        if (given) rows_of(*given, rows, n_q * d, q.scalar_type(), "out", true);
        kv4(a[1], a[2], a[3], a[4], a[10], rows, n_kv, d, here, &s.cache, &s.batch);
        at::Tensor out = given ? *given : make({rows, n_q * d}, q.scalar_type(), here);
        s.q = q.data_ptr();
        s.q_stride = rows > 1 ? q.stride(0) : n_q * d;
        s.out = out.data_ptr();
        s.out_stride = rows > 1 ? out.stride(0) : n_q * d;
        s.n_q_heads = n_q;
        s.scale = (float)real(a[8]);
        const size_t bytes = f_attn_workspace(&s);
        at::Tensor ws;
        if (bytes) {
            ws = make({(int64_t)bytes}, at::kByte, here);
            s.workspace = ws.data_ptr();
            s.workspace_size = bytes;
        }
        const am_status_code code = f_attn(&s, stream_of(here));
        if (code == AM_STATUS_OK) nowhere(s.batch, a[10], {out});
        return code != AM_STATUS_OK ? PyLong_FromLong(code) : THPVariable_Wrap(std::move(out));
    });
}

// Addresses of amcu_sample, amcu_kv4_append, amcu_kv4_gather, amcu_attn_kv4_workspace_bytes, amcu_attn_kv4
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    void* f[5];
    if (n != 5) {
        PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
        return nullptr;
    }
    for (int i = 0; i < 5; ++i)
        if (!(f[i] = PyLong_AsVoidPtr(a[i]))) return nullptr;
    f_sample = reinterpret_cast<decltype(f_sample)>(f[0]);
    f_append = reinterpret_cast<decltype(f_append)>(f[1]);
    f_gather = reinterpret_cast<decltype(f_gather)>(f[2]);
    f_attn_workspace = reinterpret_cast<decltype(f_attn_workspace)>(f[3]);
    f_attn = reinterpret_cast<decltype(f_attn)>(f[4]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
        {"bind", reinterpret_cast<PyCFunction>(py_bind), METH_FASTCALL, nullptr},
        {"sample", reinterpret_cast<PyCFunction>(py_sample), METH_FASTCALL, nullptr},
        {"kv4_append", reinterpret_cast<PyCFunction>(py_append), METH_FASTCALL, nullptr},
        {"kv4_gather", reinterpret_cast<PyCFunction>(py_gather), METH_FASTCALL, nullptr},
        {"attention_kv4", reinterpret_cast<PyCFunction>(py_attention), METH_FASTCALL, nullptr},
        {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_ops_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_native(void) { return PyModule_Create(&module_def); }
