// host.cpp -- the host side of the streaming calls (ress_b200/kernels.py):
// checks of torch tensors, allocation of outputs and workspaces, and the call
// into the C ABI (include/ress_sm100.h) on the current stream.
//
// These calls are made per token and take the GPU a few microseconds; the
// same checks in Python took 6 to 13 microseconds a call, which bounded it.
// A call runs on its tensors' device, whichever is the current one.
// The library's entry points and the addresses of the devices' status words
// are handed over by bind(); nothing here is linked against the library.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/ress_sm100.h"

namespace {

constexpr int64_t PAGE = 64, HD = 64;

struct Api {
    decltype(&ress_cache_append) cache_append;
    decltype(&ress_cache_attn) cache_attn;
    decltype(&ress_cache_attn_workspace) cache_attn_workspace;
    decltype(&ress_int8_quant_rows) int8_quant_rows;
    decltype(&ress_int8_linear) int8_linear;
    decltype(&ress_int8_linear_workspace) int8_linear_workspace;
    decltype(&ress_error_string) error_string;
} api;
PyObject *error_type = nullptr, *status_of = nullptr;  // RessError; device index -> address of its status word
int32_t *status_ptr[64] = {};

struct Refusal {
    std::string what;
};
struct PythonError {};  // an exception is set already
inline void require(bool ok, const char *what) {
    if (!ok) throw Refusal{what};
}
inline void returned(int code, const char *call) {
    if (code != RESS_OK)
        throw Refusal{std::string(call) + " failed: " + api.error_string(code) + " (code " + std::to_string(code) + ")"};
}

// A tensor argument; nullptr for None.
inline const at::Tensor *opt(PyObject *o, const char *name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) throw Refusal{std::string(name) + " must be a tensor"};
    return &THPVariable_Unpack(o);
}
inline const at::Tensor &tensor(PyObject *o, const char *name) {
    const at::Tensor *t = opt(o, name);
    if (t == nullptr) throw Refusal{std::string(name) + " must be a tensor"};
    return *t;
}
inline int cuda_index(const at::Tensor &t) {
    require(t.is_cuda(), "ress_b200 kernels run on CUDA tensors only (no CPU fallback)");
    return (int)t.get_device();
}
// Makes device i current where it is not.
struct Current {
    c10::cuda::OptionalCUDAGuard guard;
    explicit Current(int i) {
        if (c10::cuda::current_device() != i) guard.set_index((c10::DeviceIndex)i);
    }
};
inline void on_device(int i, std::initializer_list<const at::Tensor *> ts) {
    for (const at::Tensor *t : ts)
        require(t == nullptr || (t->is_cuda() && t->get_device() == i), "all tensors of a call are on one CUDA device");
}
// The operators have no backward: a result without history would cut gradients silently.
inline void no_gradients(std::initializer_list<const at::Tensor *> ts) {
    if (!c10::GradMode::is_enabled()) return;
    for (const at::Tensor *t : ts)
        require(t == nullptr || !t->requires_grad(),
                "the streaming operators are for inference: call them under torch.no_grad() or torch.inference_mode()");
}
inline int dtype_code(at::ScalarType t) {
    if (t == at::kFloat) return RESS_F32;
    if (t == at::kBFloat16) return RESS_BF16;
    throw Refusal{std::string("unsupported dtype ") + c10::toString(t) + " (float32 or bfloat16)"};
}
inline at::ScalarType dtype_of(int code) { return code == RESS_BF16 ? at::kBFloat16 : at::kFloat; }
inline int32_t *status_word(int i) {
    require(i >= 0 && i < 64, "device index out of range");
    if (status_ptr[i] == nullptr) {
        PyObject *r = PyObject_CallFunction(status_of, "i", i);
        if (r == nullptr) throw PythonError{};
        status_ptr[i] = reinterpret_cast<int32_t *>(PyLong_AsVoidPtr(r));
        Py_DECREF(r);
        if (status_ptr[i] == nullptr) throw PythonError{};
    }
    return status_ptr[i];
}
inline ress_stream_t stream_of(int i) {
    return reinterpret_cast<ress_stream_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)i).stream());
}
template <typename T> inline T *data(const at::Tensor *t) {
    return t == nullptr ? nullptr : reinterpret_cast<T *>(t->data_ptr());
}

// (B, T, heads, 64) rows; 0 for a stride that is never used
struct Rows {
    int64_t B, T, H, sb, st, sh;
};
inline Rows head_rows(const at::Tensor &x, const char *name) {
    if (x.dim() != 4 || x.size(3) != HD || x.stride(3) != 1)
        throw Refusal{std::string(name) + " must be (B, T, heads, 64) with a contiguous last dim"};
    Rows r{x.size(0), x.size(1), x.size(2), x.stride(0), x.stride(1), x.stride(2)};
    if (r.B <= 1) r.sb = 0;
    if (r.T <= 1) r.st = 0;
    if (r.H <= 1) r.sh = 0;
    return r;
}

// The cache's tensors (device i, B streams), checked.
ress_cache cache_of(int i, int64_t B, PyObject *const *o) {
    const at::Tensor &kp = tensor(o[0], "k_pages"), &vp = tensor(o[1], "v_pages"), &ks = tensor(o[2], "k_scale"),
                     &vs = tensor(o[3], "v_scale"), &table = tensor(o[4], "table"), &lens = tensor(o[5], "lens");
    on_device(i, {&kp, &vp, &ks, &vs, &table, &lens});
    require(kp.scalar_type() == at::kFloat8_e4m3fn && vp.scalar_type() == at::kFloat8_e4m3fn,
            "cache pages are float8_e4m3fn");
    require(ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu,
            "cache scales are float8_e8m0fnu");
    require(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt, "the page table and the lengths are int32");
    require(kp.dim() == 4 && kp.size(2) == PAGE && kp.size(3) == HD && vp.sizes() == kp.sizes(),
            "cache pages are (pages, heads, 64, 64), alike for k and v");
    require(kp.stride(2) == HD && kp.stride(3) == 1 && vp.strides() == kp.strides(),
            "a page's block of one head is contiguous, and k and v pages share strides");
    const int64_t n = kp.size(0), H = kp.size(1);
    require(ks.dim() == 2 && ks.size(0) == n && ks.size(1) == H && vs.sizes() == ks.sizes() &&
                vs.strides() == ks.strides() && (ks.stride(1) == 1 || H == 1),
            "cache scales are (pages, heads) with contiguous heads, alike for k and v");
    require(table.dim() == 2 && table.size(0) == B && (table.stride(1) == 1 || table.size(1) == 1),
            "the page table is (streams, pages) with contiguous rows");
    require(lens.dim() == 1 && lens.size(0) == B && lens.is_contiguous(), "lens holds one contiguous length per stream");
    // the stride of a single page or head is never used
    const int64_t hs = H > 1 ? kp.stride(1) : PAGE * HD;
    return ress_cache{data<uint8_t>(&kp), data<uint8_t>(&vp), data<uint8_t>(&ks), data<uint8_t>(&vs), n, H,
                      n > 1 ? kp.stride(0) : H * hs, hs, n > 1 ? ks.stride(0) : H, data<int32_t>(&table),
                      table.stride(0), table.size(1), data<int32_t>(&lens), B};
}

template <typename F> PyObject *guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refusal &r) {
        PyErr_SetString(error_type, r.what.c_str());
        return nullptr;
    } catch (const PythonError &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}
void count(Py_ssize_t have, Py_ssize_t want) {
    if (have != want) throw Refusal{"wrong number of arguments"};
}

// (k, v, k_pages, v_pages, k_scale, v_scale, table, lens, q, n_new, qn_weight, qn_bias, kn_weight, kn_bias, eps, pos,
//  rope_cos, rope_sin)
PyObject *cache_append(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        count(n, 18);
        const at::Tensor &k = tensor(o[0], "k"), &v = tensor(o[1], "v");
        const int i = cuda_index(k);
        const Current current(i);
        const at::Tensor *q = opt(o[8], "q"), *n_new = opt(o[9], "n_new"), *pos = opt(o[15], "pos"),
                         *cos = opt(o[16], "rope_cos"), *sin = opt(o[17], "rope_sin");
        const at::ScalarType dtype = k.scalar_type();
        ress_append_args a{};
        a.dtype = dtype_code(dtype);
        const Rows rk = head_rows(k, "k"), rv = head_rows(v, "v");
        const ress_cache c = cache_of(i, rk.B, o + 2);
        require(v.sizes() == k.sizes() && rk.H == c.heads && v.scalar_type() == dtype,
                "k and v must be alike, with the cache's heads");
        on_device(i, {&v, q, n_new, pos, cos, sin});
        no_gradients({&k, &v, q});
        a.k = data<void>(&k);
        a.v = data<void>(&v);
        a.tokens = rk.T;
        a.k_sb = rk.sb, a.k_st = rk.st, a.k_sh = rk.sh;
        a.v_sb = rv.sb, a.v_st = rv.st, a.v_sh = rv.sh;
        if (n_new != nullptr)
            require(n_new->scalar_type() == at::kInt && n_new->dim() == 1 && n_new->size(0) == rk.B && n_new->is_contiguous(),
                    "n_new holds one contiguous int32 per stream");
        a.n_new = data<int32_t>(n_new);
        const void *norms[4];
        at::Tensor wide[4];  // fp32 copies of bf16 norms, where the rows or another norm are fp32 or one is not aligned
        int n_f32 = 0, n_bf16 = 0;
        bool aligned = true;
        for (int j = 0; j < 4; ++j) {
            const at::Tensor *w = opt(o[10 + j], "a norm's weight");
            require(w == nullptr || (w->is_cuda() && w->get_device() == i &&
                                     (w->scalar_type() == at::kFloat || w->scalar_type() == at::kBFloat16) && w->dim() == 1 &&
                                     w->size(0) == HD && w->is_contiguous()),
                    "norm weights and biases are contiguous fp32 or bf16 (64,) on the call's device");
            no_gradients({w});
            norms[j] = data<void>(w);
            if (w != nullptr) ++(w->scalar_type() == at::kFloat ? n_f32 : n_bf16);
            aligned &= (reinterpret_cast<uintptr_t>(norms[j]) & 15) == 0;
        }
        if (n_bf16 > 0 && n_f32 == 0 && aligned && dtype == at::kBFloat16)
            a.dtype |= RESS_BF16_NORMS;
        else if (n_bf16 > 0 || !aligned)
            for (int j = 0; j < 4; ++j)
                if (norms[j] != nullptr) {
                    wide[j] = opt(o[10 + j], "")->to(at::kFloat, /*non_blocking=*/false, /*copy=*/true);
                    norms[j] = data<void>(&wide[j]);
                }
        require((norms[0] == nullptr) == (norms[1] == nullptr) && (norms[2] == nullptr) == (norms[3] == nullptr),
                "a norm has both weight and bias");
        a.qn_weight = norms[0], a.qn_bias = norms[1], a.kn_weight = norms[2], a.kn_bias = norms[3];
        a.eps = PyFloat_AsDouble(o[14]);
        if (PyErr_Occurred()) throw PythonError{};
        require((cos == nullptr) == (sin == nullptr), "the rotary embedding has both tables");
        at::Tensor cosc, sinc, posc;  // contiguous
        if (cos != nullptr) {
            require(pos != nullptr && pos->scalar_type() == at::kLong && pos->dim() == 3 && pos->size(0) == rk.B &&
                        pos->size(1) == rk.T && pos->size(2) == 2,
                    "pos must be (B, T, 2) int64");
            require(cos->scalar_type() == dtype && sin->scalar_type() == dtype && cos->dim() == 2 && cos->size(1) == 32 &&
                        sin->sizes() == cos->sizes(),
                    "rotary tables must be (max_pos, 32) in k's dtype");
            cosc = cos->contiguous(), sinc = sin->contiguous(), posc = pos->contiguous();
            a.rope_cos = data<void>(&cosc), a.rope_sin = data<void>(&sinc);
            a.pos = data<int64_t>(&posc);
            a.rope_len = cos->size(0);
        }
        at::Tensor out;
        if (q != nullptr) {
            const Rows rq = head_rows(*q, "q");
            require(rq.B == rk.B && rq.T == rk.T && q->scalar_type() == dtype && c.heads > 0 && rq.H > 0 && rq.H % c.heads == 0,
                    "q must have k's tokens and type, and a multiple of its heads");
            out = at::empty({rk.B, rk.T, rq.H, HD}, q->options());
            a.q = data<void>(q);
            a.q_out = data<void>(&out);
            a.q_heads = rq.H;
            a.q_sb = rq.sb, a.q_st = rq.st, a.q_sh = rq.sh;
        }
        if (rk.B > 0 && rk.T > 0) returned(api.cache_append(&c, &a, status_word(i), stream_of(i)), "ress_cache_append");
        if (q == nullptr) Py_RETURN_NONE;
        return THPVariable_Wrap(std::move(out));
    });
}

// (q, k_pages, v_pages, k_scale, v_scale, table, lens, limits, sm_scale or None, out, out_bf16)
PyObject *cache_attn(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        count(n, 11);
        const at::Tensor &q = tensor(o[0], "q");
        const int i = cuda_index(q);
        const Current current(i);
        require(q.scalar_type() == at::kBFloat16, "cache_attn takes bf16 q");
        no_gradients({&q});
        const Rows r = head_rows(q, "q");
        const ress_cache c = cache_of(i, r.B, o + 1);
        const at::Tensor *limits = opt(o[7], "limits"), *given = opt(o[9], "out");
        require(c.heads > 0 && r.H > 0 && r.H % c.heads == 0, "q's heads must be a multiple of the cache's");
        require(limits == nullptr || (limits->is_cuda() && limits->get_device() == i && limits->scalar_type() == at::kInt &&
                                      limits->dim() == 2 && limits->size(0) == r.B && limits->size(1) == r.T &&
                                      limits->is_contiguous()),
                "limits must be contiguous (B, T) int32 on the call's device");
        ress_attn_args a{};
        a.q = data<uint16_t>(&q);
        a.tokens = r.T;
        a.q_heads = r.H;
        a.q_sb = r.sb, a.q_st = r.st, a.q_sh = r.sh;
        a.limits = data<int32_t>(limits);
        a.sm_scale = o[8] == Py_None ? 0.125 : PyFloat_AsDouble(o[8]);
        const int bf16 = PyObject_IsTrue(o[10]);
        if (PyErr_Occurred()) throw PythonError{};
        at::Tensor out;
        if (given != nullptr) {
            require(given->is_cuda() && given->get_device() == i && given->sizes() == q.sizes() &&
                        (given->scalar_type() == at::kBFloat16 || given->scalar_type() == at::kFloat),
                    "cache_attn output must have q's shape, bf16 or fp32, on the call's device");
            out = *given;
        } else {
            out = at::empty(q.sizes(), q.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
        }
        const Rows ro = head_rows(out, "out");
        a.out = data<void>(&out);
        a.o_sb = ro.sb, a.o_st = ro.st, a.o_sh = ro.sh;
        a.out_bf16 = out.scalar_type() == at::kBFloat16;
        if (r.B > 0 && r.T > 0) {
            const size_t need = api.cache_attn_workspace(r.B, c.heads, r.T * (r.H / c.heads), c.table_width);
            at::Tensor ws;
            if (need > 0) {
                ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
                a.workspace = data<void>(&ws);
            }
            returned(api.cache_attn(&c, &a, status_word(i), stream_of(i)), "ress_cache_attn");
        }
        return THPVariable_Wrap(std::move(out));
    });
}

// whether the kernels can read x: (M, K) rows that do not overlap, 16-byte aligned
bool readable(const at::Tensor &x) {
    if (x.dim() != 2 || x.stride(1) != 1 || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15)) return false;
    return x.size(0) <= 1 || (x.stride(0) >= x.size(1) && x.stride(0) * x.element_size() % 16 == 0);
}
// x as (M, K) rows; a copy only where they are not readable as they lie
at::Tensor rows2d(const at::Tensor &x) {
    require(x.dim() >= 1 && x.size(-1) > 0, "x has no features");
    at::Tensor y = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    return readable(y) ? y : y.clone(at::MemoryFormat::Contiguous);
}
int64_t row_stride(const at::Tensor &x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// (x)
PyObject *int8_quant_rows(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        count(n, 1);
        const at::Tensor &x = tensor(o[0], "x");
        const int i = cuda_index(x), dt = dtype_code(x.scalar_type());
        const Current current(i);
        no_gradients({&x});
        const at::Tensor rows = rows2d(x);
        const int64_t M = rows.size(0), K = rows.size(1);
        require(M <= INT_MAX && K <= INT_MAX, "x is too large");
        at::Tensor x8 = at::empty(x.sizes(), x.options().dtype(at::kChar));
        at::Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
        if (M > 0)
            returned(api.int8_quant_rows(data<void>(&rows), dt, (int)M, (int)K, row_stride(rows), data<int8_t>(&x8),
                                         data<float>(&scale), stream_of(i)),
                     "ress_int8_quant_rows");
        PyObject *a = THPVariable_Wrap(std::move(x8)), *b = THPVariable_Wrap(std::move(scale));
        PyObject *pair = a != nullptr && b != nullptr ? PyTuple_Pack(2, a, b) : nullptr;
        Py_XDECREF(a);
        Py_XDECREF(b);
        return pair;
    });
}

// (x, w8, w_scale, bias, gelu, dtype code of the output or -1 for x's)
PyObject *int8_linear(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        count(n, 6);
        const at::Tensor &x = tensor(o[0], "x"), &w = tensor(o[1], "w8"), &ws = tensor(o[2], "w_scale");
        const at::Tensor *bias = opt(o[3], "bias");
        const int i = cuda_index(x), dt = dtype_code(x.scalar_type());
        const Current current(i);
        const int gelu = PyObject_IsTrue(o[4]);
        const long want = PyLong_AsLong(o[5]);
        if (PyErr_Occurred()) throw PythonError{};
        const int odt = want < 0 ? dt : (int)want;
        on_device(i, {&w, &ws, bias});
        no_gradients({&x, &ws, bias});
        require(w.scalar_type() == at::kChar && w.dim() == 2 && w.is_contiguous(), "w8 must be contiguous int8 (N, K)");
        const int64_t N = w.size(0), K = w.size(1);
        require(x.dim() >= 1 && x.size(-1) == K, "x and w8 have unlike numbers of features");
        for (const at::Tensor *t : {&ws, bias})
            require(t == nullptr || (t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == N && t->is_contiguous()),
                    "w_scale and bias are contiguous fp32 (N,)");
        at::Tensor copy;
        const at::Tensor *rows = &x;
        if (!readable(x)) {
            copy = rows2d(x);
            rows = &copy;
        }
        const int64_t M = rows->size(0);
        require(M <= INT_MAX && K <= INT_MAX && N <= INT_MAX, "the product is too large");
        at::DimVector shape(x.sizes());
        shape.back() = N;
        at::Tensor out = at::empty(shape, x.options().dtype(dtype_of(odt)));
        if (M > 0 && N > 0) {
            const size_t need = api.int8_linear_workspace((int)M, (int)K);
            at::Tensor work;
            if (need > 0) work = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
            returned(api.int8_linear(data<void>(rows), dt, (int)M, (int)N, (int)K, row_stride(*rows), data<int8_t>(&w),
                                     data<float>(&ws), data<float>(bias), gelu, data<void>(&out), odt, N,
                                     need > 0 ? data<void>(&work) : nullptr, status_word(i), stream_of(i)),
                     "ress_int8_linear");
        }
        return THPVariable_Wrap(std::move(out));
    });
}

// (error type, status callable, {entry point: address})
PyObject *bind(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 3 || !PyDict_Check(o[2])) {
            PyErr_SetString(PyExc_TypeError, "bind(error type, status callable, {entry point: address})");
            throw PythonError{};
        }
        auto address = [&](const char *name) -> void * {
            PyObject *v = PyDict_GetItemString(o[2], name);  // borrowed
            void *p = v == nullptr ? nullptr : PyLong_AsVoidPtr(v);
            if (p == nullptr) {
                if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", name);
                throw PythonError{};
            }
            return p;
        };
        Api a;
        a.cache_append = reinterpret_cast<decltype(a.cache_append)>(address("ress_cache_append"));
        a.cache_attn = reinterpret_cast<decltype(a.cache_attn)>(address("ress_cache_attn"));
        a.cache_attn_workspace = reinterpret_cast<decltype(a.cache_attn_workspace)>(address("ress_cache_attn_workspace"));
        a.int8_quant_rows = reinterpret_cast<decltype(a.int8_quant_rows)>(address("ress_int8_quant_rows"));
        a.int8_linear = reinterpret_cast<decltype(a.int8_linear)>(address("ress_int8_linear"));
        a.int8_linear_workspace = reinterpret_cast<decltype(a.int8_linear_workspace)>(address("ress_int8_linear_workspace"));
        a.error_string = reinterpret_cast<decltype(a.error_string)>(address("ress_error_string"));
        api = a;
        Py_INCREF(o[0]);
        Py_INCREF(o[1]);
        Py_XDECREF(error_type);
        Py_XDECREF(status_of);
        error_type = o[0];
        status_of = o[1];
        Py_RETURN_NONE;
    });
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(cache_append), FAST(cache_attn), FAST(int8_quant_rows), FAST(int8_linear),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host side of the streaming calls.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
