// Host path between PyTorch and the C ABI: what happens on the CPU for one call of a quantised linear.
//
// A decode call runs 5 to 10 us on the GPU.  The same argument handling in Python (dispatcher to a Python
// implementation, attribute reads, ctypes) took 30 to 36 us a call and was what an eager decode step ran at; here it
// is one C++ function per call: type and shape checks, one output allocation, one C ABI call.
//
// Two ways in:
//   * the CUDA implementations of torch.ops.binary_kernels.* (schemas: nanoquant_b200/ops.py), for operands in the
//     kernels' tile layout; operands in the reference's layouts go to the Python implementation, which converts them
//     once and keeps the result on the tensor;
//   * plain functions for this package's own modules (no dispatcher).  They return None whenever a call is not the
//     plain case (other types, tensor subclasses, wrappers of transforms, dispatch modes, odd dimensions, a linear that
//     autograd would record); the caller then takes the general route.
#include <Python.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/grad_mode.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/as_strided.h>
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <mutex>
#include <optional>
#include <unordered_set>
#include <vector>

#include "nanoquant_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int kMaxLinears = 4;
constexpr int kMaxDevices = 64;

// ---------------------------------------------------------------------------------------------------------------
// Python callbacks, set once by nanoquant_b200.ops
// ---------------------------------------------------------------------------------------------------------------
PyObject* g_raise_status = nullptr;    // (status, what): raises
PyObject* g_grow_scratch = nullptr;    // (device index, bytes): makes the scratch hold that many bytes, or raises
PyObject* g_dyn_general = nullptr;     // Python implementations of the operators (reference operand layouts)
PyObject* g_marlin_general = nullptr;
PyObject* g_thread_scratch = nullptr;  // () -> the tensor that this thread runs on instead of the device's scratch

// What module_call compares with: NanoQuantLinear and its forward, nn.Module and its way from a call to forward, the hooks on every module.
struct ModuleClass {
    PyTypeObject *type = nullptr, *base = nullptr;
    PyObject *forward = nullptr, *call = nullptr, *call_impl = nullptr;
    std::vector<PyObject*> global_hooks;
};
ModuleClass g_module_class;

// Calls a Python function with the GIL held and throws its exception.
PyObject* call_python(PyObject* fn, PyObject* args) {
    TORCH_CHECK(fn != nullptr, "nanoquant_b200: the host extension has not been initialised");
    PyObject* r = PyObject_CallObject(fn, args);
    Py_DECREF(args);
    if (!r) {
        python_error err;
        err.persist();
        throw std::move(err);
    }
    return r;
}

[[noreturn]] void fail(int status, const char* what) {
    pybind11::gil_scoped_acquire gil;
    Py_XDECREF(call_python(g_raise_status, Py_BuildValue("(is)", status, what)));
    TORCH_CHECK(false, what, ": nq_status ", status);
}

// ---------------------------------------------------------------------------------------------------------------
// scratch: one buffer per device (owned by nanoquant_b200.ops, which keeps it alive), a thread may override it
// ---------------------------------------------------------------------------------------------------------------
struct Scratch {
    void* ptr = nullptr;
    size_t bytes = 0;
};
Scratch g_scratch[kMaxDevices];
std::mutex g_scratch_mutex;            // pointer and size change together
thread_local Scratch t_override;

Scratch scratch_of(int dev) {
    if (t_override.ptr) return t_override;
    std::lock_guard<std::mutex> lock(g_scratch_mutex);
    return g_scratch[dev];
}

void grow_scratch(int dev, size_t bytes) {
    pybind11::gil_scoped_acquire gil;
    Py_DECREF(call_python(g_grow_scratch, Py_BuildValue("(in)", dev, (Py_ssize_t)bytes)));
}

// ---------------------------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------------------------
// Makes `dev` current for the C ABI call if it is not (a query and nothing else in the usual case).
struct OnDevice {
    explicit OnDevice(int dev) {
        if (c10::cuda::current_device() != dev) guard.emplace(dev);
    }
    std::optional<c10::cuda::CUDAGuard> guard;
};

int dtype_id(at::ScalarType t) { return t == at::kHalf ? NQ_F16 : NQ_BF16; }
bool is_16bit(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

// Up to four linears at T tokens: the decode kernel for few tokens and for sizes the tensor-core path does not
// take (columns or ranks that are no multiple of 8), the tensor-core path for the rest.
void launch(nq_linear_desc* d, int n, int64_t T, int dtype, int dev) {
    static const int gemv_max = nq_gemv_max_tokens();
    bool gemv = T <= gemv_max;
    if (!gemv && n == 1 && (d->N % 8 != 0 || d->R % 8 != 0)) gemv = true;
    OnDevice on(dev);
    const nq_stream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    const auto fwd = gemv ? nq_decode_group_fwd : nq_gemm_group_fwd;
    Scratch s = scratch_of(dev);
    int st = s.ptr ? fwd(d, n, (int)T, dtype, s.ptr, s.bytes, stream) : (int)NQ_ERR_SCRATCH;
    if (st == NQ_ERR_SCRATCH) {   // nothing has been launched: the scratch is checked first
        grow_scratch(dev, gemv ? nq_gemv_group_scratch_bytes(d, n, (int)T) : nq_gemm_group_scratch_bytes(d, n, (int)T));
        s = scratch_of(dev);
        st = fwd(d, n, (int)T, dtype, s.ptr, s.bytes, stream);
    }
    if (st < 0) fail(st, gemv ? "nq_decode_group_fwd" : "nq_gemm_group_fwd");
}

// A linear's operands.  `rank` comes from the caller: the tile layout pads it.
struct Linear {
    const Tensor *s_in, *v, *s_mid, *u, *s_out, *bias;
    int64_t rank;
};

void describe(nq_linear_desc& d, const Linear& l, const void* x, int64_t N, int64_t ldx, void* y, int64_t ldy) {
    d = nq_linear_desc{};
    d.x = x;
    d.s_in = l.s_in->const_data_ptr();
    d.v_tiles = l.v->const_data_ptr();
    d.s_mid = l.s_mid ? l.s_mid->const_data_ptr() : nullptr;
    d.u_tiles = l.u->const_data_ptr();
    d.s_out = l.s_out->const_data_ptr();
    d.y = y;
    d.N = (int)N;
    d.R = (int)l.rank;
    d.M = (int)l.s_out->size(0);
    d.ldx = ldx;
    d.ldy = ldy;
    d.bias = l.bias ? l.bias->const_data_ptr() : nullptr;
}

// Without the dispatcher (1.2 us of a call): nothing that could intercept it is active where a plain call is taken, and the kernel
// writes every element.
Tensor new_output(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}
Tensor new_output(at::IntArrayRef shape, const Tensor& like) { return new_output(shape, like, like.scalar_type()); }

// y[..., M] for a contiguous x[..., N]
Tensor linear(const Tensor& x, const Linear& l) {
    const int64_t N = x.size(-1), T = N ? x.numel() / N : 0, M = l.s_out->size(0);
    c10::SmallVector<int64_t, 4> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = M;
    Tensor y = new_output(shape, x);
    if (T == 0) return y;
    nq_linear_desc d;
    describe(d, l, x.const_data_ptr(), N, N, y.mutable_data_ptr(), M);
    launch(&d, 1, T, dtype_id(x.scalar_type()), x.get_device());
    return y;
}

// ---------------------------------------------------------------------------------------------------------------
// operators
// ---------------------------------------------------------------------------------------------------------------
void check_operand(const Tensor& t, const char* name, at::ScalarType dtype, const char* dtype_name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype_name, " tensor");
}

// The reference dispatches its tuning arguments through compile-time lists and raises ValueError on a miss
// (cuda/meta_utils.h:14-38, cuda/gemv_kernel.cu:351-354); the kernels here have no such knobs.
void check_sweep(const char* name, int64_t v, std::initializer_list<int64_t> choices) {
    for (int64_t c : choices)
        if (c == v) return;
    std::string list;
    for (int64_t c : choices) list += (list.empty() ? "" : ", ") + std::to_string(c);
    TORCH_CHECK_VALUE(false, name, " should be one of [", list, "], but ", v, " was given");
}

PyObject* wrap(const OptTensor& t) {
    if (!t) Py_RETURN_NONE;
    return THPVariable_Wrap(*t);
}
Tensor unwrap_result(PyObject* r) {
    Tensor y = THPVariable_Unpack(r);
    Py_DECREF(r);
    return y;
}

Tensor nanoquant_dyn_forward(const Tensor& x, const Tensor& scale_g, const Tensor& Ubits, const OptTensor& scale_l,
                             const Tensor& Vbits, const Tensor& scale_h, int64_t th1, int64_t th2, int64_t rpw1,
                             int64_t rpw2, int64_t acc1, int64_t acc2, int64_t pipe1, int64_t pipe2) {
    if (Ubits.dim() != 3 || Vbits.dim() != 3 || !scale_l) {   // operands to convert, or a rank to look up
        pybind11::gil_scoped_acquire gil;
        return unwrap_result(call_python(g_dyn_general, Py_BuildValue(
            "(NNNNNNLLLLLLLL)", THPVariable_Wrap(x), THPVariable_Wrap(scale_g), THPVariable_Wrap(Ubits), wrap(scale_l),
            THPVariable_Wrap(Vbits), THPVariable_Wrap(scale_h), (long long)th1, (long long)th2, (long long)rpw1,
            (long long)rpw2, (long long)acc1, (long long)acc2, (long long)pipe1, (long long)pipe2)));
    }
    const at::ScalarType dt = x.scalar_type();   // checks in the order of the reference (cuda/gemv_kernel.cu:317-338)
    TORCH_CHECK(is_16bit(dt), "Support only Half or BFloat16");
    const char* name = dt == at::kHalf ? "float16" : "bfloat16";
    check_operand(x, "x", dt, name);
    check_operand(scale_g, "scale_g", dt, name);
    check_operand(scale_h, "scale_h", dt, name);
    check_operand(Ubits, "Ubits", at::kInt, "int32");
    check_operand(Vbits, "Vbits", at::kInt, "int32");
    check_operand(*scale_l, "(*scale_l)", dt, name);
    TORCH_CHECK(scale_g.size(0) == x.size(-1), "scale_g size mismatch");
    check_sweep("n_th1", th1, {64, 128, 256});
    check_sweep("n_rpw1", rpw1, {1, 2, 4, 8});
    check_sweep("n_acc1", acc1, {1, 2});
    check_sweep("n_pipe1", pipe1, {1, 2, 4, 8, 16});
    check_sweep("n_th2", th2, {64, 128, 256});
    check_sweep("n_rpw2", rpw2, {1, 2, 4, 8});
    check_sweep("n_acc2", acc2, {1, 2});
    check_sweep("n_pipe2", pipe2, {1, 2, 4, 8, 16});
    return linear(x, Linear{&scale_g, &Ubits, &*scale_l, &Vbits, &scale_h, nullptr, scale_l->size(0)});
}

// `weight_u` is the FIRST stage (module V), `weight_v` the second (reference cuda/gemm.cpp:112-122)
Tensor marlin_nanoquant_forward(const Tensor& x, const Tensor& weight_u, const Tensor& weight_v, const OptTensor& scale_g,
                                const OptTensor& scale_l, const OptTensor& scale_h, const Tensor& workspace) {
    if (weight_u.dim() == 3 && scale_g && scale_l && scale_h && is_16bit(x.scalar_type()) && x.dim() == 2)
        return linear(x.is_contiguous() ? x : x.contiguous(),
                      Linear{&*scale_g, &weight_u, &*scale_l, &weight_v, &*scale_h, nullptr, scale_l->size(0)});
    pybind11::gil_scoped_acquire gil;
    return unwrap_result(call_python(g_marlin_general, Py_BuildValue(
        "(NNNNNNN)", THPVariable_Wrap(x), THPVariable_Wrap(weight_u), THPVariable_Wrap(weight_v), wrap(scale_g),
        wrap(scale_l), wrap(scale_h), THPVariable_Wrap(workspace))));
}

TORCH_LIBRARY_IMPL(binary_kernels, CUDA, m) {
    m.impl("nanoquant_dyn_forward", nanoquant_dyn_forward);
    m.impl("marlin_nanoquant_forward", marlin_nanoquant_forward);
}

// ---------------------------------------------------------------------------------------------------------------
// plain functions
// ---------------------------------------------------------------------------------------------------------------
// A tensor argument without anything that would have to go through the dispatcher: its keys are those of a strided CUDA tensor and of autograd
// alone.  Not so for the wrappers of transforms (vmap, grad, functionalize), subclasses that dispatch in Python and lazily negated or
// zero tensors, whose memory (if they have any) does not hold their values.
const uint64_t kPlainKeys = c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView,
                                                 c10::DispatchKey::AutocastCUDA}).raw_repr();
const Tensor* plain(PyObject* o) {
    if (!THPVariable_Check(o)) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && (t.key_set().raw_repr() & ~kPlainKeys) == 0 ? &t : nullptr;
}
// (what torch.jit.trace records are calls of the dispatcher: a result of any other call is a constant to it)
bool exact_plain(PyObject* o) { return THPVariable_CheckExact(o) && !c10::impl::dispatch_mode_enabled() && !torch::jit::tracer::isTracing(); }

// (s_in, v_tiles, s_mid | None, u_tiles, s_out, rank, bias | None) from `a[0..6]`; false: not the plain case.
bool parse_linear(PyObject* const* a, at::ScalarType dt, int64_t N, Linear& l) {
    auto vec = [&](PyObject* o, int64_t n) -> const Tensor* {
        const Tensor* t = plain(o);
        return t && t->scalar_type() == dt && t->dim() == 1 && (n < 0 || t->size(0) == n) && t->is_contiguous() ? t : nullptr;
    };
    auto tiles = [&](PyObject* o) -> const Tensor* {
        const Tensor* t = plain(o);
        return t && t->scalar_type() == at::kInt && t->dim() == 3 && t->is_contiguous() ? t : nullptr;
    };
    l.rank = PyLong_AsLongLong(a[5]);
    if (l.rank <= 0) { PyErr_Clear(); return false; }
    l.s_in = vec(a[0], N);
    l.v = tiles(a[1]);
    l.s_mid = a[2] == Py_None ? nullptr : vec(a[2], l.rank);
    l.u = tiles(a[3]);
    l.s_out = vec(a[4], -1);
    if (!l.s_in || !l.v || !l.u || !l.s_out || (a[2] != Py_None && !l.s_mid)) return false;
    const int64_t M = l.s_out->size(0);
    l.bias = a[6] == Py_None ? nullptr : vec(a[6], M);
    if (a[6] != Py_None && !l.bias) return false;
    // the tiles are what the descriptor's sizes say: 16 rows x 256 columns each
    return l.v->size(0) == (l.rank + 15) / 16 && l.v->size(1) == (N + 255) / 256 && l.u->size(0) == (M + 15) / 16 &&
           l.u->size(1) == (l.rank + 255) / 256;
}

// Autograd would record the operator behind this call (as one without a derivative, which backward then says).  A linear with a bias has
// no operator.
bool recorded(const Tensor& x, const Linear& l) {
    if (l.bias || !at::GradMode::is_enabled()) return false;
    for (const Tensor* t : {&x, l.s_in, l.s_mid, l.s_out})
        if (t && t->requires_grad()) return true;
    return false;
}

// linear_forward(x, s_in, v_tiles, s_mid, u_tiles, s_out, rank, bias) -> y or None
PyObject* py_linear_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 8, "linear_forward takes 8 arguments");
    if (!exact_plain(a[0])) Py_RETURN_NONE;
    const Tensor* x = plain(a[0]);
    Linear l;
    if (!x || !is_16bit(x->scalar_type()) || (x->dim() != 2 && x->dim() != 3) || !x->is_contiguous() ||
        !parse_linear(a + 1, x->scalar_type(), x->size(-1), l) || recorded(*x, l))
        Py_RETURN_NONE;
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        y = linear(*x, l);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// module_call(module, x) -> y or None: the call of a prepared NanoQuantLinear that nn.Module.__call__ would pass to its forward and forward
// to linear_forward, as one function.  None for everything that nn.Module would not have passed on unchanged and unseen: hooks (the
// module's or global ones), a replaced forward, nn.Module's way of calling replaced (tools do that to see every module's calls), tracing, a
// Python profiler or debugger, a subclass, or not a plain call.
PyObject* py_module_call(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 2, "module_call takes a module and its argument");
    static PyObject* const key[] = {PyUnicode_InternFromString("_forward_hooks"), PyUnicode_InternFromString("_forward_pre_hooks"),
                                    PyUnicode_InternFromString("_backward_hooks"), PyUnicode_InternFromString("_backward_pre_hooks"),
                                    PyUnicode_InternFromString("_parameters"), PyUnicode_InternFromString("forward"),
                                    PyUnicode_InternFromString("_compiled_call_impl"), PyUnicode_InternFromString("do_kernel_inference"),
                                    PyUnicode_InternFromString("kernel_type"), PyUnicode_InternFromString("V_int8"),
                                    PyUnicode_InternFromString("U_int8"), PyUnicode_InternFromString("rank"),
                                    PyUnicode_InternFromString("_call_impl"), PyUnicode_InternFromString("__call__")};
    static PyObject* const scale[2][3] = {{PyUnicode_InternFromString("scale_pre"), PyUnicode_InternFromString("scale_mid"), PyUnicode_InternFromString("scale_post")},
                                          {PyUnicode_InternFromString("s1"), PyUnicode_InternFromString("s2"), PyUnicode_InternFromString("s3")}};
    static PyObject* const bias_key = PyUnicode_InternFromString("bias");
    auto get = [](PyObject* dict, PyObject* k) { return PyDict_GetItemWithError(dict, k); };    // borrowed
    const ModuleClass& cls = g_module_class;
    if (!cls.type || Py_TYPE(a[0]) != cls.type || _PyType_Lookup(cls.type, key[5]) != cls.forward ||
        _PyType_Lookup(cls.type, key[12]) != cls.call_impl || _PyType_Lookup(cls.base, key[13]) != cls.call)
        Py_RETURN_NONE;
    if (!exact_plain(a[1])) Py_RETURN_NONE;
    // A profiler that records modules knows them by the frame of nn.Module.__call__; a debugger steps into forward.
    const PyThreadState* const thread = PyThreadState_Get();
    if (thread->c_profilefunc || thread->c_tracefunc) Py_RETURN_NONE;
    THPObjectPtr module_dict(PyObject_GenericGetDict(a[0], nullptr));
    if (!module_dict) return nullptr;
    PyObject* const dict = module_dict.get();
    for (PyObject* hooks : cls.global_hooks)
        if (PyDict_Size(hooks) != 0) Py_RETURN_NONE;
    for (int i = 0; i < 4; ++i) {
        PyObject* hooks = get(dict, key[i]);
        if (hooks && PyDict_Size(hooks) != 0) Py_RETURN_NONE;
    }
    PyObject* params = get(dict, key[4]);
    PyObject* compiled = get(dict, key[6]);
    if (!params || !PyDict_Check(params) || get(dict, key[5]) || get(dict, key[12]) || (compiled && compiled != Py_None) || get(dict, key[7]) != Py_True) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    PyObject* type = get(dict, key[8]);
    if (!type || !PyUnicode_Check(type)) Py_RETURN_NONE;
    PyObject* const* s = scale[PyUnicode_CompareWithASCIIString(type, "gemv") == 0 ? 0 : 1];
    auto or_none = [](PyObject* o) { return o ? o : Py_None; };
    PyObject* const operands[7] = {get(params, s[0]), get(dict, key[9]), or_none(get(params, s[1])), get(dict, key[10]), get(params, s[2]),
                                   get(dict, key[11]), or_none(get(params, bias_key))};
    if (PyErr_Occurred()) return nullptr;
    // The call's own references, kept until the launch is enqueued: the GIL is released below, and another thread (or Python code that
    // growing the scratch runs) may replace an operand of the module meanwhile.
    THPObjectPtr held[7];
    for (int i = 0; i < 7; ++i) {
        if (!operands[i]) Py_RETURN_NONE;
        held[i] = Py_NewRef(operands[i]);
    }
    const Tensor* x = plain(a[1]);
    Linear l;
    if (!x || !is_16bit(x->scalar_type()) || (x->dim() != 2 && x->dim() != 3) || !x->is_contiguous() ||
        !parse_linear(operands, x->scalar_type(), x->size(-1), l) || recorded(*x, l))
        Py_RETURN_NONE;
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        y = linear(*x, l);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// set_module_class(class, its forward, nn.Module, nn.Module.__call__, nn.Module._call_impl, [dictionaries of hooks on every module])
PyObject* py_set_module_class(PyObject*, PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *type, *forward, *base, *call, *call_impl, *hooks;
    if (!PyArg_ParseTuple(args, "O!OO!OOO!", &PyType_Type, &type, &forward, &PyType_Type, &base, &call, &call_impl, &PyList_Type, &hooks)) return nullptr;
    ModuleClass c;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(hooks); ++i) {
        TORCH_CHECK(PyDict_Check(PyList_GET_ITEM(hooks, i)), "a list of dictionaries");
        c.global_hooks.push_back(PyList_GET_ITEM(hooks, i));
    }
    c.type = reinterpret_cast<PyTypeObject*>(type);
    c.base = reinterpret_cast<PyTypeObject*>(base);
    c.forward = forward;
    c.call = call;
    c.call_impl = call_impl;
    for (PyObject* o : {type, forward, base, call, call_impl}) Py_INCREF(o);     // (for the life of the process)
    for (PyObject* o : c.global_hooks) Py_INCREF(o);
    g_module_class = std::move(c);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// group_forward(x | [x...], [(s_in, v_tiles, s_mid, u_tiles, s_out, rank, bias)...], residuals | None) -> [y...] or None.
// The outputs lie side by side in one [T, sum(M)] buffer.
PyObject* py_group_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 3, "group_forward takes 3 arguments");
    if (!PyList_CheckExact(a[1])) Py_RETURN_NONE;
    const Py_ssize_t count = PyList_GET_SIZE(a[1]);
    const bool many = PyList_CheckExact(a[0]), res = a[2] != Py_None;
    if (count < 1 || count > kMaxLinears || (many && PyList_GET_SIZE(a[0]) != count) ||
        (res && (!PyList_CheckExact(a[2]) || PyList_GET_SIZE(a[2]) != count)))
        Py_RETURN_NONE;
    nq_linear_desc d[kMaxLinears];
    Linear l[kMaxLinears];
    const Tensor* x[kMaxLinears];
    int64_t width = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject* xo = many ? PyList_GET_ITEM(a[0], i) : a[0];
        if (!exact_plain(xo)) Py_RETURN_NONE;
        x[i] = plain(xo);
        PyObject* t = PyList_GET_ITEM(a[1], i);
        if (!x[i] || !is_16bit(x[i]->scalar_type()) || x[i]->scalar_type() != x[0]->scalar_type() || x[i]->dim() < 2 ||
            !x[i]->is_contiguous() || !PyTuple_CheckExact(t) || PyTuple_GET_SIZE(t) != 7 ||
            !parse_linear(&PyTuple_GET_ITEM(t, 0), x[0]->scalar_type(), x[i]->size(-1), l[i]) ||
            x[i]->sizes().slice(0, x[i]->dim() - 1) != x[0]->sizes().slice(0, x[0]->dim() - 1))
            Py_RETURN_NONE;
        width += l[i].s_out->size(0);
    }
    const int64_t T = x[0]->size(-1) ? x[0]->numel() / x[0]->size(-1) : 0;
    if (T == 0) Py_RETURN_NONE;
    const Tensor* r[kMaxLinears] = {};
    for (Py_ssize_t i = 0; res && i < count; ++i) {
        PyObject* ro = PyList_GET_ITEM(a[2], i);
        if (ro == Py_None) continue;
        r[i] = exact_plain(ro) ? plain(ro) : nullptr;
        const int64_t M = l[i].s_out->size(0);
        if (!r[i] || r[i]->scalar_type() != x[0]->scalar_type() || !r[i]->is_contiguous() || r[i]->size(-1) != M || r[i]->numel() != T * M)
            Py_RETURN_NONE;
    }
    Tensor out = new_output({T, width}, *x[0]);
    char* base = static_cast<char*>(out.mutable_data_ptr());
    int64_t col = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
        const int64_t N = x[i]->size(-1), M = l[i].s_out->size(0);
        describe(d[i], l[i], x[i]->const_data_ptr(), N, N, base + 2 * col, width);
        if (r[i]) {
            d[i].residual = r[i]->const_data_ptr();
            d[i].ldr = M;
        }
        col += M;
    }
    {
        pybind11::gil_scoped_release no_gil;
        launch(d, (int)count, T, dtype_id(out.scalar_type()), out.get_device());
    }
    THPObjectPtr list(PyList_New(count));
    if (!list) return nullptr;
    // The outputs do not overlap and their buffer is nobody else's, so they need none of a view's bookkeeping.
    at::AutoDispatchBelowADInplaceOrView below;
    col = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
        // [..., M] column view with the leading dimensions of x: tokens are `width` elements apart
        c10::SmallVector<int64_t, 4> shape(x[0]->sizes().begin(), x[0]->sizes().end());
        c10::SmallVector<int64_t, 4> strides(shape.size());
        shape.back() = l[i].s_out->size(0);
        strides.back() = 1;
        int64_t step = width;
        for (int k = (int)shape.size() - 2; k >= 0; --k) {
            strides[k] = step;
            step *= shape[k];
        }
        PyObject* y = THPVariable_Wrap(out.as_strided(shape, strides, col));
        if (!y) return nullptr;
        PyList_SET_ITEM(list.get(), i, y);
        col += shape.back();
    }
    return list.release();
    END_HANDLE_TH_ERRORS
}

bool dense_gemv_takes(const Tensor& x, const Tensor& w, const Tensor* b) {
    return is_16bit(x.scalar_type()) && w.scalar_type() == x.scalar_type() && w.dim() == 2 && w.stride(1) == 1 && x.is_contiguous() && x.dim() >= 1 &&
           x.size(-1) == w.size(1) && x.numel() > 0 && (!b || (b->scalar_type() == x.scalar_type() && b->is_contiguous() && b->numel() == w.size(0)));
}
Tensor dense_gemv_launch(const Tensor& x, const Tensor& w, const Tensor* b) {
    const int64_t V = w.size(0), N = w.size(1), T = x.numel() / N;
    c10::SmallVector<int64_t, 4> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = V;
    Tensor y = new_output(shape, x);
    const int dev = x.get_device();
    OnDevice on(dev);
    const int st = nq_dense_gemv_fwd(x.const_data_ptr(), w.const_data_ptr(), b ? b->const_data_ptr() : nullptr,
                                     y.mutable_data_ptr(), (int)T, (int)N, (int)V, w.stride(0), V, dtype_id(x.scalar_type()),
                                     c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
    if (st < 0) fail(st, "nq_dense_gemv_fwd");
    return y;
}
// dense_gemv_forward(x, weight, bias | None) -> y or None
PyObject* py_dense_gemv_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 3, "dense_gemv_forward takes 3 arguments");
    if (!exact_plain(a[0])) Py_RETURN_NONE;
    const Tensor *x = plain(a[0]), *w = plain(a[1]), *b = a[2] == Py_None ? nullptr : plain(a[2]);
    if (!x || !w || (a[2] != Py_None && !b) || !dense_gemv_takes(*x, *w, b)) Py_RETURN_NONE;
    return THPVariable_Wrap(dense_gemv_launch(*x, *w, b));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------
// behind the last decoder layer: norms, the head in 8 bits, the loss over the head
// ---------------------------------------------------------------------------------------------------------------
// A tensor as rows of its last dimension, `ld` elements apart; false: its leading dimensions are not evenly spaced, or the last is not dense.
bool as_rows(const Tensor& t, int64_t& rows, int64_t& ld) {
    const int64_t n = t.dim();
    if (n < 1) return false;
    const int64_t cols = t.size(n - 1);
    if (cols > 1 && t.stride(n - 1) != 1) return false;
    rows = 1;
    ld = cols;
    int64_t next = -1;      // stride that the next outer dimension has to have
    for (int64_t k = n - 2; k >= 0; --k) {
        if (t.size(k) == 1) continue;
        if (next < 0) ld = t.stride(k);
        else if (t.stride(k) != next) return false;
        next = t.stride(k) * t.size(k);
        rows *= t.size(k);
    }
    return ld >= 0;
}
Tensor dense_rows(const Tensor& t) {
    int64_t rows, ld;
    Tensor u = t.resolve_neg();
    return as_rows(u, rows, ld) ? u : u.contiguous();
}
nq_stream_t stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
// A backward pass runs on a thread of autograd's: it keeps the scratch that the forward call's thread ran on, alive too, and runs on it.
Tensor thread_scratch() {
    if (!t_override.ptr) return Tensor();
    pybind11::gil_scoped_acquire gil;
    THPObjectPtr r(call_python(g_thread_scratch, PyTuple_New(0)));
    return THPVariable_Check(r.get()) ? THPVariable_Unpack(r.get()) : Tensor();
}
struct OnScratch {
    explicit OnScratch(const Tensor& t) : before(t_override) {
        t_override = t.defined() ? Scratch{t.data_ptr(), (size_t)t.numel()} : Scratch{};
    }
    ~OnScratch() { t_override = before; }
    Scratch before;
};
// The header of the device's scratch, whose status word an expired wait sets.
void* status_header(int dev) {
    constexpr size_t kHeader = 256;
    Scratch s = scratch_of(dev);
    if (!s.ptr || s.bytes < kHeader) {
        grow_scratch(dev, kHeader);
        s = scratch_of(dev);
    }
    return s.ptr;
}
Tensor new_bytes(int64_t n, const Tensor& like) { return new_output({n}, like, at::kByte); }

bool capturing(int dev) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(), &st) == cudaSuccess && st != cudaStreamCaptureStatusNone;
}
// A leaf's gradient is accumulated on the stream on which its accumulator was made.  While another graph holds an accumulator made on the
// default stream, a captured backward pass would have that stream wait for the capture, which it cannot, and which ends the process: refuse the
// call instead, wherever behind its inputs such a leaf is.  (Other streams join the capture and leave it again.)
void check_capture(int dev, std::initializer_list<const Tensor*> inputs) {
    if (!capturing(dev)) return;
    using torch::autograd::Node;
    const c10::Stream first = c10::cuda::getDefaultCUDAStream((c10::DeviceIndex)dev).unwrap();
    std::vector<Node*> left;
    std::unordered_set<Node*> seen;
    auto visit = [&](Node* n) {
        if (n && seen.insert(n).second) left.push_back(n);
    };
    std::shared_ptr<Node> held[3];          // (accumulators live only as long as a graph holds them)
    size_t n = 0;
    for (const Tensor* t : inputs) {
        if (!t || !t->defined() || !t->requires_grad()) continue;
        if (t->grad_fn()) held[n] = t->grad_fn();
        else held[n] = torch::autograd::impl::try_get_grad_accumulator(*t);
        visit(held[n++].get());
    }
    while (!left.empty()) {
        Node* node = left.back();
        left.pop_back();
        if (dynamic_cast<torch::autograd::AccumulateGrad*>(node))
            TORCH_CHECK(!node->stream() || *node->stream() != first,
                        "a leaf of this captured call is held by an autograd graph made on the default stream: its gradient cannot be captured; "
                        "release that graph first, or make it on another stream");
        for (const auto& e : node->next_edges()) visit(e.function.get());
    }
}

// A call that forward-mode differentiation follows: an output without a tangent would say that the tangent is zero.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs)
        if (t) TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

struct NormArgs {
    int64_t N;
    double eps;
    bool center;
};
Tensor norm_launch(const Tensor& x, const Tensor* w, const Tensor* b, const NormArgs& a, Tensor* stats) {
    int64_t rows, ld;
    as_rows(x, rows, ld);
    Tensor y = new_output(x.sizes(), x);
    if (stats) *stats = new_output({rows, 2}, x, at::kFloat);
    if (rows * a.N == 0) return y;
    const int dev = x.get_device(), dt = dtype_id(x.scalar_type());
    OnDevice on(dev);
    const int st = nq_norm_fwd(x.const_data_ptr(), w ? w->const_data_ptr() : nullptr, b ? b->const_data_ptr() : nullptr, y.mutable_data_ptr(),
                               stats ? static_cast<float*>(stats->mutable_data_ptr()) : nullptr, rows, a.N, ld, a.N, (float)a.eps, a.center, dt,
                               w && w->scalar_type() == at::kFloat ? (int)NQ_F32 : dt, stream_of(dev));
    if (st < 0) fail(st, "nq_norm_fwd");
    return y;
}
// (dx, dw, db), undefined where not wanted
std::array<Tensor, 3> norm_gradients(const Tensor& grad, const Tensor& x, const Tensor& w, const Tensor& stats, bool center, std::array<bool, 3> want) {
    int64_t rows, ldx, dy_rows, lddy;
    as_rows(x, rows, ldx);
    const int64_t N = x.size(-1);
    std::array<Tensor, 3> d;
    if (want[0]) d[0] = new_output(x.sizes(), x);
    for (int i = 1; i < 3; ++i)
        if (want[i]) d[i] = new_output({N}, w, w.scalar_type());
    if (rows * N == 0) {
        for (int i = 1; i < 3; ++i)
            if (want[i]) d[i].zero_();
        return d;
    }
    const Tensor dy = dense_rows(grad);
    as_rows(dy, dy_rows, lddy);
    const int dev = x.get_device(), dt = dtype_id(x.scalar_type());
    OnDevice on(dev);
    const size_t bytes = nq_norm_bwd_scratch_bytes(rows, N);
    const Tensor scratch = want[1] || want[2] ? new_bytes((int64_t)bytes, x) : Tensor();
    auto ptr = [](Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
    const int st = nq_norm_bwd(dy.const_data_ptr(), x.const_data_ptr(), w.defined() ? w.const_data_ptr() : nullptr,
                               static_cast<const float*>(stats.const_data_ptr()), ptr(d[0]), ptr(d[1]), ptr(d[2]),
                               scratch.defined() ? scratch.mutable_data_ptr() : nullptr, scratch.defined() ? bytes : 0, rows, N, lddy, ldx, N,
                               center, dt, w.defined() && w.scalar_type() == at::kFloat ? (int)NQ_F32 : dt, stream_of(dev));
    if (st < 0) fail(st, "nq_norm_bwd");
    return d;
}
struct NormFunction : torch::autograd::Function<NormFunction> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t N, double eps, bool center) {
        Tensor stats;
        const NormArgs a{N, eps, center};
        Tensor y = norm_launch(x, w ? &*w : nullptr, b ? &*b : nullptr, a, &stats);
        ctx->save_for_backward({x, w ? *w : Tensor(), stats});
        ctx->saved_data["center"] = center;
        ctx->saved_data["bias"] = b.has_value();
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "the norms are differentiable once");
        const auto saved = ctx->get_saved_variables();
        const Tensor& w = saved[1];
        std::array<Tensor, 3> d;
        if (grads[0].defined())
            d = norm_gradients(grads[0], saved[0], w, saved[2], ctx->saved_data["center"].toBool(),
                               {ctx->needs_input_grad(0), w.defined() && ctx->needs_input_grad(1), ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2)});
        return {d[0], d[1], d[2], Tensor(), Tensor(), Tensor()};
    }
};
bool norm_takes(const Tensor& x, const Tensor* w, const Tensor* b) {
    int64_t rows, ld;
    if ((b && !w) || !is_16bit(x.scalar_type()) || !as_rows(x, rows, ld)) return false;
    for (const Tensor* t : {w, b})
        if (t && ((t->scalar_type() != x.scalar_type() && t->scalar_type() != at::kFloat) || t->scalar_type() != w->scalar_type() || t->dim() != 1 ||
                  t->size(0) != x.size(-1) || !t->is_contiguous() || t->get_device() != x.get_device()))
            return false;
    return true;
}

// norm(x, weight | None, bias | None, eps, center) -> y or None
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 5, "norm takes 5 arguments");
    if (!exact_plain(a[0])) Py_RETURN_NONE;
    const Tensor *x = plain(a[0]), *w = a[1] == Py_None ? nullptr : plain(a[1]), *b = a[2] == Py_None ? nullptr : plain(a[2]);
    if (!x || (a[1] != Py_None && !w) || (a[2] != Py_None && !b) || !norm_takes(*x, w, b)) Py_RETURN_NONE;
    const int64_t N = x->size(-1);
    const double eps = PyFloat_AsDouble(a[3]);
    const int center = PyObject_IsTrue(a[4]);
    if (PyErr_Occurred()) return nullptr;
    refuse_tangents(center ? "layer_norm" : "rms_norm", {x, w, b});
    Tensor y;
    if (at::GradMode::is_enabled() && (x->requires_grad() || (w && w->requires_grad()) || (b && b->requires_grad()))) {
        check_capture(x->get_device(), {x, w, b});
        y = NormFunction::apply(*x, w ? OptTensor(*w) : std::nullopt, b ? OptTensor(*b) : std::nullopt, N, eps, center != 0);
    } else {
        y = norm_launch(*x, w, b, NormArgs{N, eps, center != 0}, nullptr);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

bool quantize_takes(const Tensor& x) {
    int64_t rows, ld;
    return is_16bit(x.scalar_type()) && x.dim() >= 1 && x.size(-1) > 0 && as_rows(x, rows, ld);
}
// (q, scale); rows of q start at multiples of 16 bytes
std::tuple<Tensor, Tensor> quantize_launch(const Tensor& x) {
    int64_t rows, ld;
    as_rows(x, rows, ld);
    const int64_t N = x.size(-1), ldq = (N + 15) / 16 * 16;
    c10::SmallVector<int64_t, 4> shape(x.sizes().begin(), x.sizes().end()), strides(shape.size()), lead(shape.begin(), shape.end() - 1);
    strides.back() = 1;
    int64_t step = ldq;
    for (int k = (int)shape.size() - 2; k >= 0; --k) {
        strides[k] = step;
        step *= shape[k];
    }
    Tensor buf = new_output({rows, ldq}, x, at::kChar), scale = new_output(lead, x, at::kFloat);
    if (rows > 0) {
        const int dev = x.get_device();
        OnDevice on(dev);
        const int st = nq_quantize_rows_s8(x.const_data_ptr(), static_cast<int8_t*>(buf.mutable_data_ptr()), static_cast<float*>(scale.mutable_data_ptr()),
                                           rows, N, ld, ldq, dtype_id(x.scalar_type()), stream_of(dev));
        if (st < 0) fail(st, "nq_quantize_rows_s8");
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return {buf.as_strided(shape, strides, 0), scale};
}
// quantize_rows(x) -> (q, scale) or None
PyObject* py_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 1, "quantize_rows takes 1 argument");
    if (!exact_plain(a[0])) Py_RETURN_NONE;
    const Tensor* x = plain(a[0]);
    if (!x || !quantize_takes(*x)) Py_RETURN_NONE;
    const auto [buf, scale] = quantize_launch(*x);
    PyObject* q = THPVariable_Wrap(buf);
    PyObject* s = q ? THPVariable_Wrap(scale) : nullptr;
    return s ? Py_BuildValue("(NN)", q, s) : nullptr;
    END_HANDLE_TH_ERRORS
}

bool int8_takes(const Tensor& x, const Tensor& w, const Tensor& ws, const Tensor* b) {
    int64_t T, ldx;
    if (!is_16bit(x.scalar_type()) || w.scalar_type() != at::kChar || ws.scalar_type() != at::kFloat || w.dim() != 2 || w.size(0) == 0 || w.size(1) == 0 ||
        w.stride(1) != 1 || !as_rows(x, T, ldx) || x.size(-1) != w.size(1) || ws.dim() != 1 || ws.size(0) != w.size(0) || !ws.is_contiguous())
        return false;
    const int64_t N = w.size(1), V = w.size(0), ldw = w.stride(0);
    if (b && (b->scalar_type() != x.scalar_type() || b->dim() != 1 || !b->is_contiguous() || b->size(0) != V)) return false;
    // (one channel: its row stride means nothing)
    if ((V > 1 && (ldw < N || ldw % 16 != 0)) || (reinterpret_cast<uintptr_t>(w.const_data_ptr()) & 15) || (reinterpret_cast<uintptr_t>(ws.const_data_ptr()) & 15))
        return false;
    const int dev = x.get_device();
    return w.get_device() == dev && ws.get_device() == dev && (!b || b->get_device() == dev);
}
Tensor int8_launch(const Tensor& x, const Tensor& w, const Tensor& ws, const Tensor* b) {
    int64_t T, ldx;
    as_rows(x, T, ldx);
    const int64_t N = w.size(1), V = w.size(0);
    const int dev = x.get_device();
    c10::SmallVector<int64_t, 4> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = V;
    Tensor y = new_output(shape, x);
    if (T == 0) return y;
    OnDevice on(dev);
    void* status = status_header(dev);
    const size_t bytes = nq_int8_linear_scratch_bytes(T, N);
    const Tensor scratch = bytes ? new_bytes((int64_t)bytes, x) : Tensor();
    const int st = nq_int8_linear_fwd(x.const_data_ptr(), static_cast<const int8_t*>(w.const_data_ptr()), static_cast<const float*>(ws.const_data_ptr()),
                                      b ? b->const_data_ptr() : nullptr, y.mutable_data_ptr(), bytes ? scratch.mutable_data_ptr() : nullptr, bytes, status, T, N, V, ldx,
                                      V > 1 ? w.stride(0) : (N + 15) / 16 * 16, V, dtype_id(x.scalar_type()), stream_of(dev));
    if (st < 0) fail(st, "nq_int8_linear_fwd");
    return y;
}
// int8_linear_forward(x, weight, weight_scale, bias | None) -> y or None
PyObject* py_int8_linear_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 4, "int8_linear_forward takes 4 arguments");
    if (!exact_plain(a[0])) Py_RETURN_NONE;
    const Tensor *x = plain(a[0]), *w = plain(a[1]), *ws = plain(a[2]), *b = a[3] == Py_None ? nullptr : plain(a[3]);
    if (!x || !w || !ws || (a[3] != Py_None && !b) || !int8_takes(*x, *w, *ws, b)) Py_RETURN_NONE;
    return THPVariable_Wrap(int8_launch(*x, *w, *ws, b));
    END_HANDLE_TH_ERRORS
}

struct LossArgs {
    int64_t ignore;
    int reduction;
};
// Rows of a matrix that a stride means nothing for are taken as dense.
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8; }
// `lse`, `count`: what the backward pass needs.
Tensor loss_launch(const Tensor& h, const Tensor& w, const Tensor& targets, const LossArgs& a, Tensor& lse, Tensor& count) {
    const int64_t T = h.size(0), N = h.size(1), V = w.size(0);
    const bool none = a.reduction == NQ_REDUCE_NONE;
    lse = new_output({T}, h, at::kFloat);
    count = new_output({1}, h, at::kFloat);
    if (T == 0 && !none)
        return at::full({}, a.reduction == NQ_REDUCE_MEAN ? std::numeric_limits<double>::quiet_NaN() : 0.0, lse.options());
    Tensor loss = none ? new_output({T}, h, at::kFloat) : new_output({}, h, at::kFloat);
    if (T == 0) return loss;
    const int dev = h.get_device();
    OnDevice on(dev);
    void* status = status_header(dev);
    const size_t bytes = nq_linear_ce_fwd_scratch_bytes(T, N, V);
    const Tensor scratch = new_bytes((int64_t)bytes, h);
    const int st = nq_linear_ce_fwd(h.const_data_ptr(), w.const_data_ptr(), targets.const_data_ptr(), targets.scalar_type() == at::kLong ? 64 : 32, a.ignore,
                                    static_cast<float*>(loss.mutable_data_ptr()), static_cast<float*>(lse.mutable_data_ptr()),
                                    static_cast<float*>(count.mutable_data_ptr()), scratch.mutable_data_ptr(), bytes, status, T, N, V, row_stride(h),
                                    row_stride(w), a.reduction, dtype_id(h.scalar_type()), stream_of(dev));
    if (st < 0) fail(st, "nq_linear_ce_fwd");
    return loss;
}
// (dh, dw), undefined where not wanted
std::array<Tensor, 2> loss_gradients(const Tensor& grad, const Tensor& h, const Tensor& w, const Tensor& targets, const Tensor& lse, const Tensor& count, const LossArgs& a,
                                     std::array<bool, 2> want) {
    const int64_t T = h.size(0), N = h.size(1), V = w.size(0);
    std::array<Tensor, 2> d;
    if (want[0]) d[0] = new_output({T, N}, h);
    if (want[1]) d[1] = T == 0 ? at::zeros({V, N}, w.options()) : new_output({V, N}, w);
    if (T == 0 || !(want[0] || want[1])) return d;
    const Tensor g = grad.resolve_neg();
    const int dev = h.get_device();
    OnDevice on(dev);
    void* status = status_header(dev);
    const size_t bytes = nq_linear_ce_bwd_scratch_bytes(T, N, V);
    const Tensor scratch = new_bytes((int64_t)bytes, h);
    const int st = nq_linear_ce_bwd(h.const_data_ptr(), w.const_data_ptr(), targets.const_data_ptr(), targets.scalar_type() == at::kLong ? 64 : 32, a.ignore,
                                    static_cast<const float*>(lse.const_data_ptr()), static_cast<const float*>(count.const_data_ptr()),
                                    static_cast<const float*>(g.const_data_ptr()), g.dim() == 1 ? g.stride(0) : 0, want[0] ? d[0].mutable_data_ptr() : nullptr,
                                    want[1] ? d[1].mutable_data_ptr() : nullptr, scratch.mutable_data_ptr(), bytes, status, T, N, V, row_stride(h), row_stride(w), N, N,
                                    a.reduction, dtype_id(h.scalar_type()), stream_of(dev));
    if (st < 0) fail(st, "nq_linear_ce_bwd");
    return d;
}
struct LossFunction : torch::autograd::Function<LossFunction> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& targets, int64_t ignore, int64_t reduction) {
        Tensor lse, count;
        Tensor loss = loss_launch(h, w, targets, LossArgs{ignore, (int)reduction}, lse, count);
        ctx->save_for_backward({h, w, targets, lse, count});
        if (const Tensor own = thread_scratch(); own.defined()) ctx->saved_data["scratch"] = own;
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "linear_cross_entropy is differentiable once");
        const auto saved = ctx->get_saved_variables();
        std::array<Tensor, 2> d;
        if (grads[0].defined()) {
            const auto own = ctx->saved_data.find("scratch");
            const OnScratch on_scratch(own == ctx->saved_data.end() ? Tensor() : own->second.toTensor());
            d = loss_gradients(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4],
                               LossArgs{ctx->saved_data["ignore"].toInt(), (int)ctx->saved_data["reduction"].toInt()}, {ctx->needs_input_grad(0), ctx->needs_input_grad(1)});
        }
        return {d[0], d[1], Tensor(), Tensor(), Tensor()};
    }
};
bool loss_takes(const Tensor& h, const Tensor& w, const Tensor& t) {
    if (!is_16bit(h.scalar_type()) || w.scalar_type() != h.scalar_type() || h.dim() != 2 || w.dim() != 2 || t.dim() != 1 ||
        (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) || h.size(1) != w.size(1) || t.size(0) != h.size(0) || !t.is_contiguous() ||
        h.stride(1) != 1 || w.stride(1) != 1 || w.get_device() != h.get_device() || t.get_device() != h.get_device())
        return false;
    for (const Tensor* m : {&h, &w})
        if ((reinterpret_cast<uintptr_t>(m->const_data_ptr()) & 15) || row_stride(*m) % 8 != 0 || row_stride(*m) < m->size(1)) return false;
    return true;
}

// linear_cross_entropy(h, weight, targets, ignore_index, reduction) -> loss or None
PyObject* py_linear_cross_entropy(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 5, "linear_cross_entropy takes 5 arguments");
    if (!exact_plain(a[0])) Py_RETURN_NONE;
    const Tensor *h = plain(a[0]), *w = plain(a[1]), *t = plain(a[2]);
    if (!h || !w || !t || !loss_takes(*h, *w, *t)) Py_RETURN_NONE;
    const int64_t ignore = PyLong_AsLongLong(a[3]), reduction = PyLong_AsLongLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    refuse_tangents("linear_cross_entropy", {h, w});
    Tensor loss;
    if (at::GradMode::is_enabled() && (h->requires_grad() || w->requires_grad())) {
        check_capture(h->get_device(), {h, w});
        loss = LossFunction::apply(*h, *w, *t, ignore, reduction);
    } else {
        Tensor lse, count;
        loss = loss_launch(*h, *w, *t, LossArgs{ignore, (int)reduction}, lse, count);
    }
    return THPVariable_Wrap(loss);
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------------------------
// between the projections of a decoder layer: head norms and rotation, the paged cache, attention
// ---------------------------------------------------------------------------------------------------------------
// Heads [..., heads, D] as the kernels read them: 16-bit elements, D a multiple of 8 and dense, heads and tokens (evenly spaced) multiples of 8 elements apart,
// a 16-byte boundary.  False: not so.
struct Heads {
    int64_t tokens, heads, D, token, head;
};
bool as_heads(const Tensor& t, Heads& h) {
    const int64_t n = t.dim();
    if (n < 2 || !is_16bit(t.scalar_type())) return false;
    h.D = t.size(n - 1);
    h.heads = t.size(n - 2);
    if (h.D == 0 || h.D % 8 != 0 || h.D > nq_head_max_columns() || h.heads == 0 || t.stride(n - 1) != 1 || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15)) return false;
    h.head = h.heads > 1 ? t.stride(n - 2) : h.D;
    h.tokens = 1;
    h.token = h.head * h.heads;
    int64_t next = -1;
    for (int64_t k = n - 3; k >= 0; --k) {
        if (t.size(k) == 1) continue;
        if (next < 0) h.token = t.stride(k);
        else if (t.stride(k) != next) return false;
        next = t.stride(k) * t.size(k);
        h.tokens *= t.size(k);
    }
    return h.head >= h.D && h.head % 8 == 0 && h.token >= h.D && h.token % 8 == 0;
}
bool is_index(const Tensor& t, at::ScalarType type, int64_t dim, int dev) {
    return t.scalar_type() == type && t.dim() == dim && t.get_device() == dev && (dim == 0 || t.size(dim - 1) <= 1 || t.stride(dim - 1) == 1);
}
// A cache [pages, page_size, heads, D], and the table that leads to its pages.  (A table of no sequences is one for a call without tokens.)
bool cache_takes(const Tensor& k, const Tensor& v, const Tensor& table, const Heads& h, at::ScalarType type, int dev, bool no_tokens) {
    if (k.dim() != 4 || v.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != type || v.scalar_type() != type || k.get_device() != dev || v.get_device() != dev ||
        k.size(2) != h.heads || k.size(3) != h.D || k.numel() == 0 || !is_index(table, at::kInt, 2, dev) ||
        (table.numel() == 0 && !(no_tokens && table.size(0) == 0)))
        return false;
    const int64_t page = k.size(1);
    if (page < 8 || (page & (page - 1)) != 0 || (table.size(0) > 1 && table.stride(0) < table.size(1))) return false;
    for (const Tensor* t : {&k, &v}) {
        if (t->stride(3) != 1 || (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15)) return false;
        for (int i = 0; i < 3; ++i)
            if (t->size(i) > 1 && (t->stride(i) % 8 != 0 || t->stride(i) < h.D)) return false;
    }
    return true;
}
int64_t cache_stride(const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : t.size(3); }
const void* data(const Tensor* t) { return t ? t->const_data_ptr() : nullptr; }

struct HeadsArgs {
    const Tensor *q, *k, *v, *k_cache, *v_cache, *table, *positions, *sequences, *inv_freq, *wq, *wk;
    double eps, scaling;
    bool interleaved;
};
bool heads_takes(const HeadsArgs& a) {
    Heads q{}, k{}, v{};
    const Tensor& first = a.q ? *a.q : *a.k;
    const int dev = first.get_device();
    const at::ScalarType type = first.scalar_type();
    if (!as_heads(*a.k, k) || (a.q && !as_heads(*a.q, q)) || (a.v && !as_heads(*a.v, v))) return false;
    for (const Tensor* t : {a.q, a.k, a.v})
        if (t && (t->scalar_type() != type || t->get_device() != dev || t->size(-1) != k.D)) return false;
    const Tensor& p = *a.positions;
    if (p.get_device() != dev || (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong) || !p.is_contiguous()) return false;
    for (const Tensor* t : {a.q, a.k, a.v})
        if (t && t->sizes().slice(0, t->dim() - 2) != p.sizes()) return false;
    if (a.inv_freq && (a.inv_freq->scalar_type() != at::kFloat || a.inv_freq->dim() != 1 || !a.inv_freq->is_contiguous() || a.inv_freq->get_device() != dev || 2 * a.inv_freq->size(0) > k.D))
        return false;
    if (a.wq && !a.q) return false;
    const Tensor* any = a.wq ? a.wq : a.wk;
    for (const Tensor* w : {a.wq, a.wk})
        if (w && ((w->scalar_type() != type && w->scalar_type() != at::kFloat) || w->scalar_type() != any->scalar_type() || w->dim() != 1 || w->size(0) != k.D || !w->is_contiguous() ||
                  w->get_device() != dev || (reinterpret_cast<uintptr_t>(w->const_data_ptr()) & 15)))
            return false;
    if (!a.k_cache) return true;
    if (v.heads != k.heads || !cache_takes(*a.k_cache, *a.v_cache, *a.table, k, type, dev, p.numel() == 0)) return false;
    return a.sequences ? a.sequences->sizes() == p.sizes() && a.sequences->scalar_type() == at::kInt && a.sequences->is_contiguous() && a.sequences->get_device() == dev : true;
}
// (q', k'), undefined where there is none
std::array<Tensor, 2> heads_launch(const HeadsArgs& a) {
    Heads q{}, k{}, v{};
    as_heads(*a.k, k);
    if (a.q) as_heads(*a.q, q);
    if (a.v) as_heads(*a.v, v);
    std::array<Tensor, 2> out;
    if (a.q) out[0] = new_output(a.q->sizes(), *a.q);
    if (!a.k_cache) out[1] = new_output(a.k->sizes(), *a.k);
    if (a.positions->numel() == 0) return out;
    nq_heads_desc d{};
    d.q = data(a.q); d.k = data(a.k); d.v = data(a.v);
    d.q_out = a.q ? out[0].mutable_data_ptr() : nullptr;
    d.k_out = a.k_cache ? nullptr : out[1].mutable_data_ptr();
    d.positions = data(a.positions);
    d.inv_freq = a.inv_freq && a.inv_freq->numel() ? static_cast<const float*>(data(a.inv_freq)) : nullptr;
    d.q_weight = data(a.wq); d.k_weight = data(a.wk);
    d.q_token = q.token; d.q_head = q.head; d.k_token = k.token; d.k_head = k.head; d.v_token = v.token; d.v_head = v.head;
    d.T = a.positions->numel();
    d.position_bits = a.positions->scalar_type() == at::kLong ? 64 : 32;
    d.q_heads = (int)q.heads; d.k_heads = (int)k.heads; d.D = (int)k.D;
    d.R = a.inv_freq ? 2 * (int)a.inv_freq->size(0) : 0;
    d.interleaved = a.interleaved;
    d.dtype = dtype_id(a.k->scalar_type());
    const Tensor* w = a.wq ? a.wq : a.wk;
    d.weight_dtype = w && w->scalar_type() == at::kFloat ? (int)NQ_F32 : d.dtype;
    d.eps = (float)a.eps; d.scaling = (float)a.scaling;
    if (a.k_cache) {
        const Tensor &kc = *a.k_cache, &vc = *a.v_cache;
        d.k_cache = kc.mutable_data_ptr(); d.v_cache = vc.mutable_data_ptr();
        d.sequences = static_cast<const int32_t*>(data(a.sequences));
        d.block_table = static_cast<const int32_t*>(data(a.table));
        d.kc_page = cache_stride(kc, 0); d.kc_slot = cache_stride(kc, 1); d.kc_head = cache_stride(kc, 2);
        d.vc_page = cache_stride(vc, 0); d.vc_slot = cache_stride(vc, 1); d.vc_head = cache_stride(vc, 2);
        d.table_stride = a.table->size(0) > 1 ? a.table->stride(0) : a.table->size(1);
        d.pages = kc.size(0); d.page_size = (int)kc.size(1);
        d.seqs = (int)a.table->size(0); d.max_pages = (int)a.table->size(1);
    }
    const int dev = a.k->get_device();
    OnDevice on(dev);
    const int st = nq_heads_fwd(&d, stream_of(dev));
    if (st < 0) fail(st, "nq_heads_fwd");
    for (const Tensor* c : {a.k_cache, a.v_cache})
        if (c && !c->is_inference()) c->unsafeGetTensorImpl()->bump_version();
    return out;
}
// Whether autograd would record the call: there is no gradient to record.
bool wants_gradient(std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : inputs)
        if (t && t->requires_grad()) return true;
    return false;
}
// An argument that may be None; false: neither that nor a plain tensor.
bool maybe(PyObject* o, const Tensor*& t) {
    t = o == Py_None ? nullptr : plain(o);
    return t || o == Py_None;
}
// qk_norm_rope(q, k, positions, inv_freq, q_weight | None, k_weight | None, eps, interleaved, scaling) -> (q, k) or None
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 9, "qk_norm_rope takes 9 arguments");
    if (!exact_plain(a[0]) || !THPVariable_CheckExact(a[1])) Py_RETURN_NONE;
    HeadsArgs h{};
    h.q = plain(a[0]); h.k = plain(a[1]); h.positions = plain(a[2]); h.inv_freq = plain(a[3]);
    if (!h.q || !h.k || !h.positions || !h.inv_freq || !maybe(a[4], h.wq) || !maybe(a[5], h.wk) || wants_gradient({h.q, h.k, h.inv_freq, h.wq, h.wk}) || !heads_takes(h)) Py_RETURN_NONE;
    h.eps = PyFloat_AsDouble(a[6]);
    h.interleaved = PyObject_IsTrue(a[7]) == 1;
    h.scaling = PyFloat_AsDouble(a[8]);
    if (PyErr_Occurred()) return nullptr;
    refuse_tangents("qk_norm_rope", {h.q, h.k, h.inv_freq, h.wq, h.wk});
    const auto out = heads_launch(h);
    PyObject* q = THPVariable_Wrap(out[0]);
    PyObject* k = q ? THPVariable_Wrap(out[1]) : nullptr;
    return k ? Py_BuildValue("(NN)", q, k) : nullptr;
    END_HANDLE_TH_ERRORS
}
// append_kv(q | None, k, v, k_cache, v_cache, block_table, positions, sequences | None, inv_freq | None, q_weight | None, k_weight | None, eps, interleaved, scaling) -> q,
// True (there is none), or None
PyObject* py_append_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 14, "append_kv takes 14 arguments");
    if (!exact_plain(a[1]) || !THPVariable_CheckExact(a[2]) || !(a[0] == Py_None || THPVariable_CheckExact(a[0]))) Py_RETURN_NONE;
    HeadsArgs h{};
    h.k = plain(a[1]); h.v = plain(a[2]); h.k_cache = plain(a[3]); h.v_cache = plain(a[4]); h.table = plain(a[5]); h.positions = plain(a[6]);
    if (!maybe(a[0], h.q) || !h.k || !h.v || !h.k_cache || !h.v_cache || !h.table || !h.positions || !maybe(a[7], h.sequences) || !maybe(a[8], h.inv_freq) || !maybe(a[9], h.wq) ||
        !maybe(a[10], h.wk) || wants_gradient({h.q, h.k, h.v, h.k_cache, h.v_cache, h.inv_freq, h.wq, h.wk}) || !heads_takes(h))
        Py_RETURN_NONE;
    h.eps = PyFloat_AsDouble(a[11]);
    h.interleaved = PyObject_IsTrue(a[12]) == 1;
    h.scaling = PyFloat_AsDouble(a[13]);
    if (PyErr_Occurred()) return nullptr;
    refuse_tangents("append_kv", {h.q, h.k, h.v, h.k_cache, h.v_cache, h.inv_freq, h.wq, h.wk});
    const auto out = heads_launch(h);
    if (!h.q) Py_RETURN_TRUE;
    return THPVariable_Wrap(out[0]);
    END_HANDLE_TH_ERRORS
}

struct AttentionArgs {
    const Tensor *q, *k, *v, *cu, *cu_k, *table, *lengths;
    double scale;
    int64_t window;
    bool causal;
};
bool attention_takes(const AttentionArgs& a) {
    Heads q, k, v;
    const int dev = a.q->get_device();
    const at::ScalarType type = a.q->scalar_type();
    if (a.q->dim() != 3 || !as_heads(*a.q, q)) return false;
    if (a.table) {
        if (a.k->dim() != 4) return false;
        k = Heads{0, a.k->size(2), q.D, 0, 0};
        if (!cache_takes(*a.k, *a.v, *a.table, k, type, dev, q.tokens == 0) || !is_index(*a.lengths, at::kInt, 1, dev) || a.lengths->size(0) != a.table->size(0)) return false;
    } else {
        if (a.k->dim() != 3 || !as_heads(*a.k, k) || !as_heads(*a.v, v) || a.k->sizes() != a.v->sizes() || k.D != q.D || (k.tokens == 0 && q.tokens > 0)) return false;
        for (const Tensor* t : {a.k, a.v})
            if (t->scalar_type() != type || t->get_device() != dev) return false;
    }
    if (q.heads % k.heads != 0) return false;
    if (!a.cu) return a.lengths->size(0) == a.q->size(0);
    const int64_t seqs = a.cu->size(0) - 1;
    if (q.heads / k.heads > 128 || !is_index(*a.cu, at::kInt, 1, dev) || seqs < 1 || (a.cu_k && (!is_index(*a.cu_k, at::kInt, 1, dev) || a.cu_k->size(0) != seqs + 1))) return false;
    return !a.table || a.table->size(0) == seqs;
}
Tensor attention_launch(const AttentionArgs& a) {
    Heads q, k, v;
    as_heads(*a.q, q);
    Tensor out = new_output(a.q->sizes(), *a.q);
    if (a.q->size(0) == 0) return out;
    nq_attention_desc d{};
    d.q = data(a.q); d.k = data(a.k); d.v = data(a.v);
    d.out = out.mutable_data_ptr();
    d.cu_seqlens = static_cast<const int32_t*>(data(a.cu));
    d.cu_seqlens_k = static_cast<const int32_t*>(data(a.cu_k));
    d.lengths = static_cast<const int32_t*>(data(a.lengths));
    d.block_table = static_cast<const int32_t*>(data(a.table));
    d.q_token = q.token; d.q_head = q.head;
    d.T = a.q->size(0);
    d.q_heads = (int)q.heads; d.D = (int)q.D;
    d.window = (int)a.window; d.causal = a.causal; d.scale = (float)a.scale;
    d.dtype = dtype_id(a.q->scalar_type());
    d.seqs = (int)(a.cu ? a.cu->size(0) - 1 : a.q->size(0));
    if (a.table) {
        d.k_page = cache_stride(*a.k, 0); d.k_slot = cache_stride(*a.k, 1); d.k_head = cache_stride(*a.k, 2);
        d.v_page = cache_stride(*a.v, 0); d.v_slot = cache_stride(*a.v, 1); d.v_head = cache_stride(*a.v, 2);
        d.table_stride = a.table->size(0) > 1 ? a.table->stride(0) : a.table->size(1);
        d.pages = a.k->size(0); d.page_size = (int)a.k->size(1); d.k_heads = (int)a.k->size(2);
        d.max_pages = (int)a.table->size(1);
    } else {
        as_heads(*a.k, k);
        as_heads(*a.v, v);
        d.k_slot = k.token; d.k_head = k.head; d.v_slot = v.token; d.v_head = v.head;
        d.Tk = k.tokens; d.k_heads = (int)k.heads;
    }
    const int dev = a.q->get_device();
    OnDevice on(dev);
    int st;
    if (a.cu) {
        const size_t bytes = nq_prompt_attention_scratch_bytes(&d);
        const Tensor scratch = bytes ? new_bytes((int64_t)bytes, *a.q) : Tensor();
        st = nq_prompt_attention_fwd(&d, bytes ? scratch.mutable_data_ptr() : nullptr, bytes, status_header(dev), stream_of(dev));
        if (st < 0) fail(st, "nq_prompt_attention_fwd");
    } else {
        const size_t bytes = nq_paged_attention_scratch_bytes(d.seqs, d.q_heads, d.k_heads, d.D, (int64_t)d.max_pages * d.page_size);
        const Tensor scratch = bytes ? new_bytes((int64_t)bytes, *a.q) : Tensor();
        st = nq_paged_attention_fwd(&d, bytes ? scratch.mutable_data_ptr() : nullptr, bytes, status_header(dev), stream_of(dev));
        if (st < 0) fail(st, "nq_paged_attention_fwd");
    }
    return out;
}
// prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k | None, block_table | None, lengths | None, causal, scale, window) -> o or None
PyObject* py_prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 10, "prompt_attention takes 10 arguments");
    if (!exact_plain(a[0]) || !THPVariable_CheckExact(a[1]) || !THPVariable_CheckExact(a[2])) Py_RETURN_NONE;
    AttentionArgs t{};
    t.q = plain(a[0]); t.k = plain(a[1]); t.v = plain(a[2]); t.cu = plain(a[3]);
    if (!t.q || !t.k || !t.v || !t.cu || !maybe(a[4], t.cu_k) || !maybe(a[5], t.table) || !maybe(a[6], t.lengths) || !t.table != !t.lengths || (t.table && t.cu_k) ||
        wants_gradient({t.q, t.k, t.v}) || !attention_takes(t))
        Py_RETURN_NONE;
    t.causal = PyObject_IsTrue(a[7]) == 1;
    t.scale = PyFloat_AsDouble(a[8]);
    t.window = PyLong_AsLongLong(a[9]);
    if (PyErr_Occurred()) return nullptr;
    refuse_tangents("prompt_attention", {t.q, t.k, t.v});
    return THPVariable_Wrap(attention_launch(t));
    END_HANDLE_TH_ERRORS
}
// paged_attention(q, k_cache, v_cache, block_table, lengths, scale, window) -> o or None
PyObject* py_paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 7, "paged_attention takes 7 arguments");
    if (!exact_plain(a[0]) || !THPVariable_CheckExact(a[1]) || !THPVariable_CheckExact(a[2])) Py_RETURN_NONE;
    AttentionArgs t{};
    t.q = plain(a[0]); t.k = plain(a[1]); t.v = plain(a[2]); t.table = plain(a[3]); t.lengths = plain(a[4]);
    t.causal = true;
    if (!t.q || !t.k || !t.v || !t.table || !t.lengths || wants_gradient({t.q, t.k, t.v}) || !attention_takes(t)) Py_RETURN_NONE;
    t.scale = PyFloat_AsDouble(a[5]);
    t.window = PyLong_AsLongLong(a[6]);
    if (PyErr_Occurred()) return nullptr;
    refuse_tangents("paged_attention", {t.q, t.k, t.v});
    return THPVariable_Wrap(attention_launch(t));
    END_HANDLE_TH_ERRORS
}

// The same as operators of the dispatcher, for what records calls (torch.compile, torch.jit.trace); schemas, shapes for tracing and derivatives: nanoquant_b200/ops.py.
Tensor dense(const Tensor& t) { return t.resolve_neg().contiguous(); }
OptTensor dense(const OptTensor& t) { return t ? OptTensor(dense(*t)) : t; }
const Tensor* pointer(const OptTensor& t) { return t ? &*t : nullptr; }
Tensor or_none(const Tensor& t, const Tensor& like) { return t.defined() ? t : new_output({0}, like); }

std::tuple<Tensor, Tensor> op_norm(const Tensor& x_, const OptTensor& w_, const OptTensor& b_, double eps, bool center) {
    const Tensor x = dense_rows(x_);
    const OptTensor w = dense(w_), b = dense(b_);
    TORCH_CHECK(norm_takes(x, pointer(w), pointer(b)), "nanoquant_b200::norm: 16-bit rows, and weight and bias of their columns in that type or fp32");
    Tensor stats, y = norm_launch(x, pointer(w), pointer(b), NormArgs{x.size(-1), eps, center}, &stats);
    return {y, stats};
}
std::tuple<Tensor, Tensor, Tensor> op_norm_backward(const Tensor& dy, const Tensor& x_, const OptTensor& w_, const Tensor& stats, bool center, std::array<bool, 3> want) {
    const Tensor x = dense_rows(x_);
    const OptTensor w = dense(w_);
    TORCH_CHECK(norm_takes(x, pointer(w), nullptr) && dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && (w || !(want[1] || want[2])) &&
                    stats.scalar_type() == at::kFloat && stats.is_contiguous() && (x.size(-1) == 0 || stats.numel() == 2 * (x.numel() / x.size(-1))),
                "nanoquant_b200::norm_backward: operands of nanoquant_b200::norm and its second result");
    const auto d = norm_gradients(dy, x, w ? *w : Tensor(), stats, center, want);
    return {or_none(d[0], x), or_none(d[1], x), or_none(d[2], x)};
}
std::tuple<Tensor, Tensor> op_quantize_rows(const Tensor& x_) {
    const Tensor x = x_.dim() ? dense_rows(x_) : x_;
    TORCH_CHECK(quantize_takes(x), "nanoquant_b200::quantize_rows: 16-bit rows of at least one column");
    return quantize_launch(x);
}
Tensor op_int8_linear(const Tensor& x_, const Tensor& w_, const Tensor& ws_, const OptTensor& b_) {
    const Tensor x = dense_rows(x_), w = w_.resolve_neg();
    Tensor ws = dense(ws_);
    if (reinterpret_cast<uintptr_t>(ws.const_data_ptr()) & 15) ws = ws.clone();
    const OptTensor b = dense(b_);
    TORCH_CHECK(int8_takes(x, w, ws, pointer(b)),
                "nanoquant_b200::int8_linear: 16-bit rows, an int8 weight whose rows start at multiples of 16 bytes, its fp32 scales, a bias in the type of the rows");
    return int8_launch(x, w, ws, pointer(b));
}
Tensor op_dense_gemv(const Tensor& x_, const Tensor& w_, const OptTensor& b_) {
    const Tensor x = dense(x_), w = w_.resolve_neg();
    const OptTensor b = dense(b_);
    TORCH_CHECK(dense_gemv_takes(x, w, pointer(b)), "nanoquant_b200::dense_gemv: 16-bit rows and weight, the weight's columns dense");
    return dense_gemv_launch(x, w, pointer(b));
}
// What the loss reads in place: rows at multiples of 16 bytes.
Tensor loss_matrix(const Tensor& t_) {
    const Tensor t = t_.resolve_neg();
    const bool in_place = t.dim() == 2 && t.stride(1) == 1 && row_stride(t) % 8 == 0 && row_stride(t) >= t.size(1) && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
    return in_place ? t : t.clone(at::MemoryFormat::Contiguous);
}
const char* const kLossOperands = "nanoquant_b200::linear_cross_entropy: 16-bit matrices of one type with a multiple of 8 columns, one int64 or int32 target for each row";
std::tuple<Tensor, Tensor, Tensor> op_linear_cross_entropy(const Tensor& h_, const Tensor& w_, const Tensor& t_, int64_t ignore, int64_t reduction) {
    const Tensor h = loss_matrix(h_), w = loss_matrix(w_), t = dense(t_);
    TORCH_CHECK(loss_takes(h, w, t), kLossOperands);
    Tensor lse, count, loss = loss_launch(h, w, t, LossArgs{ignore, (int)reduction}, lse, count);
    return {loss, lse, count};
}
std::tuple<Tensor, Tensor> op_linear_cross_entropy_backward(const Tensor& grad, const Tensor& h_, const Tensor& w_, const Tensor& t_, const Tensor& lse, const Tensor& count,
                                                            int64_t ignore, int64_t reduction, std::array<bool, 2> want) {
    const Tensor h = loss_matrix(h_), w = loss_matrix(w_), t = dense(t_);
    TORCH_CHECK(loss_takes(h, w, t), kLossOperands);
    const int64_t T = h.size(0);
    TORCH_CHECK(grad.scalar_type() == at::kFloat && lse.scalar_type() == at::kFloat && count.scalar_type() == at::kFloat && lse.is_contiguous() && lse.numel() == T &&
                    count.numel() == 1 && (reduction == NQ_REDUCE_NONE ? grad.dim() == 1 && grad.size(0) == T : grad.dim() == 0),
                "nanoquant_b200::linear_cross_entropy_backward: the gradient of the first result of nanoquant_b200::linear_cross_entropy, and the other two");
    const auto d = loss_gradients(grad, h, w, t, lse, count, LossArgs{ignore, (int)reduction}, want);
    return {or_none(d[0], h), or_none(d[1], h)};
}
// Heads that the kernels do not read in place are copied.
Tensor heads_in_place(const Tensor& t_) {
    const Tensor t = t_.resolve_neg();
    Heads h;
    return as_heads(t, h) ? t : t.clone(at::MemoryFormat::Contiguous);
}
OptTensor heads_in_place(const OptTensor& t) { return t ? OptTensor(heads_in_place(*t)) : t; }
Tensor at_boundary(const Tensor& t_) {
    const Tensor t = dense(t_);
    return reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15 ? t.clone() : t;
}
OptTensor at_boundary(const OptTensor& t) { return t ? OptTensor(at_boundary(*t)) : t; }
std::tuple<Tensor, Tensor> op_qk_norm_rope(const Tensor& q_, const Tensor& k_, const Tensor& p_, const Tensor& f_, const OptTensor& wq_, const OptTensor& wk_, double eps, bool interleaved,
                                           double scaling) {
    const Tensor q = heads_in_place(q_), k = heads_in_place(k_), p = dense(p_), f = dense(f_);
    const OptTensor wq = at_boundary(wq_), wk = at_boundary(wk_);
    const HeadsArgs a{&q, &k, nullptr, nullptr, nullptr, nullptr, &p, nullptr, &f, pointer(wq), pointer(wk), eps, scaling, interleaved};
    TORCH_CHECK(heads_takes(a), "nanoquant_b200::qk_norm_rope: 16-bit heads of one type and size, a position for each token, fp32 frequencies");
    const auto out = heads_launch(a);
    return {out[0], out[1]};
}
Tensor op_append_kv(const OptTensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& kc, const Tensor& vc, const Tensor& table_, const Tensor& p_, const OptTensor& s_,
                    const OptTensor& f_, const OptTensor& wq_, const OptTensor& wk_, double eps, bool interleaved, double scaling) {
    const OptTensor q = heads_in_place(q_), s = dense(s_), f = dense(f_), wq = at_boundary(wq_), wk = at_boundary(wk_);
    const Tensor k = heads_in_place(k_), v = heads_in_place(v_), table = dense(table_), p = dense(p_);
    const HeadsArgs a{pointer(q), &k, &v, &kc, &vc, &table, &p, pointer(s), pointer(f), pointer(wq), pointer(wk), eps, scaling, interleaved};
    TORCH_CHECK(!kc.is_neg() && !vc.is_neg() && heads_takes(a),
                "nanoquant_b200::append_kv: 16-bit heads of one type and size, a cache [pages, page_size, heads, D] of them, an int32 table of pages, a position for each token");
    return or_none(heads_launch(a)[0], k);
}
Tensor op_prompt_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& cu_, const OptTensor& cu_k_, const OptTensor& table_, const OptTensor& lengths_, bool causal,
                           double scale, int64_t window) {
    const Tensor q = heads_in_place(q_), k = table_ ? k_.resolve_neg() : heads_in_place(k_), v = table_ ? v_.resolve_neg() : heads_in_place(v_), cu = dense(cu_);
    const OptTensor cu_k = dense(cu_k_), table = dense(table_), lengths = dense(lengths_);
    const AttentionArgs a{&q, &k, &v, &cu, pointer(cu_k), pointer(table), pointer(lengths), scale, window, causal};
    TORCH_CHECK(!table_.has_value() == !lengths_.has_value() && !(table_ && cu_k_) && attention_takes(a),
                "nanoquant_b200::prompt_attention: 16-bit heads of one type and size, packed or in a cache with its table and lengths, int32 starts of the sequences");
    return attention_launch(a);
}
Tensor op_paged_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& table_, const Tensor& lengths_, double scale, int64_t window) {
    const Tensor q = heads_in_place(q_), k = k_.resolve_neg(), v = v_.resolve_neg(), table = dense(table_), lengths = dense(lengths_);
    const AttentionArgs a{&q, &k, &v, nullptr, nullptr, &table, &lengths, scale, window, true};
    TORCH_CHECK(attention_takes(a), "nanoquant_b200::paged_attention: 16-bit heads of one type and size, a cache [pages, page_size, heads, D], an int32 table of pages and lengths");
    return attention_launch(a);
}
TORCH_LIBRARY_IMPL(nanoquant_b200, CUDA, m) {
    m.impl("norm", op_norm);
    m.impl("qk_norm_rope", op_qk_norm_rope);
    m.impl("append_kv", op_append_kv);
    m.impl("prompt_attention", op_prompt_attention);
    m.impl("paged_attention", op_paged_attention);
    m.impl("norm_backward", op_norm_backward);
    m.impl("quantize_rows", op_quantize_rows);
    m.impl("int8_linear", op_int8_linear);
    m.impl("dense_gemv", op_dense_gemv);
    m.impl("linear_cross_entropy", op_linear_cross_entropy);
    m.impl("linear_cross_entropy_backward", op_linear_cross_entropy_backward);
}

// The pack / layout kernels on a contiguous CUDA tensor.
enum RepackOp : int { kPackRows, kUnpackRows, kRowsToTiles, kTilesToRows, kPackMarlin };
Tensor repack(RepackOp op, const Tensor& src, int64_t rows, int64_t cols, int order) {
    const int64_t words = (cols + 31) / 32, row_groups = (rows + 15) / 16, chunks = (cols + 255) / 256;
    Tensor out = op == kUnpackRows    ? new_output({rows, cols}, src, at::kChar)
                 : op == kRowsToTiles ? new_output({row_groups, chunks, 128}, src, at::kInt)
                 : op == kPackMarlin  ? new_output({cols / 16, rows / 2}, src, at::kInt)
                                      : new_output({rows, words}, src, at::kInt);
    const int dev = src.get_device();
    OnDevice on(dev);
    const nq_stream_t stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
    const void* in = src.const_data_ptr();
    void* o = out.mutable_data_ptr();
    static const char* const kNames[5] = {"nq_pack_rows", "nq_unpack_rows", "nq_rows_to_tiles", "nq_tiles_to_rows", "nq_pack_marlin"};
    const int st = op == kPackRows      ? nq_pack_rows(static_cast<const int8_t*>(in), static_cast<int32_t*>(o), rows, cols, order, stream)
                   : op == kUnpackRows  ? nq_unpack_rows(static_cast<const int32_t*>(in), static_cast<int8_t*>(o), rows, cols, order, stream)
                   : op == kRowsToTiles ? nq_rows_to_tiles(static_cast<const int32_t*>(in), o, rows, cols, order, stream)
                   : op == kTilesToRows ? nq_tiles_to_rows(in, static_cast<int32_t*>(o), rows, cols, order, stream)
                                        : nq_pack_marlin(static_cast<const int8_t*>(in), static_cast<int32_t*>(o), rows, cols, stream);
    if (st < 0) fail(st, kNames[op]);
    return out;
}

// repack(op, src, rows, cols, order) -> out or None (rows = out features for the Marlin layout)
PyObject* py_repack(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 5, "repack takes 5 arguments");
    const Tensor* src = plain(a[1]);
    const long op = PyLong_AsLong(a[0]), order = PyLong_AsLong(a[4]);
    const int64_t rows = PyLong_AsLongLong(a[2]), cols = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    const bool dense = op == kPackRows || op == kPackMarlin;
    if (!src || op < kPackRows || op > kPackMarlin || !src->is_contiguous() || src->scalar_type() != (dense ? at::kChar : at::kInt))
        Py_RETURN_NONE;
    return THPVariable_Wrap(repack((RepackOp)op, *src, rows, cols, (int)order));
    END_HANDLE_TH_ERRORS
}

// pack_rows(dense, order) -> words; words_to(op, words, shape, order) -> unpacked or tiles.  None: not a plain CUDA
// tensor of the right type, or not of the shape it is said to have; the caller sorts that out.
PyObject* py_pack_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 2, "pack_rows takes 2 arguments");
    const Tensor* src = plain(a[0]);
    const long order = PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) return nullptr;
    if (!src || src->dim() != 2 || !src->is_contiguous() || src->scalar_type() != at::kChar) Py_RETURN_NONE;
    return THPVariable_Wrap(repack(kPackRows, *src, src->size(0), src->size(1), (int)order));
    END_HANDLE_TH_ERRORS
}
PyObject* py_words_to(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 4, "words_to takes 4 arguments");
    const Tensor* src = plain(a[1]);
    if (!src || src->dim() != 2 || !src->is_contiguous() || src->scalar_type() != at::kInt || !PyTuple_Check(a[2]) ||
        PyTuple_GET_SIZE(a[2]) != 2 || !PyLong_Check(PyTuple_GET_ITEM(a[2], 0)) || !PyLong_Check(PyTuple_GET_ITEM(a[2], 1)))
        Py_RETURN_NONE;
    const long op = PyLong_AsLong(a[0]), order = PyLong_AsLong(a[3]);
    const int64_t rows = PyLong_AsLongLong(PyTuple_GET_ITEM(a[2], 0)), cols = PyLong_AsLongLong(PyTuple_GET_ITEM(a[2], 1));
    if (PyErr_Occurred()) return nullptr;
    if ((op != kUnpackRows && op != kRowsToTiles) || src->size(0) != rows || src->size(1) != (cols + 31) / 32) Py_RETURN_NONE;
    return THPVariable_Wrap(repack((RepackOp)op, *src, rows, cols, (int)order));
    END_HANDLE_TH_ERRORS
}

// permute_scale(s, kind, inverse) -> permuted copy or None
PyObject* py_permute_scale(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 3, "permute_scale takes 3 arguments");
    const Tensor* s = plain(a[0]);
    if (!s || !s->is_contiguous() || s->element_size() != 2) Py_RETURN_NONE;
    const int kind = (int)PyLong_AsLong(a[1]), inverse = (int)PyLong_AsLong(a[2]);
    if (PyErr_Occurred()) return nullptr;
    Tensor out = new_output({s->numel()}, *s);
    const int dev = s->get_device();
    OnDevice on(dev);
    const int st = nq_permute_scale16(s->const_data_ptr(), out.mutable_data_ptr(), s->numel(), kind, inverse,
                                      c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
    if (st < 0) fail(st, "nq_permute_scale16");
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// set_scratch(device, address, bytes); set_thread_scratch(address, bytes), address 0: none
PyObject* py_set_scratch(PyObject*, PyObject* args) {
    int dev;
    unsigned long long ptr, bytes;
    if (!PyArg_ParseTuple(args, "iKK", &dev, &ptr, &bytes)) return nullptr;
    if (dev < 0 || dev >= kMaxDevices) {
        PyErr_SetString(PyExc_ValueError, "device index out of range");
        return nullptr;
    }
    std::lock_guard<std::mutex> lock(g_scratch_mutex);
    g_scratch[dev] = Scratch{reinterpret_cast<void*>(ptr), (size_t)bytes};
    Py_RETURN_NONE;
}
PyObject* py_set_thread_scratch(PyObject*, PyObject* args) {
    unsigned long long ptr, bytes;
    if (!PyArg_ParseTuple(args, "KK", &ptr, &bytes)) return nullptr;
    t_override = Scratch{reinterpret_cast<void*>(ptr), (size_t)bytes};
    Py_RETURN_NONE;
}
// set_callbacks(raise_status, grow_scratch, dyn_general, marlin_general[, thread_scratch])
PyObject* py_set_callbacks(PyObject*, PyObject* args) {
    PyObject* f[5] = {};
    if (!PyArg_ParseTuple(args, "OOOO|O", &f[0], &f[1], &f[2], &f[3], &f[4])) return nullptr;
    PyObject** slot[5] = {&g_raise_status, &g_grow_scratch, &g_dyn_general, &g_marlin_general, &g_thread_scratch};
    for (int i = 0; i < 5; ++i) {
        if (!f[i]) continue;
        Py_INCREF(f[i]);
        Py_XDECREF(*slot[i]);
        *slot[i] = f[i];
    }
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"linear_forward", (PyCFunction)(void*)py_linear_forward, METH_FASTCALL, nullptr},
    {"group_forward", (PyCFunction)(void*)py_group_forward, METH_FASTCALL, nullptr},
    {"dense_gemv_forward", (PyCFunction)(void*)py_dense_gemv_forward, METH_FASTCALL, nullptr},
    {"norm", (PyCFunction)(void*)py_norm, METH_FASTCALL, nullptr},
    {"quantize_rows", (PyCFunction)(void*)py_quantize_rows, METH_FASTCALL, nullptr},
    {"int8_linear_forward", (PyCFunction)(void*)py_int8_linear_forward, METH_FASTCALL, nullptr},
    {"linear_cross_entropy", (PyCFunction)(void*)py_linear_cross_entropy, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void*)py_qk_norm_rope, METH_FASTCALL, nullptr},
    {"append_kv", (PyCFunction)(void*)py_append_kv, METH_FASTCALL, nullptr},
    {"prompt_attention", (PyCFunction)(void*)py_prompt_attention, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void*)py_paged_attention, METH_FASTCALL, nullptr},
    {"repack", (PyCFunction)(void*)py_repack, METH_FASTCALL, nullptr},
    {"pack_rows", (PyCFunction)(void*)py_pack_rows, METH_FASTCALL, nullptr},
    {"words_to", (PyCFunction)(void*)py_words_to, METH_FASTCALL, nullptr},
    {"permute_scale", (PyCFunction)(void*)py_permute_scale, METH_FASTCALL, nullptr},
    {"module_call", (PyCFunction)(void (*)(void))py_module_call, METH_FASTCALL, nullptr},
    {"set_module_class", py_set_module_class, METH_VARARGS, nullptr},
    {"set_scratch", py_set_scratch, METH_VARARGS, nullptr},
    {"set_thread_scratch", py_set_thread_scratch, METH_VARARGS, nullptr},
    {"set_callbacks", py_set_callbacks, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_nq_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nq_torch() { return PyModule_Create(&kModule); }
