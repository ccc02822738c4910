// torchode_amd._host: what AutoDiffAdjoint.solve does around the kernel of a whole solve with a built-in term -- the argument
// block from the problem's tensors, the outputs from PyTorch's allocator, the launch, the views of the statistics while
// the kernel runs, and the wait -- as one call of a Python extension.  A small solve's kernel takes 25 to 75 microseconds, and
// the same steps in Python, one ctypes or tensor call each, took 23 ahead of the launch where they now take 9 (decay, float64,
// B = 256: 52 -> 40 us a solve; Lorenz to its end point, B = 40 009: 80 -> 67; perceptron, B = 4096: 109 -> 91).  No solver logic and
// no kernel: everything here ends in the C ABI of include/torchode_amd.h, and nothing is kept from one call for the next.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/LegacyBatchedTensorImpl.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>

#include "../../include/torchode_amd.h"

namespace {

using at::Tensor;

struct PythonError {};  // (set already)

const Tensor &tensor(PyObject *o, const char *name) {
    if (THPVariable_Check(o)) return THPVariable_Unpack(o);
    PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
    throw PythonError();
}
double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError();
    return v;
}
long long integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}
int dtype_code(at::ScalarType t) {
    TORCH_CHECK_NOT_IMPLEMENTED(t == at::kFloat || t == at::kDouble, "the kernels are built for float32 and float64 (got ", t, ")");
    return t == at::kFloat ? TODE_F32 : TODE_F64;
}
[[noreturn]] void library_error(const char *call, int rc) {
    PyErr_Format(PyExc_RuntimeError, "%s failed with code %d: %s", call, rc, tode_last_error());
    throw PythonError();
}

// The library waits for the GPU in it: other Python threads run meanwhile.
struct WithoutGil {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

PyObject *append(PyObject *tuple, Py_ssize_t i, PyObject *item) {
    if (!item) {
        Py_DECREF(tuple);
        throw PythonError();
    }
    PyTuple_SET_ITEM(tuple, i, item);
    return tuple;
}

// solve(y0, t_start, t_end, t_eval, dt0, params, shared_params, method, term, term_scalars, max_steps, allow_one_kernel, has_general, kind, dt_min,
//       dt_max, atol, rtol, pcoeff, icoeff, dcoeff, safety, factor_min, factor_max)
// -> (ys, n_steps, n_accepted, n_initialized, status, iterations), or None where no whole-solve kernel takes the problem
constexpr Py_ssize_t N_ARGS = 24;

PyObject *solve_(PyObject *const *arg) {
    const Tensor &y0_ = tensor(arg[0], "y0");
    const bool has_eval = arg[3] != Py_None, has_dt0 = arg[4] != Py_None, has_params = arg[5] != Py_None, has_shared = arg[6] != Py_None;
    const Tensor y0 = y0_.contiguous();
    // t_start / t_end are usually columns of t_eval: handed over with their stride
    auto column = [](const Tensor &t) { return t.stride(0) >= 1 ? t : t.contiguous(); };
    const Tensor t_start = column(tensor(arg[1], "t_start")), t_end = column(tensor(arg[2], "t_end"));
    const Tensor t_eval = has_eval ? tensor(arg[3], "t_eval").contiguous() : Tensor();
    const auto dtype = y0.scalar_type(), time_dtype = t_start.scalar_type();
    const Tensor dt0 = has_dt0 ? tensor(arg[4], "dt0").to(time_dtype).contiguous() : Tensor();
    const int64_t B = y0.size(0), F = y0.size(1), E = has_eval ? t_eval.size(1) : 0;
    Tensor params;
    if (has_params) {
        params = tensor(arg[5], "the term's parameters");
        if (params.device() != y0.device() || params.scalar_type() != dtype) params = params.to(y0.options());
        if (params.numel() == 0 && params.size(0) != B) params = params.new_empty({B, 0});  // a term without per-sample parameters
        if (params.dim() != 2 || params.size(0) != B) {
            PyErr_SetString(PyExc_AssertionError, "built-in term parameters do not match the batch size");
            throw PythonError();
        }
        params = params.contiguous();
    }
    const Tensor shared = has_shared ? tensor(arg[6], "the shared parameters") : Tensor();

    tode_solve_args a = {};
    const int data_code = dtype_code(dtype), time_code = dtype_code(time_dtype);
    a.dtype = data_code == time_code ? data_code : TODE_DTYPES(data_code, time_code);
    a.method = (int32_t)integer(arg[7]), a.term = (int32_t)integer(arg[8]);
    a.n_features = (int32_t)F, a.n_eval = (int32_t)E, a.n_params = has_params ? (int32_t)params.size(1) : 0;
    a.batch = B, a.max_steps = arg[10] == Py_None ? -1 : integer(arg[10]), a.iteration_cap = -1;
    const Py_ssize_t n_scalars = PyTuple_Check(arg[9]) ? PyTuple_GET_SIZE(arg[9]) : 0;
    for (Py_ssize_t i = 0; i < n_scalars && i < 4; ++i) a.term_scalars[i] = number(PyTuple_GET_ITEM(arg[9], i));
    a.y0 = y0.data_ptr();
    a.t_start = t_start.data_ptr(), a.t_end = t_end.data_ptr();
    a.t_start_stride = t_start.stride(0), a.t_end_stride = t_end.stride(0);
    a.t_eval = has_eval ? t_eval.data_ptr() : nullptr, a.dt0 = has_dt0 ? dt0.data_ptr() : nullptr;
    a.params = has_params && params.numel() > 0 ? params.data_ptr() : nullptr;
    a.shared_params = has_shared ? shared.data_ptr() : nullptr, a.n_shared_params = has_shared ? shared.numel() : 0;
    const int allow_one_kernel = PyObject_IsTrue(arg[11]), has_general = PyObject_IsTrue(arg[12]);
    if (allow_one_kernel < 0 || has_general < 0) throw PythonError();

    tode_controller c = {};
    c.kind = (int32_t)integer(arg[13]);
    c.has_dt_min = arg[14] != Py_None, c.has_dt_max = arg[15] != Py_None;
    c.dt_min = c.has_dt_min ? number(arg[14]) : 0.0, c.dt_max = c.has_dt_max ? number(arg[15]) : 0.0;
    double *const values[] = {&c.atol, &c.rtol, &c.pcoeff, &c.icoeff, &c.dcoeff, &c.safety, &c.factor_min, &c.factor_max};
    for (int i = 0; i < 8; ++i) *values[i] = number(arg[16 + i]);

    const c10::DeviceGuard guard(y0.device());
    void *const stream = (void *)c10::hip::getCurrentHIPStream(y0.device().index()).stream();
    const Tensor ys = at::empty({B, E > 0 ? E : 1, F}, y0.options());
    const Tensor out = at::empty({4, B}, y0.options().dtype(at::kLong));
    const Tensor y_idle = E == 0 ? at::empty({B, F}, y0.options()) : Tensor();
    a.ys = ys.data_ptr(), a.y_idle = E == 0 ? y_idle.data_ptr() : nullptr;
    int64_t *const stats = out.data_ptr<int64_t>();

    tode_solve_ticket ticket;
    int rc;
    {
        WithoutGil released;
        rc = tode_solve_builtin_begin(&a, &c, stats, stats + B, stats + 2 * B, stats + 3 * B, allow_one_kernel, stream, &ticket);
    }
    if (rc == TODE_E_UNSUPPORTED) Py_RETURN_NONE;  // no whole-solve kernel for this case: the caller takes the per-step or the operator path
    if (rc) library_error("tode_solve_builtin_begin", rc);
    struct End {  // (a ticket that was begun is ended, whatever happens in between)
        tode_solve_ticket &ticket;
        const tode_solve_args &a;
        const int64_t *stats;
        void *stream;
        int32_t flags[TODE_FLAG_WORDS];
        bool ended = false;
        int wait() {
            ended = true;
            WithoutGil released;
            return tode_solve_builtin_end(&ticket, &a, stats, stream, flags);
        }
        ~End() {
            if (!ended) (void)wait();
        }
    } end{ticket, a, stats, stream, {}};

    // while the kernel runs
    PyObject *result = PyTuple_New(6);
    if (!result) throw PythonError();
    append(result, 0, THPVariable_Wrap(ys));
    for (int64_t i = 0; i < 4; ++i) append(result, 1 + i, THPVariable_Wrap(out.select(0, i)));

    rc = end.wait();  // (the solve's one host synchronisation)
    const char *call = "tode_solve_builtin_end";
    int64_t iterations = end.flags[TODE_FLAG_MAX_ITERATIONS];
    if (rc == TODE_OK && end.flags[TODE_FLAG_NEEDS_GENERAL]) {
        if (!has_general) {
            Py_DECREF(result);
            Py_RETURN_NONE;
        }
        call = "tode_solve_builtin_auto";
        const int64_t bytes = tode_solve_workspace_bytes(&a);
        const Tensor workspace = at::empty({bytes}, y0.options().dtype(at::kByte));
        WithoutGil released;
        rc = tode_solve_builtin_auto(&a, &c, stats, stats + B, stats + 2 * B, stats + 3 * B, workspace.data_ptr(), bytes, 0, stream, &iterations);
    }
    if (rc) {
        Py_DECREF(result);
        library_error(call, rc);
    }
    return append(result, 5, PyLong_FromLongLong(iterations));
}

// stage(state, controller, i, y, t, k, stream): stage i of an iteration around a user's right-hand side (tode_step_stage): a node time
// and a stage input made like t and y, the launch that fills them, and (time, input) as the right-hand side's arguments.  k: the
// derivative of the stage before, contiguous and of y's shape and type, or None.  state, controller, stream: addresses.
PyObject *stage_(PyObject *const *arg) {
    tode_step_state *const s = (tode_step_state *)PyLong_AsVoidPtr(arg[0]);
    const tode_controller *const c = (const tode_controller *)PyLong_AsVoidPtr(arg[1]);
    const long long i = integer(arg[2]);
    void *const stream = arg[6] == Py_None ? nullptr : PyLong_AsVoidPtr(arg[6]);
    if (PyErr_Occurred()) throw PythonError();
    if (!s || !c || i < 1 || i > 6) {
        PyErr_SetString(PyExc_ValueError, "stage: null address or stage out of range");
        throw PythonError();
    }
    const Tensor &y = tensor(arg[3], "y"), &t = tensor(arg[4], "t");
    if (arg[5] != Py_None) {
        const Tensor &k = tensor(arg[5], "k");
        TORCH_CHECK_VALUE(k.scalar_type() == y.scalar_type() && k.device() == y.device() && k.sizes() == y.sizes() && k.is_contiguous(), "stage: k must be contiguous and of y's shape, type and device");
        s->k[i - 1] = k.data_ptr();
    }
    const Tensor input = at::empty(y.sizes(), y.options()), node = at::empty(t.sizes(), t.options());
    s->ystage[i] = input.data_ptr(), s->tnode = node.data_ptr();
    int rc;
    {
        WithoutGil released;
        rc = tode_step_stage(s, c, (int32_t)i, stream);
    }
    if (rc) library_error("tode_step_stage", rc);
    PyObject *result = PyTuple_New(2);
    if (!result) throw PythonError();
    append(result, 0, THPVariable_Wrap(node));
    return append(result, 1, THPVariable_Wrap(input));
}

// ------------------------------------------------------------------------------------------
// operators of a user's right-hand side (torchode_amd/field_ops.py), with their graph nodes: an autograd.Function of Python's takes longer
// than the kernels of a small call (group norm of 16 x 16 x 16 x 24 float64 values with its gradients: 205 us a step, from here 88)
// ------------------------------------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr const char *NEEDS_GPU = "torchode_amd runs on an AMD GPU (HIP device) only; got a tensor on '";

int field_dtype(const Tensor &t, const char *name) {
    switch (t.scalar_type()) {
        case at::kFloat: return TODE_F32;
        case at::kDouble: return TODE_F64;
        case at::kBFloat16: return TODE_BF16;
        case at::kHalf: return TODE_F16;
        default: TORCH_CHECK_NOT_IMPLEMENTED(false, name, " must be float32, float64, bfloat16 or float16, got ", t.scalar_type());
    }
}
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream_on(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor optional(PyObject *o, const char *name) { return o == Py_None ? Tensor() : tensor(o, name); }
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError();
    return v != 0;
}
// (without Python: a backward pass runs in a thread that does not hold its lock)
void succeeded(int64_t rc, const char *call) { TORCH_CHECK(rc >= 0, call, " failed with code ", rc, ": ", tode_last_error()); }
Tensor workspace_of(int64_t bytes, const char *call, const Tensor &like) {
    succeeded(bytes, call);
    return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
PyObject *tuple_of(std::initializer_list<Tensor> tensors) {
    PyObject *result = PyTuple_New((Py_ssize_t)tensors.size());
    if (!result) throw PythonError();
    Py_ssize_t i = 0;
    for (const Tensor &t : tensors) {
        if (!t.defined()) Py_INCREF(Py_None);
        append(result, i++, t.defined() ? THPVariable_Wrap(t) : Py_None);
    }
    return result;
}
// With its values in memory as they are: the imaginary part of a conjugate is a view with a flag that says negative.
Tensor as_stored(const Tensor &t) { return t.resolve_neg(); }
// (a graph node's edges belong to the tensors there are)
std::optional<Tensor> if_there(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool recorded(std::initializer_list<const Tensor *> tensors) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// Whether someone records what is called or looks on: torch.jit.trace, modes like those of make_fx and FakeTensorMode, tensors that dispatch to Python. They see
// the dispatcher's operations only, so a call from here would leave the allocation of its result and not what fills it.
bool watched(std::initializer_list<const Tensor *> tensors) {
    if (torch::jit::tracer::isTracing() || c10::impl::dispatch_mode_enabled()) return true;
    for (const Tensor *t : tensors)
        if (t->defined() && t->unsafeGetTensorImpl()->is_python_dispatch()) return true;
    return false;
}
PyObject *none() {
    Py_INCREF(Py_None);
    return Py_None;
}
// There is no forward-mode derivative: a tangent (of torch.autograd.forward_ad; torch.func's has its own refusal) would be lost without a word.
void without_tangent(const char *operation, std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors) TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), operation, " has no forward-mode derivative");
}
// Gradients as a backward pass returns them: where a graph of it is asked for, results of a node that says that there is none.
variable_list once(variable_list gradients, const char *message, const variable_list &inputs, const Tensor &cotangent) {
    if (!c10::GradMode::is_enabled()) return gradients;
    const auto node = std::make_shared<torch::autograd::Error>(message, torch::autograd::collect_next_edges(inputs, cotangent));
    for (Tensor &t : gradients)
        if (t.defined()) torch::autograd::set_history(t, node);
    return gradients;
}

// gradients(cotangent), of a cotangent that torch.autograd.grad(is_grads_batched=True) or a vectorised Jacobian has wrapped for each of those in it: one
// after the other, as there are few and each is a whole backward pass.
template <typename F> variable_list each(const Tensor &cotangent, F gradients) {
    const at::BatchedTensorImpl *const batched = at::maybeGetBatchedImpl(cotangent);
    if (!batched) return gradients(cotangent);
    std::vector<int64_t> from, to, sizes;
    at::BatchDims dims;
    for (const at::BatchDim &dim : batched->bdims()) {  // (in front, in order of their levels)
        dims.emplace_back(dim.level(), (int64_t)to.size());
        from.push_back(dim.dim()), to.push_back((int64_t)to.size()), sizes.push_back(batched->value().size(dim.dim()));
    }
    const Tensor all = batched->value().movedim(from, to).flatten(0, (int64_t)to.size() - 1);
    std::vector<std::vector<Tensor>> found;
    for (int64_t n = 0; n < all.size(0); ++n) {
        variable_list one = gradients(all[n]);
        found.resize(one.size());
        for (size_t i = 0; i < one.size(); ++i)
            if (one[i].defined()) found[i].push_back(one[i]);
    }
    TORCH_CHECK_VALUE(!found.empty(), "no cotangents");
    variable_list result(found.size());
    for (size_t i = 0; i < found.size(); ++i)
        if (!found[i].empty()) result[i] = at::makeBatched(at::stack(found[i]).unflatten(0, sizes), dims);
    return result;
}

// A backward pass that something looks on at, or whose cotangent a transform of torch.func has wrapped: the functions of field_ops.py know both.
bool beyond_here(const Tensor &cotangent) {
    const auto keys = cotangent.unsafeGetTensorImpl()->key_set();
    return watched({&cotangent}) || keys.has(c10::DispatchKey::FuncTorchBatched) || keys.has(c10::DispatchKey::FuncTorchGradWrapper);
}
struct WithGil {
    PyGILState_STATE state = PyGILState_Ensure();
    ~WithGil() { PyGILState_Release(state); }
};
struct Owned {  // a reference, or a Python error to be thrown
    PyObject *object;
    explicit Owned(PyObject *o) : object(o) {
        if (o) return;
        python_error e;
        e.persist();
        throw e;
    }
    ~Owned() { Py_DECREF(object); }
    Owned(const Owned &) = delete;
};
PyObject *argument(const Tensor &t) { return t.defined() ? THPVariable_Wrap(t) : none(); }
PyObject *argument(int64_t v) { return PyLong_FromLongLong(v); }
PyObject *argument(double v) { return PyFloat_FromDouble(v); }
PyObject *argument(bool v) { return PyBool_FromLong(v); }
// torchode_amd.field_ops.<function>.apply(...), a tuple of tensors and None
template <typename... A> variable_list applied(const char *function, const A &...of) {
    const WithGil gil;
    const Owned arguments(PyTuple_New(sizeof...(A)));
    Py_ssize_t i = 0;
    ([&] {
        PyObject *const o = argument(of);
        PyTuple_SET_ITEM(arguments.object, i++, o ? o : none());
        if (!o) Owned{nullptr};
    }(), ...);
    const Owned module(PyImport_ImportModule("torchode_amd.field_ops")), type(PyObject_GetAttrString(module.object, function)), apply(PyObject_GetAttrString(type.object, "apply"));
    const Owned result(PyObject_Call(apply.object, arguments.object, nullptr));
    const Owned tuple(PySequence_Tuple(result.object));
    variable_list tensors;
    for (Py_ssize_t k = 0; k < PyTuple_GET_SIZE(tuple.object); ++k) {
        PyObject *const item = PyTuple_GET_ITEM(tuple.object, k);
        tensors.push_back(THPVariable_Check(item) ? THPVariable_Unpack(item) : Tensor());
    }
    return tensors;
}

// x [B, ..., C], weight and bias [C] ([B, C]: one for each sample), scale and shift [B, C]: checked, and as the kernels take them
struct NormCall {
    Tensor x, weight, bias, scale, shift;
    tode_group_norm_args a = {};
    at::ScalarType statistics;

    Tensor parameter(const Tensor &t, const char *name, bool may_be_shared, int32_t &dtype, bool &seen) {
        if (!t.defined()) return t;
        const int64_t B = x.size(0), C = x.size(-1);
        const bool per_sample = t.dim() == 2 && t.size(0) == B && t.size(1) == C;
        TORCH_CHECK_VALUE(per_sample || (may_be_shared && t.dim() == 1 && t.size(0) == C), "group_norm: ", name, " must be ", may_be_shared ? "[channels] or " : "", "[batch, channels] = [", B, ", ", C, "], got ", t.sizes());
        if (may_be_shared) {
            TORCH_CHECK_VALUE(!seen || (a.affine_per_sample != 0) == (t.dim() == 2), "group_norm: weight and bias must have the same shape");
            a.affine_per_sample = t.dim() == 2;
        }
        const int32_t type = field_dtype(t, name);
        TORCH_CHECK_VALUE(type == a.dtype || (type == TODE_F32 && a.dtype != TODE_F64), "group_norm: ", name, " must be of x's type (", x.scalar_type(), ")", a.dtype == TODE_F64 ? "" : " or float32", ", got ", t.scalar_type());
        TORCH_CHECK_VALUE(!seen || type == dtype, "group_norm: ", may_be_shared ? "weight and bias" : "scale and shift", " must have the same type");
        TORCH_CHECK_VALUE(t.device() == x.device(), "group_norm: ", name, " is on ", t.device(), ", x on ", x.device());
        dtype = type, seen = true;
        return as_stored(t).contiguous();
    }
    NormCall(const Tensor &x_, const Tensor &weight_, const Tensor &bias_, const Tensor &scale_, const Tensor &shift_, int64_t G, int64_t activation) : x(x_) {
        TORCH_CHECK_VALUE(x.dim() >= 2, "group_norm: x must be [batch, ..., channels], got ", x.sizes());
        a.dtype = a.affine_dtype = a.modulation_dtype = field_dtype(x, "x");
        a.activation = (int32_t)activation;
        const int64_t B = x.size(0), C = x.size(-1);
        TORCH_CHECK_VALUE(G >= 1 && C >= 1 && C % G == 0, "group_norm: ", C, " channels cannot be divided into ", G, " groups");
        TORCH_CHECK_VALUE(C <= (1 << 20), "group_norm: at most 2^20 channels, got ", C);
        bool affine = false, modulation = false;
        weight = parameter(weight_, "weight", true, a.affine_dtype, affine), bias = parameter(bias_, "bias", true, a.affine_dtype, affine);
        scale = parameter(scale_, "scale", false, a.modulation_dtype, modulation), shift = parameter(shift_, "shift", false, a.modulation_dtype, modulation);
        without_tangent("group_norm", {&x, &weight_, &bias_, &scale_, &shift_});
        TORCH_CHECK(x.is_cuda(), NEEDS_GPU, x.device(), "'. There is no CPU implementation to fall back to.");
        x = as_stored(x).contiguous();
        a.n_groups = (int32_t)G, a.channels = (int32_t)C, a.batch = B, a.positions = 1;
        for (int64_t i = 1; i + 1 < x.dim(); ++i) a.positions *= x.size(i);
        a.x = x.data_ptr();
        a.weight = address(weight), a.bias = address(bias), a.scale = address(scale), a.shift = address(shift);
        statistics = a.dtype == TODE_F64 ? at::kDouble : at::kFloat;
    }
    // (y, mean, rstd); the latter two undefined unless `keep` is set
    std::tuple<Tensor, Tensor, Tensor> forward(double eps, bool keep) {
        TORCH_CHECK_VALUE(eps >= 0, "group_norm: eps must not be negative, got ", eps);
        a.eps = eps;
        const c10::DeviceGuard guard(x.device());
        const Tensor y = at::empty(x.sizes(), x.options());
        Tensor mean, rstd;
        if (keep) {
            mean = at::empty({a.batch, a.n_groups}, x.options().dtype(statistics)), rstd = at::empty_like(mean);
            a.mean = mean.data_ptr(), a.rstd = rstd.data_ptr();
        }
        a.y = y.data_ptr();
        const Tensor workspace = workspace_of(a.workspace_bytes = tode_group_norm_workspace_bytes(&a, 0), "tode_group_norm_workspace_bytes", x);
        a.workspace = address(workspace);
        succeeded(tode_group_norm(&a, stream_on(x)), "tode_group_norm");
        return {y, mean, rstd};
    }
    // of x, weight, bias, scale, shift: undefined where bit i of `want` is not set
    variable_list backward(const Tensor &dy_, const Tensor &mean_, const Tensor &rstd_, int64_t want) {
        TORCH_CHECK_VALUE(dy_.sizes() == x.sizes() && dy_.scalar_type() == x.scalar_type() && dy_.device() == x.device(), "group_norm: the cotangent must be like x");
        without_tangent("group_norm's gradient", {&dy_});
        for (const Tensor *t : {&mean_, &rstd_})
            TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == a.batch && t->size(1) == a.n_groups && t->scalar_type() == statistics && t->device() == x.device(), "group_norm: mean and rstd must be [batch, groups] as the forward pass returned them");
        const Tensor dy = as_stored(dy_).contiguous(), mean = mean_.contiguous(), rstd = rstd_.contiguous();  // (repeated for mapped cotangents of one sample)
        const c10::DeviceGuard guard(x.device());
        a.dy = dy.data_ptr(), a.mean = mean.data_ptr(), a.rstd = rstd.data_ptr();
        const Tensor *like[5] = {&x, &weight, &bias, &scale, &shift};
        void **const out[5] = {&a.dx, &a.dweight, &a.dbias, &a.dscale, &a.dshift};
        variable_list gradients(5);
        for (int i = 0; i < 5; ++i)
            if (((want >> i) & 1) && like[i]->defined()) gradients[i] = at::empty(like[i]->sizes(), like[i]->options()), *out[i] = gradients[i].data_ptr();
        const Tensor workspace = workspace_of(a.workspace_bytes = tode_group_norm_workspace_bytes(&a, 1), "tode_group_norm_workspace_bytes", x);
        a.workspace = address(workspace);
        succeeded(tode_group_norm_backward(&a, stream_on(x)), "tode_group_norm_backward");
        return gradients;
    }
};

struct NormNode : torch::autograd::Function<NormNode> {
    typedef const std::optional<Tensor> &Optional;
    static Tensor forward(AutogradContext *ctx, const Tensor &x, Optional weight, Optional bias, Optional scale, Optional shift, int64_t groups, int64_t activation, double eps) {
        NormCall call(x, weight.value_or(Tensor()), bias.value_or(Tensor()), scale.value_or(Tensor()), shift.value_or(Tensor()), groups, activation);
        const auto [y, mean, rstd] = call.forward(eps, true);
        ctx->saved_data["groups"] = groups, ctx->saved_data["activation"] = activation;
        ctx->save_for_backward({call.x, call.weight, call.bias, call.scale, call.shift, mean, rstd});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        if (!grads[0].defined()) return variable_list(8);
        const variable_list saved = ctx->get_saved_variables();
        const int64_t groups = ctx->saved_data["groups"].toInt(), activation = ctx->saved_data["activation"].toInt();
        int64_t want = 0;
        size_t edge = 0;
        for (int i = 0; i < 5; ++i)
            if (saved[i].defined()) want |= (int64_t)ctx->needs_input_grad(edge++) << i;
        variable_list gradients;
        if (beyond_here(grads[0]))
            gradients = applied("_GroupNormBackward", grads[0], saved[0], saved[5], saved[6], saved[1], saved[2], saved[3], saved[4], groups, activation, want);
        else {
            {
                const at::AutoDispatchBelowADInplaceOrView below;
                NormCall call(saved[0], saved[1], saved[2], saved[3], saved[4], groups, activation);
                gradients = each(grads[0], [&](const Tensor &dy) { return call.backward(dy, saved[5], saved[6], want); });
            }
            gradients = once(std::move(gradients), "group_norm is not differentiable twice", saved, grads[0]);
        }
        gradients.resize(8);
        return gradients;
    }
};

// group_norm(x, n_groups, weight, bias, scale, shift, activation, eps) -> y, or None: to go through the dispatcher
PyObject *group_norm_(PyObject *const *arg) {
    const Tensor &x = tensor(arg[0], "x");
    const Tensor weight = optional(arg[2], "weight"), bias = optional(arg[3], "bias"), scale = optional(arg[4], "scale"), shift = optional(arg[5], "shift");
    if (watched({&x, &weight, &bias, &scale, &shift})) return none();
    const long long groups = integer(arg[1]), activation = integer(arg[6]);
    const double eps = number(arg[7]);
    if (recorded({&x, &weight, &bias, &scale, &shift})) return THPVariable_Wrap(NormNode::apply(x, if_there(weight), if_there(bias), if_there(scale), if_there(shift), (int64_t)groups, (int64_t)activation, eps));
    NormCall call(x, weight, bias, scale, shift, groups, activation);
    return THPVariable_Wrap(std::get<0>(call.forward(eps, false)));
}
// group_norm_forward(the same) -> (y, mean, rstd), outside of any graph
PyObject *group_norm_forward_(PyObject *const *arg) {
    NormCall call(tensor(arg[0], "x"), optional(arg[2], "weight"), optional(arg[3], "bias"), optional(arg[4], "scale"), optional(arg[5], "shift"), integer(arg[1]), integer(arg[6]));
    const auto [y, mean, rstd] = call.forward(number(arg[7]), true);
    return tuple_of({y, mean, rstd});
}
// group_norm_backward(dy, x, mean, rstd, n_groups, weight, bias, scale, shift, activation, want) -> (dx, dweight, dbias, dscale, dshift), None where
// bit i of want is not set
PyObject *group_norm_backward_(PyObject *const *arg) {
    NormCall call(tensor(arg[1], "x"), optional(arg[5], "weight"), optional(arg[6], "bias"), optional(arg[7], "scale"), optional(arg[8], "shift"), integer(arg[4]), integer(arg[9]));
    const variable_list g = call.backward(tensor(arg[0], "the cotangent"), tensor(arg[2], "mean"), tensor(arg[3], "rstd"), integer(arg[10]));
    return tuple_of({g[0], g[1], g[2], g[3], g[4]});
}

// q [B, queries, heads, D], k and v [B, keys, kv_heads, D], lengths [B] or undefined, mask [B, keys] or undefined
struct AttentionCall {
    Tensor q, k, v, lengths, mask;
    tode_cross_attention_args a = {};

    // any strides will do as long as a row's values lie side by side
    static Tensor rows(const Tensor &t, int64_t (&strides)[3]) {
        const Tensor s = as_stored(t), r = s.stride(3) == 1 || s.size(3) == 1 ? s : s.contiguous();
        for (int i = 0; i < 3; ++i) strides[i] = r.stride(i);
        return r;
    }
    AttentionCall(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &lengths_, const Tensor &mask_, std::optional<double> scale) : q(q_), k(k_), v(v_), lengths(lengths_), mask(mask_) {
        TORCH_CHECK_VALUE(q.dim() == 4, "cross_attention: q must be [batch, queries, heads, head_dim], got ", q.sizes());
        TORCH_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes(), "cross_attention: k and v must both be [batch, keys, kv_heads, head_dim], got ", k.sizes(), " and ", v.sizes());
        const int64_t B = q.size(0), D = q.size(3);
        TORCH_CHECK_VALUE(k.size(0) == B && k.size(3) == D, "cross_attention: q ", q.sizes(), " and k ", k.sizes(), " differ in batch or head_dim");
        TORCH_CHECK_VALUE(k.size(2) >= 1 && q.size(2) >= 1 && q.size(2) % k.size(2) == 0, "cross_attention: ", q.size(2), " heads cannot share ", k.size(2), " heads of keys evenly");
        const auto type = q.scalar_type();
        TORCH_CHECK_NOT_IMPLEMENTED(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "cross_attention is built for float32, bfloat16 and float16, got ", type);
        TORCH_CHECK_VALUE(k.scalar_type() == type && v.scalar_type() == type, "cross_attention: q, k and v must have the same type, got ", type, ", ", k.scalar_type(), " and ", v.scalar_type());
        const int64_t most = type == at::kFloat ? TODE_ATTENTION_MAX_HEAD_DIM_F32 : TODE_ATTENTION_MAX_HEAD_DIM;
        TORCH_CHECK_VALUE(D >= 1 && D <= most, "cross_attention: head_dim must be 1 to ", most, " in ", type, ", got ", D);
        if (lengths.defined())
            TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == B && (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong), "cross_attention: lengths must be [batch] of int32 or int64, got ", lengths.sizes(), " of ", lengths.scalar_type());
        if (mask.defined())
            TORCH_CHECK_VALUE(mask.dim() == 2 && mask.size(0) == B && mask.size(1) == k.size(1) && mask.scalar_type() == at::kBool, "cross_attention: mask must be [batch, keys] of bool, got ", mask.sizes(), " of ", mask.scalar_type());
        a.scale = scale ? *scale : 1 / std::sqrt((double)D);
        TORCH_CHECK_VALUE(std::isfinite(a.scale), "cross_attention: scale must be finite, got ", a.scale);
        for (const Tensor *t : {&k, &v, &lengths, &mask})
            TORCH_CHECK_VALUE(!t->defined() || t->device() == q.device(), "cross_attention: a tensor is on ", t->device(), ", q on ", q.device());
        without_tangent("cross_attention", {&q, &k, &v});
        TORCH_CHECK(q.is_cuda(), NEEDS_GPU, q.device(), "'. There is no CPU implementation to fall back to.");
        q = rows(q, a.q_strides), k = rows(k, a.k_strides), v = rows(v, a.v_strides);
        if (lengths.defined()) lengths = lengths.contiguous();
        if (mask.defined() && mask.stride(1) != 1) mask = mask.contiguous();
        a.dtype = type == at::kFloat ? TODE_F32 : type == at::kBFloat16 ? TODE_BF16 : TODE_F16;
        a.batch = B, a.queries = q.size(1), a.keys = k.size(1);
        a.heads = (int32_t)q.size(2), a.kv_heads = (int32_t)k.size(2), a.head_dim = (int32_t)D;
        a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
        a.lengths = address(lengths), a.lengths_are_64 = lengths.defined() && lengths.scalar_type() == at::kLong;
        a.mask = (const uint8_t *)address(mask), a.mask_stride = mask.defined() ? mask.stride(0) : 0;
    }
    // (out, low, lse); the latter two undefined unless `keep` is set.  low: what rounding to 16 bits took off out ([..., 0] in float32)
    std::tuple<Tensor, Tensor, Tensor> forward(bool keep) {
        const c10::DeviceGuard guard(q.device());
        const Tensor out = at::empty(q.sizes(), q.options());
        Tensor low, lse;
        if (keep) {
            lse = at::empty(q.sizes().slice(0, 3), q.options().dtype(at::kFloat)), a.lse = lse.data_ptr<float>();
            low = a.dtype == TODE_F32 ? at::empty({q.size(0), q.size(1), q.size(2), 0}, q.options()) : at::empty(q.sizes(), q.options());
            a.out_low = low.numel() > 0 ? low.data_ptr() : nullptr;
        }
        a.out = out.data_ptr();
        const Tensor workspace = workspace_of(a.workspace_bytes = tode_cross_attention_workspace_bytes(&a, 0), "tode_cross_attention_workspace_bytes", q);
        a.workspace = address(workspace);
        succeeded(tode_cross_attention(&a, stream_on(q)), "tode_cross_attention");
        return {out, low, lse};
    }
    // of q, k, v: undefined where not wanted
    variable_list backward(const Tensor &grad_, const Tensor &out_, const Tensor &low_, const Tensor &lse_, bool want_q, bool want_kv) {
        for (const Tensor *t : {&grad_, &out_})
            TORCH_CHECK_VALUE(t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type() && t->device() == q.device(), "cross_attention: the output and its cotangent must be like q");
        TORCH_CHECK_VALUE(low_.scalar_type() == q.scalar_type() && low_.device() == q.device() && (a.dtype == TODE_F32 ? low_.numel() == 0 : low_.sizes() == q.sizes()) && lse_.sizes() == q.sizes().slice(0, 3) && lse_.scalar_type() == at::kFloat && lse_.device() == q.device(), "cross_attention: out, low and lse must be as the forward pass returned them");
        const Tensor out = out_.contiguous(), low = low_.contiguous(), lse = lse_.contiguous();  // (repeated for mapped cotangents of one sample)
        without_tangent("cross_attention's gradient", {&grad_});
        const Tensor grad = rows(grad_, a.grad_strides);
        const c10::DeviceGuard guard(q.device());
        variable_list g(3);
        if (want_q) g[0] = at::empty(q.sizes(), q.options()), a.dq = g[0].data_ptr();
        if (want_kv) g[1] = at::empty(k.sizes(), k.options()), g[2] = at::empty(v.sizes(), v.options()), a.dk = g[1].data_ptr(), a.dv = g[2].data_ptr();
        a.grad_out = grad.data_ptr(), a.out = out.data_ptr(), a.lse = lse.data_ptr<float>(), a.out_low = low.numel() > 0 ? low.data_ptr() : nullptr;
        const Tensor workspace = workspace_of(a.workspace_bytes = tode_cross_attention_workspace_bytes(&a, 1), "tode_cross_attention_workspace_bytes", q);
        a.workspace = address(workspace);
        succeeded(tode_cross_attention_backward(&a, stream_on(q)), "tode_cross_attention_backward");
        return g;
    }
};

struct AttentionNode : torch::autograd::Function<AttentionNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &lengths, const std::optional<Tensor> &mask, std::optional<double> scale) {
        AttentionCall call(q, k, v, lengths.value_or(Tensor()), mask.value_or(Tensor()), scale);
        const auto [out, low, lse] = call.forward(true);
        ctx->saved_data["scale"] = call.a.scale;
        ctx->save_for_backward({call.q, call.k, call.v, call.lengths, call.mask, out, low, lse});
        return out;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        if (!grads[0].defined()) return variable_list(6);
        const variable_list saved = ctx->get_saved_variables();
        const double scale = ctx->saved_data["scale"].toDouble();
        const bool want_q = ctx->needs_input_grad(0), want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
        variable_list gradients;
        if (beyond_here(grads[0]))
            gradients = applied("_CrossAttentionBackward", grads[0], saved[0], saved[1], saved[2], saved[5], saved[6], saved[7], saved[3], saved[4], scale, want_q, want_kv);
        else {
            {
                const at::AutoDispatchBelowADInplaceOrView below;
                AttentionCall call(saved[0], saved[1], saved[2], saved[3], saved[4], scale);
                gradients = each(grads[0], [&](const Tensor &grad) { return call.backward(grad, saved[5], saved[6], saved[7], want_q, want_kv); });
            }
            gradients = once(std::move(gradients), "cross_attention is not differentiable twice", saved, grads[0]);
        }
        for (int i = 0; i < 3; ++i)
            if (!ctx->needs_input_grad(i)) gradients[i] = Tensor();
        gradients.resize(6);
        return gradients;
    }
};

std::optional<double> scale_of(PyObject *o) { return o == Py_None ? std::nullopt : std::optional<double>(number(o)); }

// cross_attention(q, k, v, lengths, mask, scale) -> out, or None: to go through the dispatcher
PyObject *cross_attention_(PyObject *const *arg) {
    const Tensor &q = tensor(arg[0], "q"), &k = tensor(arg[1], "k"), &v = tensor(arg[2], "v");
    const Tensor lengths = optional(arg[3], "lengths"), mask = optional(arg[4], "mask");
    if (watched({&q, &k, &v, &lengths, &mask})) return none();
    const std::optional<double> scale = scale_of(arg[5]);
    if (recorded({&q, &k, &v})) return THPVariable_Wrap(AttentionNode::apply(q, k, v, if_there(lengths), if_there(mask), scale));
    AttentionCall call(q, k, v, lengths, mask, scale);
    return THPVariable_Wrap(std::get<0>(call.forward(false)));
}
// cross_attention_forward(the same) -> (out, low, lse), outside of any graph
PyObject *cross_attention_forward_(PyObject *const *arg) {
    AttentionCall call(tensor(arg[0], "q"), tensor(arg[1], "k"), tensor(arg[2], "v"), optional(arg[3], "lengths"), optional(arg[4], "mask"), scale_of(arg[5]));
    const auto [out, low, lse] = call.forward(true);
    return tuple_of({out, low, lse});
}
// cross_attention_backward(grad, q, k, v, out, low, lse, lengths, mask, scale, want_q, want_kv) -> (dq, dk, dv), None where not wanted
PyObject *cross_attention_backward_(PyObject *const *arg) {
    AttentionCall call(tensor(arg[1], "q"), tensor(arg[2], "k"), tensor(arg[3], "v"), optional(arg[7], "lengths"), optional(arg[8], "mask"), scale_of(arg[9]));
    const variable_list g = call.backward(tensor(arg[0], "the cotangent"), tensor(arg[4], "out"), tensor(arg[5], "low"), tensor(arg[6], "lse"), truth(arg[10]), truth(arg[11]));
    return tuple_of({g[0], g[1], g[2]});
}

// watched(tensor) -> bool
PyObject *watched_(PyObject *const *arg) { return PyBool_FromLong(watched({&tensor(arg[0], "the argument")})); }

template <Py_ssize_t N, PyObject *(*F)(PyObject *const *)> PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "takes %zd arguments, got %zd", N, n);
        return nullptr;
    }
    HANDLE_TH_ERRORS
    try {
        return F(args);
    } catch (const PythonError &) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"solve", (PyCFunction)(void (*)())entry<N_ARGS, solve_>, METH_FASTCALL, "One whole solve with a built-in term (see torchode_amd.adjoints)."},
    {"stage", (PyCFunction)(void (*)())entry<7, stage_>, METH_FASTCALL, "One stage around a user's right-hand side (see torchode_amd.adjoints)."},
    {"watched", (PyCFunction)(void (*)())entry<1, watched_>, METH_FASTCALL, "Whether a tracer or a mode looks on at operations on this tensor."},
    {"group_norm", (PyCFunction)(void (*)())entry<8, group_norm_>, METH_FASTCALL, "See torchode_amd.field_ops."},
    {"group_norm_forward", (PyCFunction)(void (*)())entry<8, group_norm_forward_>, METH_FASTCALL, "The same with its statistics."},
    {"group_norm_backward", (PyCFunction)(void (*)())entry<11, group_norm_backward_>, METH_FASTCALL, "Its vector-Jacobian products."},
    {"cross_attention", (PyCFunction)(void (*)())entry<6, cross_attention_>, METH_FASTCALL, "See torchode_amd.field_ops."},
    {"cross_attention_forward", (PyCFunction)(void (*)())entry<6, cross_attention_forward_>, METH_FASTCALL, "The same with its rows' log-sums."},
    {"cross_attention_backward", (PyCFunction)(void (*)())entry<12, cross_attention_backward_>, METH_FASTCALL, "Its vector-Jacobian products."},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
