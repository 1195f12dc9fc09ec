// Autograd nodes of the training path in native code: one node per LogicLayer, one for GroupSum and one per dense layer.
//
// What a training step of a small network costs is the host: a Python autograd function with its views, checks and ctypes calls took
// 40 us forward and 60 us backward per layer, for kernels of 3 to 10 us.  These nodes do the same -- same kernels, same
// launches, same saved tensors -- without the interpreter: a step of 784 -> 4 x 8000, batch 100, in a plain loop
// 626 -> 340 us (forward 206 -> 102, backward 312 -> 164; what is left is mostly PyTorch's modules, loss, engine and optimizer hooks).
//
// A call that does not have the ordinary form returns None, and the Python functions of difflogic.py take it, with their checks and
// messages: other tensor types, dtypes and layouts, functorch transforms, tensor and function modes, forward mode, tracing.  So does a
// backward pass that has more to do than the layer's gradients (an optimizer that steps inside it, an exchange between GPUs,
// backward_w on a stream of its own): those are asked for when it runs, since they may be switched on after the forward pass.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <atomic>
#include <string>

#include "difflogic_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct WithGil {  // for the engine's threads
    PyGILState_STATE state = PyGILState_Ensure();
    ~WithGil() { PyGILState_Release(state); }
};
struct WithoutGil {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

std::atomic<long long> g_launches{0};  // kernels launched from here, as _native.launch_count() counts
PyObject *g_module_dict = nullptr;     // difflogic.py's: `_backward_w_stream` and `_backward_of_node`

void check(int status) {
    // one string: a number in the message would go through a stream, and a compiler that brings its own C++ library links one here whose
    // locale is not PyTorch's (the process ended there instead of raising)
    TORCH_CHECK(status == DL_OK, "difflogic_b200 (status " + std::to_string(status) + "): " + dl_last_error_string());
    ++g_launches;
}

bool ordinary(PyObject *o) { return THPVariable_CheckExact(o); }
bool plain(const Tensor &t, at::ScalarType type, int64_t dim, const c10::Device &device) {
    return t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.device() == device && t.scalar_type() == type && t.dim() == dim;
}
bool vector_of(const Tensor &t, at::ScalarType type, int64_t n, const c10::Device &device) {
    return plain(t, type, 1, device) && t.size(0) == n && t.is_contiguous();
}
bool matrix_of(const Tensor &t, at::ScalarType type, int64_t rows, int64_t cols, const c10::Device &device) {
    return plain(t, type, 2, device) && t.size(0) == rows && t.size(1) == cols && t.is_contiguous();
}
// Whether something wants to see every operation, which these nodes would pass by.
bool observed() {
    return c10::impl::tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode) || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           at::impl::torch_function_mode_enabled() || torch::jit::tracer::isTracing();
}
bool aligned16(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
// A [batch][features] tensor as it is stored between layers: feature-major, and no view.
Tensor feature_major(int64_t batch, int64_t features, const Tensor &like) {
    return at::empty_strided({batch, features}, {1, batch}, like.options().requires_grad(false));
}

struct Layer {
    Tensor a, b, start, plan, grad_out, walk;  // grad_out, walk: may be undefined
    double grad_factor;
    bool complete;
    bool transposed;  // x is batch-major: the library transposes it
};

PyObject *wrap(const Tensor &t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_RETURN_NONE;
}

struct LayerNode : torch::autograd::Function<LayerNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &input, const Tensor &weights, const Layer &l) {
        const int64_t batch = input.size(0), n_in = input.size(1), n_out = weights.size(0);
        Tensor x = input.t();
        void *stream = stream_of(input);
        if (l.transposed) {
            x = at::empty({n_in, batch}, input.options().requires_grad(false));
            check(dl_transpose_f32(input.data_ptr<float>(), x.data_ptr<float>(), batch, n_in, stream));
        } else if (!x.is_contiguous()) {
            x = x.contiguous();
        }
        Tensor y = feature_major(batch, n_out, input), coef = at::empty({n_out, 4}, input.options().requires_grad(false));
        if (l.walk.defined())
            check(dl_forward_walk_f32(x.data_ptr<float>(), weights.data_ptr<float>(), DL_W_LOGITS, y.data_ptr<float>(), coef.data_ptr<float>(),
                                      l.walk.data_ptr<int32_t>(), l.walk.size(0), n_in, n_out, batch, DL_LAUNCH_OVERLAP_SETUP, stream));
        else
            check(dl_forward_f32(x.data_ptr<float>(), l.a.data_ptr<int64_t>(), l.b.data_ptr<int64_t>(), weights.data_ptr<float>(), DL_W_LOGITS,
                                 y.data_ptr<float>(), coef.data_ptr<float>(), n_in, n_out, batch, DL_LAUNCH_OVERLAP_SETUP, stream));
        ctx->save_for_backward({x, weights, l.a, l.b, l.start, l.plan, coef});
        ctx->saved_data["grad_factor"] = l.grad_factor;
        ctx->saved_data["complete"] = l.complete;
        if (l.grad_out.defined()) ctx->saved_data["grad_out"] = l.grad_out;
        if (l.walk.defined()) ctx->saved_data["walk"] = l.walk;
        return y;
    }

    // Whether the weights' gradient is somebody's business beside autograd's, or a stream is set for it.
    static bool managed(const Tensor &weights) {
        PyObject *stream = PyDict_GetItemString(g_module_dict, "_backward_w_stream");
        if (stream != nullptr && stream != Py_None) return true;
        PyObject *w = THPVariable_Wrap(weights);
        if (w == nullptr) throw python_error();
        PyObject *dict = PyObject_GenericGetDict(w, nullptr);
        const bool found = dict != nullptr && (PyDict_GetItemString(dict, "_dl_adam") != nullptr || PyDict_GetItemString(dict, "_dl_exchange") != nullptr);
        if (dict == nullptr) PyErr_Clear();
        Py_XDECREF(dict);
        Py_DECREF(w);
        return found;
    }

    static variable_list in_python(AutogradContext *ctx, const variable_list &saved, const Tensor &grad_y, const Tensor &grad_out, const Tensor &walk,
                                   bool want_x, bool want_w) {
        PyObject *run = PyDict_GetItemString(g_module_dict, "_backward_of_node");
        TORCH_CHECK(run != nullptr, "difflogic_b200: difflogic._backward_of_node is missing");
        THPObjectPtr args(PyTuple_New(13));
        if (!args) throw python_error();
        for (int i = 0; i < 7; ++i) PyTuple_SET_ITEM(args.get(), i, wrap(saved[i]));
        PyTuple_SET_ITEM(args.get(), 7, wrap(grad_y));
        PyTuple_SET_ITEM(args.get(), 8, PyFloat_FromDouble(ctx->saved_data["grad_factor"].toDouble()));
        PyTuple_SET_ITEM(args.get(), 9, wrap(grad_out));
        PyTuple_SET_ITEM(args.get(), 10, walk.defined() ? Py_BuildValue("(NO)", wrap(walk), ctx->saved_data["complete"].toBool() ? Py_True : Py_False)
                                                       : Py_NewRef(Py_None));
        PyTuple_SET_ITEM(args.get(), 11, PyBool_FromLong(want_x));
        PyTuple_SET_ITEM(args.get(), 12, PyBool_FromLong(want_w));
        THPObjectPtr got(PyObject_CallObject(run, args.get()));
        if (!got) throw python_error();
        variable_list out(3);
        for (int i = 0; i < 2; ++i) {
            PyObject *t = PyTuple_GET_ITEM(got.get(), i);
            if (t != Py_None) out[i] = THPVariable_Unpack(t);
        }
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weights = saved[1], &start = saved[4], &plan = saved[5], &coef = saved[6];
        const int64_t n_in = x.size(0), batch = x.size(1), n_out = weights.size(0);
        auto kept = [&](const char *name) {
            auto it = ctx->saved_data.find(name);
            return it == ctx->saved_data.end() ? Tensor() : it->second.toTensor();
        };
        const Tensor grad_out = kept("grad_out"), walk = kept("walk");
        const c10::cuda::CUDAGuard guard(x.device());
        Tensor gy = grads[0].t();
        if (!gy.is_contiguous()) gy = gy.contiguous();
        variable_list out(3);
        {
            const WithGil gil;
            if (managed(weights)) {
                out = in_python(ctx, saved, gy, grad_out, walk, want_x, want_w);
                if (out[0].defined()) out[0] = out[0].t();
                return out;
            }
        }
        // what the hooks for saved tensors handed back, and the gradient, are what the kernels take
        const c10::Device device = x.device();
        TORCH_CHECK(matrix_of(x, at::kFloat, n_in, batch, device) && matrix_of(weights, at::kFloat, n_out, 16, device) &&
                        matrix_of(coef, at::kFloat, n_out, 4, device) && matrix_of(gy, at::kFloat, n_out, batch, device) &&
                        vector_of(saved[2], at::kLong, n_out, device) && vector_of(saved[3], at::kLong, n_out, device) &&
                        vector_of(start, at::kLong, n_in + 1, device) && matrix_of(plan, at::kInt, 2 * n_out, 2, device),
                    "difflogic_b200: the backward pass of a LogicLayer got tensors of other types, sizes or layouts than its forward pass");
        const float *xp = x.data_ptr<float>(), *gp = gy.data_ptr<float>(), *cp = coef.data_ptr<float>();
        const float scale = (float)ctx->saved_data["grad_factor"].toDouble();
        void *stream = stream_of(x);
        Tensor gx, gw;
        if (want_x) gx = at::empty({n_in, batch}, x.options().requires_grad(false));
        if (want_w) gw = grad_out.defined() ? grad_out.view(grad_out.sizes()) : at::empty({n_out, 16}, x.options().requires_grad(false));
        float *gxp = want_x ? gx.data_ptr<float>() : nullptr, *gwp = want_w ? gw.data_ptr<float>() : nullptr;
        if (walk.defined() && want_w && (!want_x || ctx->saved_data["complete"].toBool()) && aligned16(weights) && aligned16(gw)) {
            check(dl_backward_walk_f32(xp, gp, cp, weights.data_ptr<float>(), gwp, gxp, scale, walk.data_ptr<int32_t>(), walk.size(0),
                                       ctx->saved_data["complete"].toBool() ? 1 : 0, n_in, n_out, batch, 1, nullptr, nullptr, 0.f, 0.f, 0.f, 0.f, 1.f,
                                       nullptr, DL_LAUNCH_OVERLAP_SETUP, stream));
        } else {
            if (want_x)
                check(dl_backward_x_f32(xp, cp, gp, start.data_ptr<int64_t>(), plan.data_ptr<int32_t>(), scale, gxp, n_in, n_out, batch,
                                        DL_LAUNCH_OVERLAP_SETUP, stream));
            if (want_w)
                check(dl_backward_w_f32(xp, saved[2].data_ptr<int64_t>(), saved[3].data_ptr<int64_t>(), gp, weights.data_ptr<float>(), DL_W_LOGITS, gwp,
                                        n_in, n_out, batch, DL_LAUNCH_OVERLAP_SETUP, stream));
        }
        if (want_x) out[0] = gx.t();
        if (want_w) out[1] = gw;
        return out;
    }
};

struct GroupSumNode : torch::autograd::Function<GroupSumNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &input, const Tensor &workspace, int64_t k, double tau) {
        const int64_t batch = input.size(0), n = input.size(1);
        Tensor x = input.t();
        if (!x.is_contiguous()) x = x.contiguous();
        Tensor out = at::empty({batch, k}, input.options().requires_grad(false));
        check(dl_groupsum_f32(x.data_ptr<float>(), out.data_ptr<float>(), workspace.data_ptr(), n, batch, k, (float)tau, stream_of(input)));
        ctx->saved_data["n"] = n;
        ctx->saved_data["tau"] = tau;
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor grad = grads[0].contiguous();
        const int64_t n = ctx->saved_data["n"].toInt(), batch = grad.size(0), k = grad.size(1);
        TORCH_CHECK(matrix_of(grad, at::kFloat, batch, k, grad.device()), "difflogic_b200: the gradient of a GroupSum must be float32 on a CUDA device");
        const c10::cuda::CUDAGuard guard(grad.device());
        Tensor gx = at::empty({n, batch}, grad.options().requires_grad(false));
        check(dl_groupsum_backward_f32(grad.data_ptr<float>(), gx.data_ptr<float>(), n, batch, k, (float)ctx->saved_data["tau"].toDouble(), stream_of(grad)));
        return {gx.t(), Tensor(), Tensor(), Tensor()};
    }
};

// layer(x, weights, a, b, start, plan, grad_factor, grad_out | None, walk entries | None, walk gives grad_x) -> output, or None
PyObject *layer(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 10) {
        PyErr_SetString(PyExc_TypeError, "layer: ten arguments");
        return nullptr;
    }
    for (int i = 0; i < 6; ++i)
        if (!ordinary(args[i])) Py_RETURN_NONE;
    const Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
    const c10::Device device = x.device();
    if (!plain(x, at::kFloat, 2, device) || x.size(0) == 0 || x.size(1) == 0 || w.dim() != 2 || w.size(0) == 0 ||
        !matrix_of(w, at::kFloat, w.size(0), 16, device))
        Py_RETURN_NONE;
    const int64_t n_in = x.size(1), n_out = w.size(0);
    Layer l = {THPVariable_Unpack(args[2]), THPVariable_Unpack(args[3]), THPVariable_Unpack(args[4]), THPVariable_Unpack(args[5])};
    if (!vector_of(l.a, at::kLong, n_out, device) || !vector_of(l.b, at::kLong, n_out, device) || !vector_of(l.start, at::kLong, n_in + 1, device) ||
        !matrix_of(l.plan, at::kInt, 2 * n_out, 2, device))
        Py_RETURN_NONE;
    l.grad_factor = PyFloat_AsDouble(args[6]);
    if (l.grad_factor == -1. && PyErr_Occurred()) return nullptr;
    if (args[7] != Py_None) {
        if (!ordinary(args[7])) Py_RETURN_NONE;
        l.grad_out = THPVariable_Unpack(args[7]);
        if (!matrix_of(l.grad_out, at::kFloat, n_out, 16, device)) Py_RETURN_NONE;
    }
    if (args[8] != Py_None) {
        if (!ordinary(args[8])) Py_RETURN_NONE;
        l.walk = THPVariable_Unpack(args[8]);
        if (!matrix_of(l.walk, at::kInt, l.walk.size(0), 2, device)) Py_RETURN_NONE;
    }
    l.complete = args[9] == Py_True;
    if (observed() || x._fw_grad(0).defined() || w._fw_grad(0).defined()) Py_RETURN_NONE;
    l.transposed = !x.t().is_contiguous() && x.is_contiguous();
    Tensor y;
    {
        const WithoutGil nogil;
        const c10::cuda::CUDAGuard guard(device);
        y = LayerNode::apply(x, w, l);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// group_sum(x, workspace, k, tau) -> output, or None
PyObject *group_sum(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 4) {
        PyErr_SetString(PyExc_TypeError, "group_sum: four arguments");
        return nullptr;
    }
    if (!ordinary(args[0]) || !ordinary(args[1])) Py_RETURN_NONE;
    const Tensor &x = THPVariable_Unpack(args[0]), &workspace = THPVariable_Unpack(args[1]);
    const long long k = PyLong_AsLongLong(args[2]);
    const double tau = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!plain(x, at::kFloat, 2, x.device()) || x.numel() == 0 || k <= 0 || x.size(1) % k != 0 || observed() || x._fw_grad(0).defined()) Py_RETURN_NONE;
    Tensor y;
    {
        const WithoutGil nogil;
        const c10::cuda::CUDAGuard guard(x.device());
        y = GroupSumNode::apply(x, workspace, (int64_t)k, tau);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// -- dense layers -----------------------------------------------------------------------------------------------------------------
// What denselayer.py's Python functions do, with its messages left to them.

struct Matrix {   // a 2-D tensor as the kernels read it: its rows apart, or its columns
    Tensor t;
    int64_t pitch;
    bool feature_major;
};
Matrix readable(const Tensor &t) {
    const int64_t rows = t.size(0), cols = t.size(1), s0 = t.stride(0), s1 = t.stride(1);
    if ((s1 == 1 || cols == 1) && (s0 >= cols || rows == 1)) return {t, rows > 1 ? s0 : cols, false};
    if ((s0 == 1 || rows == 1) && (s1 >= rows || cols == 1)) return {t, cols > 1 ? s1 : rows, true};
    return {t.contiguous(), cols, false};
}
int kind_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2; }
Tensor bytes(int64_t n, const Tensor &like) { return n > 0 ? at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor(); }
void *pointer(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

struct DenseOut {
    Tensor y, slope, x_planes, w_planes;
    Matrix x;
};
DenseOut dense_forward(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &residual, int act, bool feature_major, bool want_slope) {
    const int64_t batch = x.size(0), inner = x.size(1), outer = w.size(0);
    const int kind = kind_of(x.scalar_type()) | dl_matmul_choice();
    const auto options = x.options().requires_grad(false);
    DenseOut o;
    o.y = feature_major ? at::empty_strided({batch, outer}, {1, batch}, options) : at::empty({batch, outer}, options);
    if (want_slope && act != DL_ACT_NONE) o.slope = at::empty({batch * outer}, options.dtype(x.scalar_type() == at::kBFloat16 ? at::kHalf : at::kFloat));
    o.x = readable(x);
    int64_t sizes[3];
    dl_dense_forward_sizes(o.x.t.data_ptr(), o.x.pitch, o.x.feature_major, w.data_ptr(), batch, inner, outer, feature_major, kind, sizes);
    o.x_planes = bytes(sizes[0], x);
    o.w_planes = bytes(sizes[1], x);
    const Tensor work = bytes(sizes[2], x);
    check(dl_dense_forward(o.x.t.data_ptr(), o.x.pitch, o.x.feature_major, w.data_ptr(), pointer(bias), pointer(residual),
                           residual.defined() ? residual.stride(0) : 0, residual.defined() ? residual.stride(1) : 0, act, o.y.data_ptr(), feature_major,
                           pointer(o.slope), pointer(o.x_planes), pointer(o.w_planes), pointer(work), batch, inner, outer, kind, stream_of(x)));
    return o;
}

// The planes of an operand, as its products read them.
Tensor lay_out(const Matrix &m) {
    const int64_t rows = m.t.size(m.feature_major), cols = m.t.size(!m.feature_major);
    const int kind = kind_of(m.t.scalar_type());
    const Tensor planes = bytes(dl_dense_planes_bytes(rows, cols, kind), m.t);
    check(dl_dense_lay_out(m.t.data_ptr(), rows, cols, m.pitch, kind, planes.data_ptr(), stream_of(m.t)));
    return planes;
}

struct DenseNode : torch::autograd::Function<DenseNode> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &b, const std::optional<Tensor> &r,
                          int64_t act, bool feature_major) {
        const Tensor bias = b.value_or(Tensor()), residual = r.value_or(Tensor());
        DenseOut o = dense_forward(x, w, bias, residual, (int)act, feature_major, true);
        ctx->set_materialize_grads(false);
        bool keep_x = !o.x_planes.defined(), keep_w = !o.w_planes.defined();
        if (x.scalar_type() == at::kFloat && keep_w) {
            // Few samples.  An optimizer's kernels may change fp32 parameters before the backward pass, without autograd's version counters: it
            // gets the values that were read here, laid out now as it would do itself.
            if (w.requires_grad()) o.x_planes = lay_out(o.x);
            if (x.requires_grad()) o.w_planes = lay_out({w, w.size(1), false});
            keep_x = keep_w = false;
        }
        // what was laid out for the product serves the backward pass too, in place of the tensor itself
        ctx->save_for_backward({keep_x ? o.x.t : Tensor(), keep_w ? w : Tensor(), o.x_planes, o.w_planes, o.slope});
        ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), x.size(1), w.size(0), o.x.pitch, o.x.feature_major, feature_major, b.has_value(), r.has_value()};
        // their alignment decided what was laid out
        ctx->saved_data["at"] = std::vector<int64_t>{(int64_t)o.x.t.data_ptr(), (int64_t)w.data_ptr()};
        return o.y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(6);
        Tensor gy = grads[0];
        if (!gy.defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &x_planes = saved[2], &w_planes = saved[3], &slope = saved[4];
        const auto sizes = ctx->saved_data["sizes"].toIntVector(), at = ctx->saved_data["at"].toIntVector();
        const int64_t batch = sizes[0], inner = sizes[1], outer = sizes[2], pitch = sizes[3];
        const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_b = sizes[6] && ctx->needs_input_grad(2);
        const c10::cuda::CUDAGuard guard(gy.device());
        if (want_x || want_w || want_b) {
            TORCH_CHECK(gy.dim() == 2 && gy.size(0) == batch && gy.size(1) == outer && gy.is_cuda() &&
                            (!x.defined() || (x.scalar_type() == gy.scalar_type() && x.device() == gy.device() && x.dim() == 2 && x.size(0) == batch &&
                                              x.size(1) == inner && readable(x).t.is_same(x))) &&
                            (!w.defined() || matrix_of(w, gy.scalar_type(), outer, inner, gy.device())),
                        "difflogic_b200: the backward pass of a dense layer got tensors of other types, sizes or layouts than its forward pass");
            const at::NoGradGuard no_grad;
            Tensor g = gy;
            bool feature_major = false;
            if (!g.is_contiguous()) {
                feature_major = g.t().is_contiguous();
                if (!feature_major) g = g.contiguous();
            }
            if (slope.defined() && feature_major != (bool)sizes[5] && batch > 1 && outer > 1) {
                feature_major = sizes[5];
                g = feature_major ? g.t().contiguous().t() : g.contiguous();
            }
            const auto options = gy.options().requires_grad(false);
            if (want_x) out[0] = at::empty({batch, inner}, options);
            if (want_w) out[1] = at::empty({outer, inner}, options);
            if (want_b) out[2] = at::empty({outer}, options);
            const Matrix read = x.defined() ? readable(x) : Matrix{Tensor(), pitch, (bool)sizes[4]};
            const void *px = x.defined() ? x.data_ptr() : (const void *)at[0], *pw = w.defined() ? w.data_ptr() : (const void *)at[1];
            const int kind = kind_of(gy.scalar_type()) | dl_matmul_choice();
            const Tensor work = bytes(dl_dense_backward_workspace_bytes(g.data_ptr(), feature_major, slope.defined(), px, read.pitch, read.feature_major,
                                                                        pw, want_w && !x_planes.defined(), want_x && !w_planes.defined(), batch, inner,
                                                                        outer, kind),
                                      gy);
            check(dl_dense_backward(g.data_ptr(), feature_major, pointer(slope), px, read.pitch, read.feature_major, pw, pointer(x_planes),
                                    pointer(w_planes), pointer(out[0]), pointer(out[1]), pointer(out[2]), pointer(work), batch, inner, outer, kind,
                                    stream_of(gy)));
        }
        if (sizes[7] && ctx->needs_input_grad(sizes[6] ? 3 : 2)) out[3] = gy;   // counted without what was not given
        if (at::GradMode::is_enabled()) {   // a graph of the gradients is wanted: it would end here without a word
            variable_list once(out.begin(), out.begin() + 3);
            for (Tensor &t : once)
                if (t.defined()) t = t.detach().requires_grad_(true);
            once = (*std::make_shared<torch::autograd::DelayedError>("difflogic_b200: dense layers are differentiable once", 3))(std::move(once));
            std::copy(once.begin(), once.end(), out.begin());
        }
        return out;
    }
};

// A leaf of a graph that lives has its accumulator on the stream that the graph was made on, and a captured backward pass brings that
// stream into the capture.  The default stream cannot be brought in, and the process ends: refused here instead.  t is a leaf, or made of
// one by operations on it alone (views, reshaping, copies).
void refuse_older_graph(const Tensor &t) {
    if (!t.defined() || !t.requires_grad()) return;
    std::shared_ptr<torch::autograd::Node> node = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn();
    while (node != nullptr && dynamic_cast<torch::autograd::AccumulateGrad *>(node.get()) == nullptr)
        node = node->num_outputs() == 1 ? node->next_edge(0).function : nullptr;
    if (node == nullptr) return;
    const auto stream = node->stream();
    TORCH_CHECK(!stream || *stream != c10::cuda::getDefaultCUDAStream(t.device().index()).unwrap(),
                "difflogic_b200: dense is captured while a graph of the same tensors, made on the default stream, is alive; delete its outputs before the "
                "capture");
}
bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

// refuse_older_graphs(x, weight, bias | None, residual | None): for calls that take the Python functions
PyObject *refuse_older_graphs(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t i = 0; i < count; ++i) {
        if (!THPVariable_Check(args[i])) continue;
        const Tensor &t = THPVariable_Unpack(args[i]);
        if (!t.is_cuda()) continue;
        const c10::cuda::CUDAGuard guard(t.device());
        if (capturing()) refuse_older_graph(t);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// dense(x, weight, bias | None, residual | None, activation, feature_major) -> output, or None
PyObject *dense(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 6) {
        PyErr_SetString(PyExc_TypeError, "dense: six arguments");
        return nullptr;
    }
    if (!ordinary(args[0]) || !ordinary(args[1])) Py_RETURN_NONE;
    Tensor x = THPVariable_Unpack(args[0]), residual, bias;
    const Tensor &w = THPVariable_Unpack(args[1]);
    const c10::Device device = x.device();
    const at::ScalarType type = x.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) Py_RETURN_NONE;
    if (!plain(x, type, x.dim(), device) || x.dim() < 1 || x.numel() == 0 || w.dim() != 2 || w.size(0) == 0 ||
        !matrix_of(w, type, w.size(0), x.size(-1), device))
        Py_RETURN_NONE;
    const int64_t outer = w.size(0);
    if (args[2] != Py_None) {
        if (!ordinary(args[2])) Py_RETURN_NONE;
        bias = THPVariable_Unpack(args[2]);
        if (!vector_of(bias, type, outer, device)) Py_RETURN_NONE;
    }
    auto sizes = x.sizes().vec();
    sizes.back() = outer;
    if (args[3] != Py_None) {
        if (!ordinary(args[3])) Py_RETURN_NONE;
        residual = THPVariable_Unpack(args[3]);
        if (!plain(residual, type, x.dim(), device) || residual.sizes() != at::IntArrayRef(sizes)) Py_RETURN_NONE;
    }
    const long act = PyLong_AsLong(args[4]);
    if (act == -1 && PyErr_Occurred()) return nullptr;
    const int feature_major = PyObject_IsTrue(args[5]);
    if (feature_major < 0) return nullptr;
    if (act < DL_ACT_NONE || act > DL_ACT_GELU || (feature_major && x.dim() != 2)) Py_RETURN_NONE;
    if (observed() || x._fw_grad(0).defined() || w._fw_grad(0).defined() || (bias.defined() && bias._fw_grad(0).defined()) ||
        (residual.defined() && residual._fw_grad(0).defined()))
        Py_RETURN_NONE;
    Tensor y;
    {
        const WithoutGil nogil;
        const c10::cuda::CUDAGuard guard(device);
        const bool graph = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad()) ||
                                                          (residual.defined() && residual.requires_grad()));
        if (graph && capturing())
            for (const Tensor &t : {x, w, bias, residual}) refuse_older_graph(t);
        if (x.dim() != 2) {
            x = x.reshape({-1, x.size(-1)});
            if (residual.defined()) residual = residual.reshape({-1, outer});
        }
        const auto given = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
        y = graph ? DenseNode::apply(x, w, given(bias), given(residual), (int64_t)act, (bool)feature_major)
                  : dense_forward(x, w, bias, residual, (int)act, feature_major, false).y;
        if (sizes.size() != 2) y = y.reshape(sizes);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// -- orthogonalised updates ---------------------------------------------------------------------------------------------------------
// What ops.muon_step does once it has its numbers: checks, addresses, workspace and launch, 2 us for 15 tensors that take the interpreter 15.

// The tensor of item i where it is one, float32, contiguous, two-dimensional and on `device`; else null.
const Tensor *matrix_at(PyObject *list, Py_ssize_t i, const c10::Device &device) {
    PyObject *o = PyList_GET_ITEM(list, i);
    if (!ordinary(o)) return nullptr;
    const Tensor &t = THPVariable_Unpack(o);
    return plain(t, at::kFloat, 2, device) && t.is_contiguous() ? &t : nullptr;
}

// muon_step(weights, grads, momenta, lr, momentum, nesterov, weight_decay, steps, address of the coefficients, eps) -> True, or None
PyObject *muon_step(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 10) {
        PyErr_SetString(PyExc_TypeError, "muon_step: ten arguments");
        return nullptr;
    }
    for (int i = 0; i < 3; ++i)
        if (!PyList_Check(args[i]) || PyList_GET_SIZE(args[i]) != PyList_GET_SIZE(args[0])) Py_RETURN_NONE;
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    if (n == 0 || !ordinary(PyList_GET_ITEM(args[0], 0))) Py_RETURN_NONE;
    const c10::Device device = THPVariable_Unpack(PyList_GET_ITEM(args[0], 0)).device();
    if (!device.is_cuda()) Py_RETURN_NONE;
    std::vector<int64_t> table, written;
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor *w = matrix_at(args[0], i, device), *g = matrix_at(args[1], i, device), *m = matrix_at(args[2], i, device);
        if (w == nullptr || g == nullptr || m == nullptr || w->sizes() != g->sizes() || w->sizes() != m->sizes()) Py_RETURN_NONE;
        if (w->numel() == 0) continue;
        for (const Tensor *t : {w, g, m}) table.push_back((int64_t)t->data_ptr());
        table.push_back(w->size(0));
        table.push_back(w->size(1));
        written.push_back((int64_t)w->data_ptr());
        written.push_back((int64_t)m->data_ptr());
    }
    std::sort(written.begin(), written.end());
    if (table.empty() || std::adjacent_find(written.begin(), written.end()) != written.end()) Py_RETURN_NONE;
    const double lr = PyFloat_AsDouble(args[3]), momentum = PyFloat_AsDouble(args[4]), decay = PyFloat_AsDouble(args[6]), eps = PyFloat_AsDouble(args[9]);
    const int nesterov = PyObject_IsTrue(args[5]);
    const long steps = PyLong_AsLong(args[7]);
    const float *coefficients = reinterpret_cast<const float *>(PyLong_AsUnsignedLongLong(args[8]));
    if (PyErr_Occurred()) return nullptr;
    if (observed()) Py_RETURN_NONE;
    const Tensor &first = THPVariable_Unpack(PyList_GET_ITEM(args[0], 0));
    {
        const WithoutGil nogil;
        const c10::cuda::CUDAGuard guard(device);
        const int64_t matrices = (int64_t)table.size() / 5;
        const Tensor work = bytes(dl_muon_workspace_bytes(table.data(), matrices), first);
        check(dl_muon_step_f32(table.data(), matrices, lr, momentum, nesterov, decay, (int)steps, coefficients, eps, pointer(work), stream_of(first)));
    }
    // in place, for whoever has kept these for a backward pass; tensors of inference mode have no counters
    for (Py_ssize_t i = 0; i < n; ++i)
        for (int j : {0, 2}) {
            const Tensor &t = THPVariable_Unpack(PyList_GET_ITEM(args[j], i));
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// orthogonalize(x, steps, address of the coefficients, eps) -> the result, or None
PyObject *orthogonalize(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 4) {
        PyErr_SetString(PyExc_TypeError, "orthogonalize: four arguments");
        return nullptr;
    }
    if (!ordinary(args[0])) Py_RETURN_NONE;
    const Tensor &x = THPVariable_Unpack(args[0]);
    const at::ScalarType type = x.scalar_type();
    if ((type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) || x.dim() < 2 || x.numel() == 0 || !plain(x, type, x.dim(), x.device()) ||
        !x.is_contiguous() || observed() || x._fw_grad(0).defined())
        Py_RETURN_NONE;
    const long steps = PyLong_AsLong(args[1]);
    const float *coefficients = reinterpret_cast<const float *>(PyLong_AsUnsignedLongLong(args[2]));
    const double eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) return nullptr;
    Tensor out;
    {
        const WithoutGil nogil;
        const c10::cuda::CUDAGuard guard(x.device());
        const at::NoGradGuard no_grad;
        out = at::empty_like(x, x.options().requires_grad(false));
        const int64_t rows = x.size(-2), cols = x.size(-1), batch = x.numel() / (rows * cols);
        const int kind = kind_of(type) | dl_matmul_choice();
        const Tensor work = bytes(dl_orthogonalize_workspace_bytes(batch, rows, cols, kind), x);
        check(dl_orthogonalize(x.data_ptr(), out.data_ptr(), batch, rows, cols, kind, (int)steps, coefficients, eps, pointer(work), stream_of(x)));
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

PyObject *launches(PyObject *, PyObject *) { return PyLong_FromLongLong(g_launches.load()); }

// connect(dict of difflogic.py)
PyObject *connect(PyObject *, PyObject *dict) {
    if (!PyDict_Check(dict)) {
        PyErr_SetString(PyExc_TypeError, "connect: a dict");
        return nullptr;
    }
    Py_XDECREF(g_module_dict);
    g_module_dict = Py_NewRef(dict);
    Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {{"layer", (PyCFunction)(void *)layer, METH_FASTCALL, nullptr},
                          {"group_sum", (PyCFunction)(void *)group_sum, METH_FASTCALL, nullptr},
                          {"dense", (PyCFunction)(void *)dense, METH_FASTCALL, nullptr},
                          {"refuse_older_graphs", (PyCFunction)(void *)refuse_older_graphs, METH_FASTCALL, nullptr},
                          {"muon_step", (PyCFunction)(void *)muon_step, METH_FASTCALL, nullptr},
                          {"orthogonalize", (PyCFunction)(void *)orthogonalize, METH_FASTCALL, nullptr},
                          {"launches", launches, METH_NOARGS, nullptr},
                          {"connect", connect, METH_O, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "dl_autograd", nullptr, -1, kMethods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit_dl_autograd(void) { return PyModule_Create(&kModule); }
