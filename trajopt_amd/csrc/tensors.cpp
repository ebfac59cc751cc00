// Python module `_tensors`: the entry points of the C ABI that work on torch tensors, called with the tensors themselves.
// Reading the address, type, layout and device of a tensor from Python costs half a microsecond or more, which for lists of
// hundreds of gradients is many times what the kernels take; here it costs nanoseconds.  The library is the one trajopt_amd._lib
// has loaded: bind() receives the addresses of its functions.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>

#include <vector>

#include "../../include/mppi_hip.h"

namespace {

decltype(&mppi_last_error) last_error;
decltype(&mppi_draw_workspace) draw_workspace;
decltype(&mppi_draw_from_returns) draw_from_returns;
decltype(&mppi_gradient_workspace) gradient_workspace;
decltype(&mppi_gradient_norm) gradient_norm;
decltype(&mppi_clip_gradients) clip_gradients;
PyObject* library_error;              // trajopt_amd._lib.MppiError

struct Raised {};                     // a Python exception has been set

[[noreturn]] void raise(PyObject* type, const std::string& message) {
    PyErr_SetString(type, message.c_str());
    throw Raised();
}
void check(int rc) {
    if (rc == 0) return;
    const char* m = last_error();
    raise(library_error, "mppi_hip error " + std::to_string(rc) + ": " + (m ? m : "?"));
}
std::string text(at::IntArrayRef shape) {
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); i++) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + (shape.size() == 1 ? ",)" : ")");
}
std::string text(const at::Device& d) { return d.str(); }

int element_type(const at::Tensor& t, bool doubles) {
    switch (t.scalar_type()) {
    case at::kFloat: return MPPI_F32;
    case at::kHalf: return MPPI_F16;
    case at::kBFloat16: return MPPI_BF16;
    case at::kDouble: if (doubles) return MPPI_F64; break;
    default: break;
    }
    raise(PyExc_TypeError, std::string("unsupported element type ") + c10::toString(t.scalar_type()));
}
void* stream_of(const at::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

// (straight to the allocator: at::empty goes through the dispatcher first, half a microsecond of a call of five)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Device& d) { return at::Tensor(at::detail::empty_cuda(sizes, type, d, std::nullopt)); }

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }

// None of these functions has a derivative.  A tensor that autograd would have to follow through one is refused: the result would look
// like a constant, and a write would go past the graph.  What is recorded is asked for once per call: a tensor's own forward gradient
// takes 24 ns to look for (384 views and their outputs: 50 us per call with that for each, 34 without), and none has one outside a
// dual level.  Whether a view requires grad, which asks its base as well, takes 4 ns; an ordinary gradient is told by a null pointer.
struct Recorded {
    const bool backward = c10::GradMode::is_enabled(), forward = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
    void refuse(const at::Tensor& t, const char* what) const {
        if (!t.unsafeGetTensorImpl()->autograd_meta()) return;           // (autograd has never met it)
        if ((backward && t.requires_grad()) || (forward && t._fw_grad(0).defined()))
            raise(PyExc_RuntimeError, std::string(what) + ": part of a graph, and this function has no derivative (detach() it, or call under torch.no_grad())");
    }
};

// a draw's parameter: a number, or a tensor of one value per row
struct PerRow {
    at::Tensor held;
    const void* data = nullptr;
    PerRow(PyObject* o, const char* name, int64_t rows, at::ScalarType type, const at::Device& device, const Recorded& recorded) {
        if (!is_tensor(o)) return;
        const at::Tensor& t = tensor(o);
        if (t.device() != device) raise(PyExc_ValueError, std::string(name) + " lies on " + text(t.device()) + ", the returns on " + text(device));
        if (t.dim() != 1 || t.size(0) != rows)
            raise(PyExc_ValueError, std::string(name) + ": one value per row, shape (" + std::to_string(rows) + ",), got " + text(t.sizes()));
        if (t.is_complex() || (type == at::kLong && t.is_floating_point()))
            raise(PyExc_TypeError, std::string(name) + ": unsupported element type " + c10::toString(t.scalar_type()));
        if (type == at::kDouble) recorded.refuse(t, name);
        held = t.detach().to(type).contiguous().resolve_neg();
        data = held.const_data_ptr();
    }
};
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised();
    return v;
}
int64_t whole(PyObject* o) {
    PyObject* i = PyNumber_Index(o);
    if (!i) throw Raised();
    const long long v = PyLong_AsLongLong(i);
    Py_DECREF(i);
    if (v == -1 && PyErr_Occurred()) throw Raised();
    return v;
}

// draw(R, u, kappa, top_k, top_p, min_p) -> (index, weight)
PyObject* draw(PyObject* const* args) {
    if (!is_tensor(args[0]) || !is_tensor(args[1])) raise(PyExc_TypeError, "draw_from_returns works on CUDA tensors");
    const at::Tensor &R = tensor(args[0]), &u = tensor(args[1]);
    if (!R.is_cuda() || !u.is_cuda() || R.layout() != at::kStrided || u.layout() != at::kStrided)
        raise(PyExc_TypeError, "draw_from_returns works on CUDA tensors");
    if ((R.dim() != 1 && R.dim() != 2) || u.dim() != R.dim() || (R.dim() == 2 && u.size(0) != R.size(0)))
        raise(PyExc_ValueError, "R is (K,) with u (D,), or (P, K) with u (P, D): got " + text(R.sizes()) + " and " + text(u.sizes()));
    const at::Device device = R.device();
    if (u.device() != device) raise(PyExc_ValueError, "u lies on " + text(u.device()) + ", the returns on " + text(device));
    if (u.scalar_type() != at::kDouble && u.scalar_type() != at::kFloat)
        raise(PyExc_TypeError, std::string("u must be float64 or float32, got ") + c10::toString(u.scalar_type()));
    if (R.is_neg()) raise(PyExc_ValueError, "the returns are a lazily negated view: resolve_neg() them first");
    const Recorded recorded;
    recorded.refuse(R, "the returns");
    const int type = element_type(R, true);
    const bool one = R.dim() == 1;
    const int64_t rows = one ? 1 : R.size(0), K = R.size(one ? 0 : 1), D = u.size(one ? 0 : 1);
    if (rows > INT32_MAX || K > INT32_MAX || D > INT32_MAX)
        raise(PyExc_ValueError, "too many rows, samples or draws: " + std::to_string(rows) + ", " + std::to_string(K) + ", " + std::to_string(D));
    const PerRow kappa(args[2], "kappa", rows, at::kDouble, device, recorded), top_k(args[3], "top_k", rows, at::kLong, device, recorded),
        top_p(args[4], "top_p", rows, at::kDouble, device, recorded), min_p(args[5], "min_p", rows, at::kDouble, device, recorded);
    mppi_draw_filter f;
    f.kappa = kappa.data ? 0.0 : number(args[2]);
    f.top_k = top_k.data ? 0 : whole(args[3]);
    f.top_p = top_p.data ? 1.0 : number(args[4]);
    f.min_p = min_p.data ? 0.0 : number(args[5]);
    f.kappa_of = (const double*)kappa.data; f.top_k_of = (const int64_t*)top_k.data;
    f.top_p_of = (const double*)top_p.data; f.min_p_of = (const double*)min_p.data;
    at::Tensor u64 = u;
    if (u.scalar_type() != at::kDouble || !u.is_contiguous() || u.is_neg()) u64 = u.detach().to(at::kDouble).contiguous().resolve_neg();
    at::Tensor index = fresh(u.sizes(), at::kLong, device);
    at::Tensor weight = fresh(u.sizes(), at::kFloat, device);
    size_t bytes = 0;
    at::Tensor ws;
    if (rows > 0 && K > 0 && D > 0) check(draw_workspace(type, (int32_t)rows, (int32_t)K, &bytes));
    if (bytes) ws = fresh({(int64_t)(bytes + 7) / 8}, at::kDouble, device);
    check(draw_from_returns(device.index(), R.const_data_ptr(), type, (int32_t)rows, (int32_t)K, one ? 0 : R.stride(0), R.stride(one ? 0 : 1),
                            (const double*)u64.const_data_ptr(), (int32_t)D, &f, (int64_t*)index.mutable_data_ptr(),
                            (float*)weight.mutable_data_ptr(), bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(device)));
    PyObject* out = PyTuple_New(2);
    if (!out) throw Raised();
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(index)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(weight)));
    return out;
}

// The tensors of a list, borrowed: `owner` keeps the list alive.
struct List {
    std::vector<const at::Tensor*> t;
    PyObject* owner = nullptr;
    ~List() { Py_XDECREF(owner); }
    List() = default;
    List(const List&) = delete;
    void fill(PyObject* o, const char* what, const Recorded& recorded) {
        PyObject* const* items = &o;
        Py_ssize_t n = 1;
        if (!is_tensor(o)) {
            owner = PySequence_Fast(o, "a list of tensors is needed");
            if (!owner) throw Raised();
            items = PySequence_Fast_ITEMS(owner);
            n = PySequence_Fast_GET_SIZE(owner);
        }
        t.reserve(n);
        for (Py_ssize_t i = 0; i < n; i++) {
            if (!is_tensor(items[i])) raise(PyExc_TypeError, std::string(what) + " must be dense CUDA tensors");
            const at::Tensor& x = tensor(items[i]);
            if (!x.is_cuda() || x.layout() != at::kStrided) raise(PyExc_TypeError, std::string(what) + " must be dense CUDA tensors");
            if (!x.is_non_overlapping_and_dense())
                raise(PyExc_ValueError, std::string(what) + " must fill their memory without gaps or overlaps (a slice or an expanded tensor does not)");
            if (x.is_neg()) raise(PyExc_ValueError, std::string(what) + " must not be lazily negated views (resolve_neg())");
            recorded.refuse(x, what);
            t.push_back(&x);
        }
    }
};

// gradients(grads, out or None, norm type, max_norm or None) -> norm
PyObject* gradients(PyObject* const* args) {
    const bool clip = args[3] != Py_None, elsewhere = args[1] != Py_None;
    const Recorded recorded;
    List grads, outs;
    grads.fill(args[0], "gradients", recorded);
    if (grads.t.empty()) raise(PyExc_ValueError, "no gradients");
    if (grads.t.size() > INT32_MAX) raise(PyExc_ValueError, "too many gradients");
    if (elsewhere) outs.fill(args[1], "outputs", recorded);
    const size_t n = grads.t.size();
    if (elsewhere && outs.t.size() != n) raise(PyExc_ValueError, std::to_string(n) + " gradients, " + std::to_string(outs.t.size()) + " outputs");
    const at::Device device = grads.t[0]->device();
    std::vector<const void*> in(n);
    std::vector<void*> out(n);
    std::vector<int64_t> sizes(n);
    std::vector<int32_t> types(n);
    for (size_t i = 0; i < n; i++) {
        const at::Tensor& g = *grads.t[i];
        if (g.device() != device) raise(PyExc_ValueError, "all tensors must lie on one device");
        types[i] = element_type(g, false);
        sizes[i] = g.numel();
        in[i] = g.const_data_ptr();
        if (!clip) continue;
        const at::Tensor& o = elsewhere ? *outs.t[i] : g;
        if (elsewhere) {
            if (o.device() != device) raise(PyExc_ValueError, "all tensors must lie on one device");
            if (o.scalar_type() != g.scalar_type() || o.sizes() != g.sizes() || o.strides() != g.strides())
                raise(PyExc_ValueError, "an output has another shape, type or layout than its gradient");
        }
        out[i] = o.mutable_data_ptr();
    }
    size_t bytes = 0;
    check(gradient_workspace((int32_t)n, &bytes));
    at::Tensor ws = fresh({(int64_t)(bytes + 7) / 8}, at::kDouble, device);
    at::Tensor norm = fresh({}, at::kFloat, device);
    const int32_t kind = (int32_t)whole(args[2]);
    if (clip) {
        const double most = number(args[3]);
        check(clip_gradients(device.index(), (int32_t)n, in.data(), out.data(), sizes.data(), types.data(), kind, most,
                             (float*)norm.mutable_data_ptr(), ws.mutable_data_ptr(), bytes, stream_of(device)));
        for (const at::Tensor* o : elsewhere ? outs.t : grads.t)
            if (!o->is_inference()) o->unsafeGetTensorImpl()->bump_version();        // written in place: autograd has to know
    } else {
        check(gradient_norm(device.index(), (int32_t)n, in.data(), sizes.data(), types.data(), kind, (float*)norm.mutable_data_ptr(),
                            ws.mutable_data_ptr(), bytes, stream_of(device)));
    }
    return THPVariable_Wrap(std::move(norm));
}

// bind(MppiError, addresses of mppi_last_error, ..._draw_workspace, ..._draw_from_returns, ..._gradient_workspace, ..._gradient_norm,
// ..._clip_gradients)
PyObject* bind(PyObject* const* args) {
    void* address[6];
    for (int i = 0; i < 6; i++) {
        address[i] = PyLong_AsVoidPtr(args[1 + i]);
        if (!address[i]) raise(PyExc_ValueError, "null function address");
    }
    Py_INCREF(args[0]);
    Py_XDECREF(library_error);
    library_error = args[0];
    last_error = (decltype(last_error))address[0];
    draw_workspace = (decltype(draw_workspace))address[1];
    draw_from_returns = (decltype(draw_from_returns))address[2];
    gradient_workspace = (decltype(gradient_workspace))address[3];
    gradient_norm = (decltype(gradient_norm))address[4];
    clip_gradients = (decltype(clip_gradients))address[5];
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int N> PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        if (n != N) raise(PyExc_TypeError, "wrong number of arguments");
        if (F != &bind && !library_error) raise(PyExc_RuntimeError, "bind() has not been called");
        return F(args);
    } catch (const Raised&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)())&entry<bind, 7>, METH_FASTCALL, nullptr},
    {"draw", (PyCFunction)(void (*)())&entry<draw, 6>, METH_FASTCALL, nullptr},
    {"gradients", (PyCFunction)(void (*)())&entry<gradients, 4>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
