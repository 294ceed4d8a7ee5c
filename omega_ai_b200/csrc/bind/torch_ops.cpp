// Binding of the operators without a handle (include/omoe.h) for torch tensors.
//
// A call of these operators on a small batch is mostly its way to the GPU: through ctypes, with the checks of the tensors and the
// allocations made in Python, 7 to 19 us of the host against 2 to 10 on the device.  Here the same checks, allocations and
// the call itself take 2.5 to 7.  The entry points are not linked: init() gets their addresses from the library
// that native.py has loaded, so that there is one copy of it in the process.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>
#include <vector>

#include "../../../include/omoe.h"

// The torch and the Python that this is built for; native.build_binding() looks for it in the file.
extern "C" __attribute__((visibility("default"), used)) const char omoe_binding_mark[] = OMOE_BINDING_MARK;

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Entries {
    decltype(&omoe_ops_error) error;
    decltype(&omoe_sort_rows_cap) sort_rows_cap;
    decltype(&omoe_sort_plan) sort_plan;
    decltype(&omoe_sort_rows) sort_rows;
    decltype(&omoe_sort_rows_backward) sort_rows_backward;
    decltype(&omoe_unsort_rows) unsort_rows;
    decltype(&omoe_unsort_rows_backward) unsort_rows_backward;
    decltype(&omoe_layer_norm) layer_norm;
    decltype(&omoe_layer_norm_backward_workspace) layer_norm_backward_workspace;
    decltype(&omoe_layer_norm_backward) layer_norm_backward;
    decltype(&omoe_grad_norm) grad_norm;
    decltype(&omoe_grad_scale) grad_scale;
    decltype(&omoe_grad_clip) grad_clip;
} lib;
PyObject *error_class = nullptr;  // OmoeError(code, message), kept for the life of the process

[[noreturn]] void fail(int code, const std::string &message) {
    py::object e = py::reinterpret_borrow<py::object>(error_class)(code, message);
    PyErr_SetObject(error_class, e.ptr());
    throw py::error_already_set();
}
[[noreturn]] void bad(const std::string &message) { fail(OMOE_ERR_INVALID, message); }
void check(int rc) {
    if (rc != OMOE_OK) fail(rc, lib.error());
}

void init(const py::dict &addresses, const py::object &error) {
    auto at = [&](const char *name, auto &fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>()); };
    at("omoe_ops_error", lib.error);
    at("omoe_sort_rows_cap", lib.sort_rows_cap);
    at("omoe_sort_plan", lib.sort_plan);
    at("omoe_sort_rows", lib.sort_rows);
    at("omoe_sort_rows_backward", lib.sort_rows_backward);
    at("omoe_unsort_rows", lib.unsort_rows);
    at("omoe_unsort_rows_backward", lib.unsort_rows_backward);
    at("omoe_layer_norm", lib.layer_norm);
    at("omoe_layer_norm_backward_workspace", lib.layer_norm_backward_workspace);
    at("omoe_layer_norm_backward", lib.layer_norm_backward);
    at("omoe_grad_norm", lib.grad_norm);
    at("omoe_grad_scale", lib.grad_scale);
    at("omoe_grad_clip", lib.grad_clip);
    if (!error_class) error_class = error.inc_ref().ptr();
}

std::string text(const c10::Device &d) { return d.str(); }
std::string text(at::IntArrayRef sizes) {
    std::string s = "[";
    for (size_t i = 0; i < sizes.size(); i++) s += (i ? ", " : "") + std::to_string(sizes[i]);
    return s + "]";
}

int32_t dtype_of(at::ScalarType t) {
    if (t == at::kFloat) return OMOE_F32;
    if (t == at::kBFloat16) return OMOE_BF16;
    bad(std::string("unsupported dtype ") + c10::toString(t));
}

// The tensors' device, current for the duration of a call, and its current stream.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    void *stream;
    explicit On(const c10::Device &device) {
        if (!device.is_cuda()) bad("tensors must be on a GPU, got " + text(device));
        guard.set_device(device);
        stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    }
};

int32_t fits(int64_t n, const char *name) {
    if (n < 0 || n > INT32_MAX) fail(OMOE_ERR_TOO_LARGE, std::string(name) + ": too large");
    return (int32_t)n;
}

// A [rows, d] matrix on `device`: address, leading dimension and element type.
struct Matrix {
    void *p;
    int64_t ld;
    int32_t dtype;
    Matrix(const Tensor &t, int64_t rows, int64_t d, const char *name, const c10::Device &device) {
        if (t.dim() != 2 || t.size(0) != rows || t.size(1) != d || t.device() != device)
            bad(std::string(name) + ": expected " + text({rows, d}) + " on " + text(device) + ", got " + text(t.sizes()) + " on " + text(t.device()));
        if (t.stride(1) != 1 && d > 1) bad(std::string(name) + ": the elements of a row must be contiguous");
        if (rows > 1 && t.stride(0) < d) bad(std::string(name) + ": rows overlap");
        p = t.data_ptr();
        ld = rows > 1 ? t.stride(0) : d;
        dtype = dtype_of(t.scalar_type());
    }
};

void *vector(const OptTensor &t, int64_t n, const char *name, const c10::Device &device, at::ScalarType type = at::kFloat) {
    if (!t) return nullptr;
    if (t->numel() != n || t->scalar_type() != type || t->device() != device || !t->is_contiguous())
        bad(std::string(name) + ": expected " + std::to_string(n) + " contiguous " + c10::toString(type) + " on " + text(device));
    return t->data_ptr();
}
template <typename T>
T *vec(const OptTensor &t, int64_t n, const char *name, const c10::Device &device, at::ScalarType type = at::kFloat) {
    return static_cast<T *>(vector(t, n, name, device, type));
}

// An uninitialised tensor on the GPU, without the way through the dispatcher.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const c10::Device &device) {
    return Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}
// A tensor that the caller has was written: autograd has to refuse what saved it before.
void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor matrix_or_new(const OptTensor &out, int64_t rows, int64_t d, at::ScalarType type, const c10::Device &device) {
    return out ? *out : fresh({rows, d}, type, device);
}
// A vector of n floats and a second one behind it in the same storage: what lives and dies together takes one allocation.  The second starts on a
// vector of its own, so that both move as vectors where they go next (a list of gradients).
std::pair<Tensor, Tensor> two_floats(int64_t n, const c10::Device &device) {
    const int64_t second = (n + 7) / 8 * 8;
    Tensor a = fresh({second + n}, at::kFloat, device);
    auto b = c10::make_intrusive<c10::TensorImpl>(c10::Storage(a.storage()), a.key_set(), a.dtype());
    b->set_sizes_contiguous({n});
    b->set_storage_offset(second);
    a.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return {a, Tensor(std::move(b))};
}
Tensor floats(at::IntArrayRef sizes, const c10::Device &device) { return fresh(sizes, at::kFloat, device); }

// A call's dtype is for the tensor that it makes: beside `out` it may only repeat that one's.
void agree(const OptTensor &out, const std::optional<at::ScalarType> &dtype) {
    if (out && dtype && out->scalar_type() != *dtype) bad(std::string("dtype: out has ") + c10::toString(out->scalar_type()) + ", not " + c10::toString(*dtype));
}

int64_t width(const Tensor &t, const char *name) {
    if (t.dim() != 2) bad(std::string(name) + ": expected a matrix, got " + text(t.sizes()));
    return t.size(1);
}

// ---- token rows by expert -------------------------------------------------------------------------------------------

struct TokenSort {
    int64_t tokens, top_k, n_experts, row_align, rows_cap;
    Tensor pos, perm, counts, offsets;
    c10::Device device{c10::kCPU};

    TokenSort(int64_t tokens_, int64_t top_k_, int64_t n_experts_, int64_t row_align_, const c10::Device &where)
        : tokens(tokens_), top_k(top_k_), n_experts(n_experts_), row_align(row_align_) {
        auto small = [](int64_t v) { return v < INT32_MIN || v > INT32_MAX ? -1 : (int32_t)v; };
        rows_cap = lib.sort_rows_cap(small(tokens), small(top_k), small(n_experts), small(row_align));
        if (rows_cap < 0)
            fail((int)rows_cap, "sizes out of range: " + std::to_string(tokens) + " tokens, " + std::to_string(top_k) + " picks, " +
                                    std::to_string(n_experts) + " experts, align " + std::to_string(row_align));
        const auto options = at::TensorOptions().dtype(at::kInt).device(where);
        pos = at::empty({tokens, top_k}, options);
        perm = at::empty({rows_cap}, options);
        counts = at::empty({n_experts}, options);
        offsets = at::empty({n_experts + 1}, options);
        device = pos.device();
    }
    omoe_sort c() const {
        return {(int32_t)tokens, (int32_t)top_k, (int32_t)n_experts, (int32_t)row_align, rows_cap, static_cast<int32_t *>(pos.data_ptr()),
                static_cast<int32_t *>(perm.data_ptr()), static_cast<int32_t *>(counts.data_ptr()), static_cast<int32_t *>(offsets.data_ptr())};
    }
    // One value for every pick: [tokens, top_k], or without a shape.
    template <typename T>
    T *of_picks(const OptTensor &t, const char *name, at::ScalarType type) const {
        if (t && t->dim() == 2 && (t->size(0) != tokens || t->size(1) != top_k))
            bad(std::string(name) + ": expected " + text({tokens, top_k}) + ", got " + text(t->sizes()));
        return vec<T>(t, tokens * top_k, name, device, type);
    }
    const float *weights_of(const OptTensor &w) const { return of_picks<float>(w, "weights", at::kFloat); }

    void plan(const Tensor &topk_idx) const {
        const auto *idx = of_picks<int32_t>(topk_idx, "topk_idx", at::kInt);
        const On on(device);
        const omoe_sort p = c();
        check(lib.sort_plan(&p, idx, on.stream));
        for (const Tensor *t : {&pos, &perm, &counts, &offsets}) written(*t);
    }
    Tensor sort(const Tensor &x, const OptTensor &out, const std::optional<at::ScalarType> &dtype) const {
        const int64_t d = width(x, "x");
        agree(out, dtype);
        const Matrix in(x, tokens, d, "x", device);
        const On on(device);
        Tensor to = matrix_or_new(out, rows_cap, d, dtype.value_or(x.scalar_type()), device);
        const Matrix o(to, rows_cap, d, "out", device);
        const omoe_sort p = c();
        check(lib.sort_rows(&p, in.p, in.ld, in.dtype, o.p, o.ld, o.dtype, fits(d, "x"), on.stream));
        if (out) written(to);
        return to;
    }
    Tensor sort_backward(const Tensor &dxs, const OptTensor &out, const std::optional<at::ScalarType> &dtype) const {
        const int64_t d = width(dxs, "dxs");
        agree(out, dtype);
        const Matrix in(dxs, rows_cap, d, "dxs", device);
        const On on(device);
        Tensor to = matrix_or_new(out, tokens, d, dtype.value_or(dxs.scalar_type()), device);
        const Matrix o(to, tokens, d, "out", device);
        const omoe_sort p = c();
        check(lib.sort_rows_backward(&p, in.p, in.ld, in.dtype, o.p, o.ld, o.dtype, fits(d, "dxs"), on.stream));
        if (out) written(to);
        return to;
    }
    Tensor unsort(const Tensor &ys, const OptTensor &weights, const OptTensor &out, const std::optional<at::ScalarType> &dtype) const {
        const int64_t d = width(ys, "ys");
        agree(out, dtype);
        const Matrix in(ys, rows_cap, d, "ys", device);
        const float *w = weights_of(weights);
        const On on(device);
        Tensor to = matrix_or_new(out, tokens, d, dtype.value_or(ys.scalar_type()), device);
        const Matrix o(to, tokens, d, "out", device);
        const omoe_sort p = c();
        check(lib.unsort_rows(&p, in.p, in.ld, in.dtype, w, o.p, o.ld, o.dtype, fits(d, "ys"), on.stream));
        if (out) written(to);
        return to;
    }
    std::pair<Tensor, OptTensor> unsort_backward(const Tensor &dy, const Tensor &ys, const OptTensor &weights, const OptTensor &out) const {
        const int64_t d = width(dy, "dy");
        const Matrix g(dy, tokens, d, "dy", device), y(ys, rows_cap, d, "ys", device);
        const float *w = weights_of(weights);
        const On on(device);
        Tensor to = matrix_or_new(out, rows_cap, d, ys.scalar_type(), device);
        const Matrix o(to, rows_cap, d, "out", device);
        if (o.dtype != y.dtype) bad("out: must have the type of ys");
        OptTensor dw;
        if (weights) dw = floats({tokens, top_k}, device);
        const omoe_sort p = c();
        check(lib.unsort_rows_backward(&p, g.p, g.ld, g.dtype, y.p, y.ld, y.dtype, w, o.p, o.ld, dw ? static_cast<float *>(dw->data_ptr()) : nullptr,
                                       fits(d, "dy"), on.stream));
        if (out) written(to);
        return {to, dw};
    }
};

// ---- layer norm -----------------------------------------------------------------------------------------------------

py::object layer_norm(const Tensor &x, const OptTensor &gamma, const OptTensor &beta, double eps, const OptTensor &out,
                      const std::optional<at::ScalarType> &dtype, bool stats) {
    const int64_t d = width(x, "x"), T = x.size(0);
    const c10::Device dev = x.device();
    agree(out, dtype);
    const Matrix in(x, T, d, "x", dev);
    const auto *g = vec<float>(gamma, d, "gamma", dev), *b = vec<float>(beta, d, "beta", dev);
    const On on(dev);
    Tensor y = matrix_or_new(out, T, d, dtype.value_or(x.scalar_type()), dev), mean, rstd;
    const Matrix o(y, T, d, "out", dev);
    if (stats) std::tie(mean, rstd) = two_floats(T, dev);
    check(lib.layer_norm(in.p, in.ld, in.dtype, g, b, (float)eps, o.p, o.ld, o.dtype, stats ? static_cast<float *>(mean.data_ptr()) : nullptr,
                         stats ? static_cast<float *>(rstd.data_ptr()) : nullptr, fits(T, "x"), fits(d, "x"), on.stream));
    if (out) written(y);
    if (!stats) return py::cast(y);
    return py::make_tuple(y, mean, rstd);
}

std::tuple<Tensor, OptTensor, OptTensor> layer_norm_backward(const Tensor &dy, const Tensor &x, const OptTensor &gamma, const Tensor &mean,
                                                             const Tensor &rstd, const OptTensor &out, bool param_grads) {
    const int64_t d = width(x, "x"), T = x.size(0);
    const c10::Device dev = x.device();
    const Matrix in(x, T, d, "x", dev), g(dy, T, d, "dy", dev);
    const auto *gm = vec<float>(gamma, d, "gamma", dev), *m = vec<float>(mean, T, "mean", dev), *r = vec<float>(rstd, T, "rstd", dev);
    const On on(dev);
    Tensor dx = matrix_or_new(out, T, d, x.scalar_type(), dev);
    const Matrix o(dx, T, d, "out", dev);
    if (o.dtype != in.dtype) bad("out: must have the type of x");
    const int64_t bytes = lib.layer_norm_backward_workspace(fits(T, "x"), fits(d, "x"));
    if (bytes < 0) bad("x: no columns");
    const Tensor ws = fresh({bytes}, at::kByte, dev);
    OptTensor dgamma, dbeta;
    if (param_grads) std::tie(dgamma, dbeta) = two_floats(d, dev);
    check(lib.layer_norm_backward(g.p, g.ld, g.dtype, in.p, in.ld, in.dtype, gm, m, r, o.p, o.ld,
                                  dgamma ? static_cast<float *>(dgamma->data_ptr()) : nullptr, dbeta ? static_cast<float *>(dbeta->data_ptr()) : nullptr,
                                  (int32_t)T, (int32_t)d, ws.data_ptr(), bytes, on.stream));
    if (out) written(dx);
    return {dx, dgamma, dbeta};
}

// ---- gradient norm --------------------------------------------------------------------------------------------------

struct GradList {
    std::vector<Tensor> grads, out;  // kept alive
    std::vector<omoe_tensor> in, to;
    bool in_place;
    c10::Device device{c10::kCPU};

    GradList(std::vector<Tensor> grads_, std::optional<std::vector<Tensor>> out_) : grads(std::move(grads_)), in_place(!out_) {
        if (out_) out = std::move(*out_);
        bool same = in_place || out.size() == grads.size();
        for (size_t i = 0; same && i < out.size(); i++) same = out[i].scalar_type() == grads[i].scalar_type() && out[i].numel() == grads[i].numel();
        if (!same) bad("out: must have the sizes and types of the gradients");
        device = grads.empty() ? c10::Device(c10::kCUDA, c10::cuda::current_device()) : grads[0].device();
        auto list = [&](const std::vector<Tensor> &ts, std::vector<omoe_tensor> &refs) {
            for (const Tensor &t : ts) {
                if (t.device() != device || !t.is_contiguous()) bad("gradients must be contiguous and on one device");
                refs.push_back({t.data_ptr(), t.numel(), dtype_of(t.scalar_type()), 0});
            }
        };
        fits((int64_t)grads.size(), "gradients");
        list(grads, in);
        list(out, to);
    }
    const omoe_tensor *target() const { return in_place ? nullptr : to.data(); }
    // The tensors are still the ones that were checked: theirs is the memory at the addresses kept.
    void same(bool writes) const {
        auto moved = [](const std::vector<Tensor> &ts, const std::vector<omoe_tensor> &refs) {
            bool any = false;
            for (size_t i = 0; i < ts.size(); i++) any |= ts[i].const_data_ptr() != refs[i].ptr || ts[i].numel() != refs[i].count;
            return any;
        };
        if (moved(grads, in) || (writes && moved(out, to))) bad("a tensor of the list has another storage or size than when the list was built");
    }
    void scaled() const {
        for (const Tensor &t : in_place ? grads : out) written(t);
    }
    Tensor workspace() const { return fresh({OMOE_GRAD_WORKSPACE_BYTES}, at::kByte, device); }

    Tensor norm() const {
        same(false);
        const On on(device);
        const Tensor n = floats({}, device), ws = workspace();
        check(lib.grad_norm(in.data(), (int32_t)in.size(), static_cast<float *>(n.data_ptr()), ws.data_ptr(), OMOE_GRAD_WORKSPACE_BYTES, on.stream));
        return n;
    }
    void scale(const Tensor &n, double max_norm) const {
        same(true);
        const auto *p = vec<float>(n, 1, "norm", device);
        const On on(device);
        check(lib.grad_scale(in.data(), target(), (int32_t)in.size(), p, (float)max_norm, on.stream));
        scaled();
    }
    Tensor clip(double max_norm) const {
        same(true);
        const On on(device);
        const Tensor n = floats({}, device), ws = workspace();
        check(lib.grad_clip(in.data(), target(), (int32_t)in.size(), (float)max_norm, static_cast<float *>(n.data_ptr()), ws.data_ptr(),
                            OMOE_GRAD_WORKSPACE_BYTES, on.stream));
        scaled();
        return n;
    }
};

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.def("init", &init);
    py::class_<TokenSort>(m, "TokenSort")
        .def(py::init<int64_t, int64_t, int64_t, int64_t, const c10::Device &>())
        .def_readonly("tokens", &TokenSort::tokens)
        .def_readonly("top_k", &TokenSort::top_k)
        .def_readonly("n_experts", &TokenSort::n_experts)
        .def_readonly("row_align", &TokenSort::row_align)
        .def_readonly("rows_cap", &TokenSort::rows_cap)
        .def_readonly("pos", &TokenSort::pos)
        .def_readonly("perm", &TokenSort::perm)
        .def_readonly("counts", &TokenSort::counts)
        .def_readonly("offsets", &TokenSort::offsets)
        .def_readonly("device", &TokenSort::device)
        .def("plan", &TokenSort::plan)
        .def("sort", &TokenSort::sort)
        .def("sort_backward", &TokenSort::sort_backward)
        .def("unsort", &TokenSort::unsort)
        .def("unsort_backward", &TokenSort::unsort_backward);
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_backward", &layer_norm_backward);
    py::class_<GradList>(m, "GradList")
        .def(py::init<std::vector<Tensor>, std::optional<std::vector<Tensor>>>())
        .def_readonly("grads", &GradList::grads)
        .def("norm", &GradList::norm)
        .def("scale", &GradList::scale)
        .def("clip", &GradList::clip);
}
