// binding.cpp -- PyTorch binding of the training-step ops of libgenre_hip.so (include/genre_hip.h, at its end).
//
// The geometric ops are called a few times a step on a few tensors; ctypes (_loader.py) serves them.  These are called once per
// norm layer, on maps whose kernels may take 5 us, or on lists of hundreds of tensors: reading a tensor's address, size, type and
// layout costs 0.05 us here and 0.5 us from Python (434 tensors: the norm and clip took 256 us, 75 us of it on the GPU), and an
// autograd node in C++ saves some 30 us of forward and backward.  The checks of arguments are here with them.
#include <dlfcn.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "genre_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::variable_list;

// ---- the library (the one that _loader.py loaded) ---------------------------------------------------------------
struct Lib {
    decltype(&genre_last_error) last_error;
    decltype(&genre_group_norm_workspace) gn_workspace;
    decltype(&genre_group_norm_forward) gn_forward;
    decltype(&genre_group_norm_backward) gn_backward;
    decltype(&genre_grad_workspace) grad_workspace;
    decltype(&genre_grad_norm) grad_norm;
    decltype(&genre_grad_scale) grad_scale;
    decltype(&genre_adam_step) adam_step;
} lib;

template <class F>
void find(void *handle, const char *name, F &f)
{
    f = (F)dlsym(handle, name);
    TORCH_CHECK(f, "libgenre_hip.so does not export ", name, " -- rebuild (make -C genre-shapehd_amd/csrc)");
}

void bind_library(const std::string &path)
{
    void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(h, "cannot load ", path, ": ", dlerror());
    find(h, "genre_last_error", lib.last_error);
    find(h, "genre_group_norm_workspace", lib.gn_workspace);
    find(h, "genre_group_norm_forward", lib.gn_forward);
    find(h, "genre_group_norm_backward", lib.gn_backward);
    find(h, "genre_grad_workspace", lib.grad_workspace);
    find(h, "genre_grad_norm", lib.grad_norm);
    find(h, "genre_grad_scale", lib.grad_scale);
    find(h, "genre_adam_step", lib.adam_step);
}

#define GENRE_CALL(what, call) TORCH_CHECK((call) == 1, what, " failed: ", lib.last_error())

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int type_of(const Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return GENRE_F32;
    case at::kBFloat16: return GENRE_BF16;
    case at::kHalf: return GENRE_F16;
    default: return -1;
    }
}

// uninitialised memory from torch's allocator, without the dispatcher's share of the call (a half of it)
Tensor fresh(at::IntArrayRef size, at::ScalarType type, at::Device device) { return Tensor(at::detail::empty_cuda(size, type, device, std::nullopt)); }

// its values as they lie in memory (a view may hold the negatives of them)
Tensor plain(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

genre_tensor flat(const Tensor &t, int type)
{
    genre_tensor d{};
    d.data = t.data_ptr();
    d.ndim = 1;
    d.dtype = type;
    d.size[0] = t.numel();
    d.stride[0] = 1;
    return d;
}

// ---- group normalisation ----------------------------------------------------------------------------------------
// How the kernels walk a map [N, C, space...]: element strides of image, channel and position, and whether it is channels last
// (a row of channels per position; gaps between rows are fine) or first (a plane of positions per channel).
struct Walk { bool ok, last; int64_t image, channel, position; };

Walk walk_of(const Tensor &t)
{
    const auto size = t.sizes(), stride = t.strides();
    const int64_t c = size[1], s = t.numel() / (size[0] * c);
    int64_t step = 0, expect = 0;                                          // distance of two positions, if they all lie at one
    for (int64_t i = t.dim() - 1; i >= 2; i--) {
        if (size[i] == 1) continue;
        if (!step) step = stride[i];
        else if (stride[i] != expect) return {};
        if (!step) return {};                                              // expanded
        expect = stride[i] * size[i];
    }
    const int64_t image = size[0] == 1 ? c * s : stride[0], channel = stride[1];
    if (s == 1) return {c == 1 || channel == 1, true, image, 1, c};
    if (step == 1 && (c == 1 || channel >= s)) return {true, false, image, c == 1 ? s : channel, 1};
    return {c > 1 && channel == 1 && step >= c, true, image, 1, step};
}

// an uninitialised gap-free map in x's layout
Tensor like(const Tensor &x, const Walk &w, Walk &out)
{
    const int64_t c = x.size(1), s = x.numel() / (x.size(0) * c);
    if (w.image == c * s && (w.last ? w.position == c : w.channel == s)) {
        out = w;
        return Tensor(at::detail::empty_strided_cuda(x.sizes(), x.strides(), x.scalar_type(), x.device()));
    }
    std::vector<int64_t> stride(x.dim());
    int64_t at = w.last ? c : 1;
    for (int64_t i = x.dim() - 1; i >= 2; i--) {
        stride[i] = at;
        at *= x.size(i);
    }
    stride[0] = c * s;
    stride[1] = w.last ? 1 : s;
    out = {true, w.last, c * s, stride[1], w.last ? c : 1};
    return Tensor(at::detail::empty_strided_cuda(x.sizes(), stride, x.scalar_type(), x.device()));
}

genre_tensor map(const Tensor &t, const Walk &w)
{
    genre_tensor d{};
    d.data = t.data_ptr();
    d.ndim = 3;
    d.dtype = type_of(t);
    d.size[0] = t.size(0);
    d.size[1] = t.size(1);
    d.size[2] = t.numel() / (d.size[0] * d.size[1]);
    d.stride[0] = w.image;
    d.stride[1] = w.channel;
    d.stride[2] = w.position;
    return d;
}

// a [C] parameter (or none) as an argument
struct Param {
    Tensor keep;
    genre_tensor d;
    const genre_tensor *arg = nullptr;
    explicit Param(const Tensor &t)
    {
        if (!t.defined()) return;
        keep = t.contiguous();
        d = flat(keep, type_of(keep));
        arg = &d;
    }
};

struct Forward { Tensor x, y, stats; };

// the call's scratch memory, if it needs any
struct Scratch {
    Tensor keep;
    genre_tensor d;
    const genre_tensor *arg = nullptr;
    Scratch(const genre_tensor &x, int64_t groups, int backward, const Tensor &like)
    {
        const int64_t need = lib.gn_workspace(&x, (int)groups, backward);
        TORCH_CHECK(need >= 0, lib.last_error());
        if (!need) return;
        keep = fresh({need}, at::kDouble, like.device());
        d = flat(keep, GENRE_F64);
        arg = &d;
    }
};

Forward gn_forward(const Tensor &given, const Tensor &weight, const Tensor &bias, int64_t groups, double eps, int64_t act, double slope)
{
    const c10::DeviceGuard guard(given.device());
    Forward f{given, {}, fresh({2, given.size(0), groups}, at::kDouble, given.device())};
    if (!given.numel()) {
        f.y = at::empty_like(given);
        return f;
    }
    Walk in = walk_of(f.x), out;
    if (!in.ok) {
        f.x = given.contiguous();
        in = walk_of(f.x);
        TORCH_CHECK(in.ok, "group_norm_act: cannot walk a map of strides ", f.x.strides());
    }
    f.y = like(f.x, in, out);
    const genre_tensor x = map(f.x, in), y = map(f.y, out), stats = flat(f.stats, GENRE_F64);
    const Scratch ws(x, groups, 0, given);
    const Param p(weight), b(bias);
    GENRE_CALL("group_norm_act", lib.gn_forward(&x, &y, p.arg, b.arg, &stats, ws.arg, (int)groups, eps, (int)act, (float)slope, stream_of(given)));
    return f;
}

class GroupNormAct : public torch::autograd::Function<GroupNormAct> {
public:
    static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const OptTensor &w, const OptTensor &b, int64_t groups, double eps,
                          int64_t act, double slope)
    {
        const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
        Forward f = gn_forward(x, weight, bias, groups, eps, act, slope);
        ctx->save_for_backward({f.x, weight, bias, f.stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["slope"] = slope;
        return f.y;
    }

    static variable_list backward(torch::autograd::AutogradContext *ctx, variable_list grads)
    {
        const bool again = at::GradMode::is_enabled();                     // create_graph: a second differentiation is refused
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        Tensor dy = grads[0], dx, dw, db;
        const c10::DeviceGuard guard(x.device());
        // (the edges are those of the tensors that were given)
        if (weight.defined() && ctx->needs_input_grad(1)) dw = fresh({x.size(1)}, weight.scalar_type(), x.device());
        if (bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1)) db = fresh({x.size(1)}, bias.scalar_type(), x.device());
        dy = dy.defined() ? plain(dy) : at::zeros_like(x);
        if (!x.numel()) {
            if (ctx->needs_input_grad(0)) dx = at::empty_like(x);
            if (dw.defined()) dw.zero_();
            if (db.defined()) db.zero_();
        } else {
            const Walk in = walk_of(x);
            Walk grad = walk_of(dy), out{};
            if (!grad.ok || grad.last != in.last) {                        // in another layout than x: into x's
                Tensor t = like(x, in, grad);
                t.copy_(dy);
                dy = t;
            }
            if (ctx->needs_input_grad(0)) dx = like(x, in, out);
            const genre_tensor mx = map(x, in), md = map(dy, grad), st = flat(stats, GENRE_F64), mo = dx.defined() ? map(dx, out) : genre_tensor{};
            const Scratch ws(mx, groups, 1, x);
            const Param p(weight), b(bias), gw(dw), gb(db);
            GENRE_CALL("group_norm_act backward",
                       lib.gn_backward(&mx, &md, p.arg, b.arg, &st, dx.defined() ? &mo : nullptr, gw.arg, gb.arg, ws.arg, (int)groups,
                                       (int)ctx->saved_data["act"].toInt(), (float)ctx->saved_data["slope"].toDouble(), stream_of(x)));
        }
        variable_list out = {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
        if (again) {
            variable_list some;
            for (const Tensor &t : {dx, dw, db})
                if (t.defined()) some.push_back(t.detach().requires_grad_(true));
            const auto refuse = std::make_shared<torch::autograd::DelayedError>("group_norm_act can be differentiated only once", (int64_t)some.size());
            some = (*refuse)(std::move(some));
            size_t k = 0;
            for (int i = 0; i < 3; i++)
                if (out[i].defined()) out[i] = some[k++];
        }
        return out;
    }
};

void check_param(const char *what, const Tensor &t, const Tensor &x)
{
    if (!t.defined()) return;
    TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(1) && type_of(t) >= 0 && t.device() == x.device() && t.layout() == at::kStrided, "group_norm_act: ", what,
                " must be a [", x.size(1), "] tensor of fp32, bf16 or fp16 on ", x.device(), ", got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
}

Tensor group_norm_act(const Tensor &given, int64_t groups, const OptTensor &weight, const OptTensor &bias, double eps, int64_t act, double slope)
{
    const Tensor x = plain(given), w = weight ? plain(*weight) : Tensor(), b = bias ? plain(*bias) : Tensor();
    TORCH_CHECK(x.is_cuda(), "group_norm_act: x is on ", x.device(), "; GPU tensors only -- there is no CPU path");
    TORCH_CHECK(type_of(x) >= 0 && x.layout() == at::kStrided, "group_norm_act: ", x.scalar_type(), " ", x.layout(), " not supported (dense fp32, bf16 or fp16)");
    TORCH_CHECK(x.dim() >= 2, "group_norm_act: x must be [N, C, ...], got ", x.sizes());
    TORCH_CHECK(groups >= 1 && groups <= x.size(1) && x.size(1) % groups == 0, "group_norm_act: ", x.size(1), " channels do not split into ", groups, " groups");
    TORCH_CHECK(eps > 0, "group_norm_act: eps must be positive, got ", eps);
    check_param("weight", w, x);
    check_param("bias", b, x);
    for (const Tensor &t : {x, w, b}) TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "group_norm_act: forward-mode derivatives are not supported");
    if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()))) {
        pybind11::gil_scoped_release no_gil;
        return GroupNormAct::apply(x, w.defined() ? OptTensor(w) : std::nullopt, b.defined() ? OptTensor(b) : std::nullopt, groups, eps, act, slope);
    }
    pybind11::gil_scoped_release no_gil;
    const at::AutoDispatchBelowADInplaceOrView below;
    return gn_forward(x, w, b, groups, eps, act, slope).y;
}

// ---- many tensors at once ---------------------------------------------------------------------------------------
// the host arrays that the library reads: an address of each tensor of each list, sizes and types
struct Lists {
    std::vector<std::vector<void *>> at;
    std::vector<int64_t> numel;
    std::vector<int32_t> type;
    std::vector<Tensor> copies;
    c10::Device device{c10::kCPU};
    int n() const { return (int)numel.size(); }
};

const Tensor &item(const char *op, PyObject *list, Py_ssize_t i)
{
    PyObject *o = PySequence_Fast_GET_ITEM(list, i);
    TORCH_CHECK(THPVariable_Check(o), op, ": item ", i, " is no tensor");
    return THPVariable_Unpack(o);
}

bool gap_free(const Tensor &t) { return !t.is_neg() && (t.is_contiguous() || t.is_non_overlapping_and_dense()); }

// the first list: any gap-free tensors of one GPU and of the three types; others are refused where they are `written`, else copied
Lists first_list(const char *op, pybind11::handle list, bool written)
{
    Lists l;
    PyObject *p = list.ptr();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(p);
    l.at.emplace_back(n);
    l.numel.resize(n);
    l.type.resize(n);
    for (Py_ssize_t i = 0; i < n; i++) {
        const Tensor &t = item(op, p, i);
        if (i == 0) l.device = t.device();
        TORCH_CHECK(t.is_cuda() && t.device() == l.device, op, ": tensor ", i, " is on ", t.device(), "; all must be on one GPU -- there is no CPU path");
        l.type[i] = type_of(t);
        TORCH_CHECK(l.type[i] >= 0 && t.layout() == at::kStrided, op, ": tensor ", i, " is ", t.scalar_type(), " ", t.layout(), "; dense fp32, bf16 or fp16 tensors only");
        l.numel[i] = t.numel();
        if (gap_free(t)) {
            l.at[0][i] = t.data_ptr();
            continue;
        }
        TORCH_CHECK(!written, op, ": tensor ", i, " ", t.sizes(), " with strides ", t.strides(), " has gaps or overlaps, or is a view of negatives, and cannot be written in place");
        l.copies.push_back(plain(t.detach()).contiguous());
        l.at[0][i] = l.copies.back().data_ptr();
    }
    return l;
}

// whether t's values lie in memory as those of the gap-free p do (a dimension of one value may have any stride)
bool lies_as(const Tensor &t, const Tensor &p)
{
    if (t.sizes() != p.sizes() || t.is_neg()) return false;
    if (t.is_contiguous() && p.is_contiguous()) return true;
    for (int64_t i = 0; i < t.dim(); i++)
        if (t.size(i) != 1 && t.stride(i) != p.stride(i)) return false;
    return true;
}

// the places at which `others` does not lie as `weights` (of the same length)
std::vector<int64_t> laid_otherwise(pybind11::handle weights, pybind11::handle others)
{
    std::vector<int64_t> at;
    for (Py_ssize_t i = 0, n = PySequence_Fast_GET_SIZE(weights.ptr()); i < n; i++)
        if (!lies_as(item("laid_otherwise", others.ptr(), i), item("laid_otherwise", weights.ptr(), i))) at.push_back(i);
    return at;
}

void bump(pybind11::handle list)
{
    PyObject *p = list.ptr();
    for (Py_ssize_t i = 0, n = PySequence_Fast_GET_SIZE(p); i < n; i++) {
        const Tensor &t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(p, i));
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
}

// Refuses a tensor that is written (all lists but the second: of an Adam step the gradients) and shares memory with another: two
// workgroups would read and write it at once.  (1736 tensors: 25 to 60 us, while the norm runs.)
void check_apart(const char *op, const Lists &l)
{
    struct Span { uintptr_t begin, end; int index; bool written; };
    std::vector<Span> spans;
    spans.reserve(l.at.size() * l.n());
    for (size_t k = 0; k < l.at.size(); k++)
        for (int i = 0; i < l.n(); i++) {
            const uintptr_t p = (uintptr_t)l.at[k][i];
            if (l.numel[i]) spans.push_back({p, p + l.numel[i] * (k >= 2 || l.type[i] == GENRE_F32 ? 4 : 2), i, k != 1});
        }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;                                        // the ends of those that begin before
    for (const Span &s : spans) {
        TORCH_CHECK(s.begin >= (s.written ? any : written), op, ": tensor ", s.index, " shares memory with another one (or is listed twice)");
        any = std::max(any, s.end);
        if (s.written) written = std::max(written, s.end);
    }
}

Tensor norm_and_factor(const char *op, const Lists &l, int64_t kind, double max_norm)
{
    Tensor out = fresh({2}, at::kFloat, l.device);
    const int64_t need = lib.grad_workspace(l.numel.data(), l.n());
    TORCH_CHECK(need >= 0, lib.last_error());
    const Tensor ws = fresh({need}, at::kDouble, l.device);
    const genre_tensor o = flat(out, GENRE_F32), w = flat(ws, GENRE_F64);
    GENRE_CALL(op, lib.grad_norm(l.at[0].data(), l.numel.data(), l.type.data(), l.n(), (int)kind, (float)max_norm, &o, &w, stream_of(out)));
    return out;
}

Tensor grad_norm(pybind11::handle tensors, double max_norm, int64_t kind)
{
    const Lists l = first_list("grad_norm", tensors, false);
    const c10::DeviceGuard guard(l.device);
    return norm_and_factor("grad_norm", l, kind, max_norm);
}

Tensor clip_grads(pybind11::handle tensors, double max_norm, int64_t kind, bool error_if_nonfinite)
{
    const Lists l = first_list("clip_grads_", tensors, true);
    const c10::DeviceGuard guard(l.device);
    const Tensor out = norm_and_factor("clip_grads_", l, kind, max_norm), norm = out.select(0, 0);
    if (error_if_nonfinite) {
        const double v = [&] {
            pybind11::gil_scoped_release no_gil;                           // (this waits for the GPU: other threads go on)
            return norm.item<float>();
        }();
        TORCH_CHECK(std::isfinite(v), "clip_grads_: the norm of the gradients is ", v);
    }
    check_apart("clip_grads_", l);
    genre_tensor f = flat(out, GENRE_F32);
    f.data = (float *)f.data + 1;
    f.size[0] = 1;
    GENRE_CALL("clip_grads_", lib.grad_scale(l.at[0].data(), l.numel.data(), l.type.data(), l.n(), &f, stream_of(out)));
    bump(tensors);
    return norm;
}

OptTensor adam_step(pybind11::handle params, pybind11::handle grads, pybind11::handle exp_avgs, pybind11::handle exp_avg_sqs, int64_t step, double lr, double beta1,
                    double beta2, double eps, double weight_decay, bool decoupled, std::optional<double> max_norm, int64_t kind, const OptTensor &factor)
{
    const char *op = "clip_adam_step_";
    Lists l = first_list(op, params, true);
    const pybind11::handle more[3] = {grads, exp_avgs, exp_avg_sqs};
    const char *const names[3] = {"gradient", "exp_avg", "exp_avg_sq"};
    for (int k = 0; k < 3; k++) {
        std::vector<void *> at(l.n());
        for (int i = 0; i < l.n(); i++) {
            const Tensor &p = THPVariable_Unpack(PySequence_Fast_GET_ITEM(params.ptr(), i)), &t = item(op, more[k].ptr(), i);
            TORCH_CHECK(t.device() == l.device && t.layout() == at::kStrided && t.scalar_type() == (k ? at::kFloat : p.scalar_type()), op, ": ", names[k], " ", i, " is ",
                        t.scalar_type(), " ", t.layout(), " on ", t.device(), " for ", p.scalar_type(), " on ", l.device, " (", k ? "fp32 is wanted" : "the same is wanted", ")");
            TORCH_CHECK(lies_as(t, p), op, ": ", names[k], " ", i, " ", t.sizes(), " with strides ", t.strides(), " does not lie as its weight ", p.sizes(),
                        " with strides ", p.strides());
            at[i] = t.data_ptr();
        }
        l.at.push_back(std::move(at));
    }
    const c10::DeviceGuard guard(l.device);
    Tensor out;
    genre_tensor f{};
    void *st = (void *)c10::hip::getCurrentHIPStream(l.device.index()).stream();
    if (max_norm) {
        std::swap(l.at[0], l.at[1]);
        out = norm_and_factor(op, l, kind, *max_norm);
        std::swap(l.at[0], l.at[1]);
        f = flat(out, GENRE_F32);
        f.data = (float *)f.data + 1;
        f.size[0] = 1;
    } else if (factor) {
        TORCH_CHECK(factor->device() == l.device && factor->scalar_type() == at::kFloat && factor->numel() == 1 && factor->layout() == at::kStrided, op,
                    ": factor must be one fp32 value on ", l.device);
        f = flat(*factor, GENRE_F32);
    }
    check_apart(op, l);
    GENRE_CALL(op, lib.adam_step(l.at[0].data(), l.at[1].data(), l.at[2].data(), l.at[3].data(), l.numel.data(), l.type.data(), l.n(), f.data ? &f : nullptr,
                                 step, lr, beta1, beta2, eps, weight_decay, decoupled, st));
    bump(params);
    bump(exp_avgs);
    bump(exp_avg_sqs);
    return max_norm ? OptTensor(out.select(0, 0)) : std::nullopt;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("bind_library", &bind_library);
    m.def("group_norm_act", &group_norm_act);
    m.def("grad_norm", &grad_norm);
    m.def("clip_grads", &clip_grads);
    m.def("adam_step", &adam_step);
    m.def("laid_otherwise", &laid_otherwise);
}
