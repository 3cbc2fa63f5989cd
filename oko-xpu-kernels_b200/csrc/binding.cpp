// The Python binding of the MXFP4 and experts' entries: torch tensors in, torch tensors out.
//
// These calls are short (a decoded token's linear is 9 us on the device), and by ctypes and Python's
// autograd the host took as long as that for each and five times as long for a training step.  Here an
// entry costs the allocation of its output and the launch, and the gradients are nodes of torch's own
// engine.  Everything is on torch's current stream of the tensors' device; nothing synchronises.
//
// The library itself is not linked: bind() takes the addresses of its C entries from the loaded library,
// so that the loader's search order holds.  The Python modules check what a user passes; here only what the
// C entries report is raised.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <functional>
#include <stdexcept>
#include <string>

#include "xpu_kernels/convrot.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------------------------------ the C entries

struct Entries {
#define ENTRY(name) decltype(&xpuint8_##name) name = nullptr;
#define ENTRIES(X)                                                                                              \
    X(last_error) X(mxfp4_quantize_stream) X(mxfp4_quantize_columns_stream) X(mxfp4_dequantize_stream)          \
    X(mxfp4_mm_stream) X(mxfp4_linear_workspace_bytes) X(mxfp4_linear_stream)                                   \
    X(mxfp4_train_saved_workspace_bytes) X(mxfp4_train_workspace_bytes) X(mxfp4_train_stream)                   \
    X(mxfp4_grad_workspace_bytes) X(mxfp4_grad_stream) X(mxfp4_expert_linear_workspace_bytes)                   \
    X(mxfp4_expert_linear_stream) X(mxfp4_expert_train_saved_workspace_bytes)                                   \
    X(mxfp4_expert_train_workspace_bytes) X(mxfp4_expert_train_stream) X(mxfp4_expert_grad_workspace_bytes)     \
    X(mxfp4_expert_grad_stream) X(expert_sort_workspace_bytes) X(expert_sort_stream) X(expert_gather_stream)    \
    X(expert_combine_stream) X(expert_combine_grad_stream)
    ENTRIES(ENTRY)
} lib;

void check(int rc, const char *what) {
    if (rc != 0) throw std::runtime_error(std::string(what) + ": " + lib.last_error());
}

int type_of(const Tensor &x) { return x.scalar_type() == at::kBFloat16 ? 0 : x.scalar_type() == at::kHalf ? 1 : 2; }
at::ScalarType scalar_type(int64_t type) { return type == 0 ? at::kBFloat16 : type == 1 ? at::kHalf : at::kFloat; }

// the tensors' device made current, and torch's stream on it
struct On {
    c10::cuda::CUDAGuard guard;
    cudaStream_t stream;
    explicit On(const Tensor &x) : guard(x.device()), stream(c10::cuda::getCurrentCUDAStream(x.device().index()).stream()) {}
};

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor scratch(int64_t bytes, const Tensor &like) { return empty({bytes}, at::kByte, like); }

// x [R, K] with unit column stride (a copy where it has none), and its row stride
Tensor rows(const Tensor &x, int64_t &ld) {
    const int64_t r = x.size(0), k = x.size(1);
    ld = k;
    if (x.is_contiguous()) return x;
    if ((k != 1 && x.stride(1) != 1) || (r > 1 && x.stride(0) < k)) return x.contiguous();
    if (r > 1) ld = x.stride(0);
    return x;
}
// A gradient of a gradient is refused, as by torch's once_differentiable: the products' gradients are
// taken straight through the roundings and are not differentiated again.
variable_list once(variable_list out, const variable_list &grads) {
    bool again = false;
    for (const Tensor &g : grads) again |= g.defined() && g.requires_grad();
    if (!again || !at::GradMode::is_enabled()) return out;
    for (Tensor &t : out)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    const size_t n = out.size();
    return torch::autograd::DelayedError("trying to differentiate twice a function that was marked with once_differentiable", n)(std::move(out));
}

const float *bias_of(const Tensor &b) { return b.defined() ? b.data_ptr<float>() : nullptr; }
uint8_t *bytes(const Tensor &t) { return t.defined() ? static_cast<uint8_t *>(t.data_ptr()) : nullptr; }

// a bias as the entries take it: fp32, contiguous, 16-byte aligned
Tensor prepared_bias(const Tensor &b, const Tensor &like) {
    if (!b.defined()) return b;
    Tensor t = b.detach();
    if (t.scalar_type() != at::kFloat || t.device() != like.device() || !t.is_contiguous()) t = t.to(like.device(), at::kFloat).contiguous();
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t;
}

// --------------------------------------------------------------------------------------- MXFP4

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// codes and scales in one buffer, the scales at the next multiple of 256 bytes
Tensor quantize(const Tensor &in, bool rotate, bool transpose) {
    int64_t ldx;
    Tensor x = in.dim() == 2 ? rows(in, ldx) : in.contiguous();
    const int64_t n = in.dim() == 3 ? x.size(0) : 1, r = x.size(-2), k = x.size(-1);
    if (in.dim() == 3) ldx = k;
    const int64_t R = transpose ? k : r, K = transpose ? r : k;
    const int64_t at = round_up(n * R * ((K + 31) / 32) * 16, 256);
    Tensor q = scratch(at + n * ((R + 127) / 128) * ((K + 127) / 128) * 512, x);
    if (n * r * k == 0) return q;
    On on(x);
    uint8_t *codes = bytes(q), *scales = codes + at;
    if (transpose) check(lib.mxfp4_quantize_columns_stream(on.stream, x.data_ptr(), type_of(x), ldx, codes, scales, r, k, n, nullptr, nullptr, 0, 0), "mxfp4_quantize_columns");
    else check(lib.mxfp4_quantize_stream(on.stream, x.data_ptr(), type_of(x), ldx, codes, scales, nullptr, n * r, k, r, rotate), "mxfp4_quantize");
    return q;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias_in, bool rotate, int64_t want) {
        const Tensor bias = bias_in.value_or(Tensor());
        const int64_t n = w.size(0), k = w.size(1);
        int64_t ldx, ldw;
        const Tensor x2 = rows(x.dim() == 2 ? x : x.reshape({-1, k}), ldx), w2 = rows(w, ldw);
        const int64_t m = x2.size(0);
        std::vector<int64_t> shape = x.sizes().vec();
        ctx->saved_data["x"] = shape;
        shape.back() = n;
        Tensor y = empty(shape, x.scalar_type(), x), saved;
        if (m && n) {
            On on(x);
            if (want) saved = scratch(lib.mxfp4_train_saved_workspace_bytes(m, n, k, want), x);
            const Tensor work = scratch(lib.mxfp4_train_workspace_bytes(m, n, k), x), b = prepared_bias(bias, x);
            check(lib.mxfp4_train_stream(on.stream, x2.data_ptr(), type_of(x), ldx, w2.data_ptr(), type_of(w), ldw, bias_of(b), y.data_ptr(), bytes(saved),
                                         bytes(work), m, n, k, rotate, want),
                  "mxfp4_train");
        }
        if (saved.defined()) ctx->save_for_backward({saved});
        ctx->saved_data["s"] = std::vector<int64_t>{m, n, k, rotate, want, type_of(x), type_of(w), bias.defined() ? static_cast<int64_t>(bias.scalar_type()) : -1};
        if (bias.defined() && bias.requires_grad()) {
            ctx->saved_data["b"] = bias.sizes().vec();
            ctx->saved_data["d"] = bias.device();
        }
        return y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        const std::vector<int64_t> s = ctx->saved_data["s"].toIntVector(), shape = ctx->saved_data["x"].toIntVector();
        const int64_t m = s[0], n = s[1], k = s[2], want = s[4];
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = s[7] >= 0 && ctx->needs_input_grad(2);
        int64_t ld;
        const Tensor dy = rows(grads[0].reshape({m, n}), ld);
        Tensor dx, dw, db;
        if (need_x) dx = empty(shape, scalar_type(s[5]), dy);
        if (need_w) dw = empty({n, k}, scalar_type(s[6]), dy);
        if (m && n && (need_x || need_w)) {
            On on(dy);
            const Tensor saved = ctx->get_saved_variables()[0];
            const Tensor work = scratch(lib.mxfp4_grad_workspace_bytes(m, n, k, s[6], s[3], (need_x ? 1 : 0) | (need_w ? 2 : 0)), dy);
            check(lib.mxfp4_grad_stream(on.stream, dy.data_ptr(), s[5], ld, bytes(saved), bytes(dx), bytes(dw), s[6], bytes(work), m, n, k, s[3], want), "mxfp4_grad");
        } else {
            if (need_x) dx.zero_();
            if (need_w) dw.zero_();
        }
        if (need_b) {  // as the bias is: any shape of n values, any type, any device
            db = dy.sum(at::IntArrayRef{0}, false, at::kFloat).reshape(ctx->saved_data["b"].toIntVector());
            db = db.to(ctx->saved_data["d"].toDevice(), static_cast<at::ScalarType>(s[7]));
        }
        return once({dx, dw, db, Tensor(), Tensor()}, grads);
    }
};

// ------------------------------------------------------------------------------------- experts

// The arrays of a plan in its buffer, and its sizes (xpu_kernels/experts.py: ExpertPlan).
struct Plan {
    Tensor buffer;
    int64_t tokens, top, experts;
    int64_t slots() const { return tokens * top; }
    int64_t max_tiles() const { return slots() / 128 + std::min(experts, slots()); }
    const int32_t *at(int64_t i) const { return buffer.data_ptr<int32_t>() + i; }
    const int32_t *order() const { return at(0); }
    const int32_t *positions() const { return at(slots()); }
    const int32_t *scale_rows() const { return at(2 * slots()); }
    const int32_t *offsets() const { return at(3 * slots()); }
    const int32_t *tiles() const { return at(3 * slots() + experts + 1); }
};

Tensor sorted_plan(const Tensor &ids, int64_t experts) {
    const int64_t n = ids.numel(), work = lib.expert_sort_workspace_bytes(n, experts);
    if (work < 0) throw std::runtime_error("expert_sort: too many slots");
    Tensor buffer = empty({3 * n + 2 * (experts + 1) + work / 4}, at::kInt, ids);
    if (!n) return buffer.zero_();
    On on(ids);
    int32_t *p = buffer.data_ptr<int32_t>(), *offsets = p + 3 * n, *tiles = offsets + experts + 1;
    check(lib.expert_sort_stream(on.stream, ids.data_ptr(), static_cast<int32_t>(ids.element_size()), n, experts, p, p + n, p + 2 * n, offsets, tiles, tiles + experts + 1),
          "expert_sort");
    return buffer;
}

Tensor gather(const Tensor &in, const Plan &p) {
    int64_t ld;
    const Tensor x = rows(in, ld);
    const int64_t w = x.size(1);
    Tensor out = empty({p.slots(), w}, x.scalar_type(), x);
    if (!w || !p.slots()) return out;
    On on(x);
    check(lib.expert_gather_stream(on.stream, x.data_ptr(), type_of(x), ld, out.data_ptr(), p.positions(), p.scale_rows(), p.tokens, p.top, w), "expert_gather");
    return out;
}

Tensor combine(const Tensor &in, const Tensor &weights, const Plan &p) {
    int64_t ld;
    const Tensor y = rows(in, ld);
    const int64_t w = y.size(1);
    Tensor out = empty({p.tokens, w}, y.scalar_type(), y);
    if (!w || !p.slots()) return out.zero_();
    On on(y);
    check(lib.expert_combine_stream(on.stream, y.data_ptr(), type_of(y), ld, weights.defined() ? weights.data_ptr<float>() : nullptr, out.data_ptr(), p.positions(),
                                    p.scale_rows(), p.tokens, p.top, w),
          "expert_combine");
    return out;
}

void save_plan(AutogradContext *ctx, const Plan &p) { ctx->saved_data["p"] = std::vector<int64_t>{p.tokens, p.top, p.experts}; }
Plan saved_plan(AutogradContext *ctx, const Tensor &buffer) {
    const std::vector<int64_t> s = ctx->saved_data["p"].toIntVector();
    return Plan{buffer, s[0], s[1], s[2]};
}

struct GatherFn : torch::autograd::Function<GatherFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &buffer, int64_t tokens, int64_t top, int64_t experts) {
        const Plan p{buffer, tokens, top, experts};
        save_plan(ctx, p);
        ctx->save_for_backward({buffer});
        return gather(x, p);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        return once({combine(grads[0], Tensor(), saved_plan(ctx, ctx->get_saved_variables()[0])), Tensor(), Tensor(), Tensor(), Tensor()}, grads);
    }
};

struct CombineFn : torch::autograd::Function<CombineFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &weights, const Tensor &buffer, int64_t tokens, int64_t top, int64_t experts) {
        const Plan p{buffer, tokens, top, experts};
        save_plan(ctx, p);
        ctx->save_for_backward({y, weights, buffer});
        return combine(y, weights, p);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list saved = ctx->get_saved_variables();
        const Plan p = saved_plan(ctx, saved[2]);
        int64_t ld_dy, ld_y;
        const Tensor dy = rows(grads[0], ld_dy), y = rows(saved[0], ld_y);
        const int64_t w = y.size(1);
        Tensor grad_y = empty({p.slots(), w}, y.scalar_type(), y), grad_w = empty({p.tokens, p.top}, at::kFloat, y);
        if (w && p.slots()) {
            On on(y);
            check(lib.expert_combine_grad_stream(on.stream, dy.data_ptr(), type_of(y), ld_dy, y.data_ptr(), ld_y, saved[1].data_ptr<float>(), grad_y.data_ptr(),
                                                 grad_w.data_ptr<float>(), p.positions(), p.scale_rows(), p.tokens, p.top, w),
                  "expert_combine_grad");
        } else {
            grad_w.zero_();
        }
        return once({grad_y, grad_w, Tensor(), Tensor(), Tensor(), Tensor()}, grads);
    }
};

struct ExpertLinearFn : torch::autograd::Function<ExpertLinearFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_in, const Tensor &buffer, int64_t tokens, int64_t top, bool rotate, bool sorted, int64_t want) {
        const Tensor w = w_in.contiguous();
        const int64_t e = w.size(0), n = w.size(1), k = w.size(2);
        const Plan p{buffer, tokens, top, e};
        int64_t ldx;
        const Tensor x2 = rows(x, ldx);
        Tensor y = empty({p.slots(), n}, x.scalar_type(), x), saved;
        if (n) {
            On on(x);
            if (want) saved = scratch(lib.mxfp4_expert_train_saved_workspace_bytes(p.max_tiles(), n, k, e, want), x);
            const Tensor work = scratch(lib.mxfp4_expert_train_workspace_bytes(p.slots(), p.max_tiles(), n, k, e), x);
            check(lib.mxfp4_expert_train_stream(on.stream, x2.data_ptr(), type_of(x), ldx, w.data_ptr(), type_of(w), y.data_ptr(), bytes(saved), bytes(work), p.order(),
                                                p.positions(), p.scale_rows(), p.offsets(), p.tiles(), tokens, top, p.max_tiles(), n, k, e, rotate, sorted, want),
                  "mxfp4_expert_train");
        }
        if (saved.defined()) ctx->save_for_backward({saved, buffer});
        save_plan(ctx, p);
        ctx->saved_data["s"] = std::vector<int64_t>{n, k, rotate, sorted, want, type_of(x), type_of(w)};
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        at::AutoDispatchBelowADInplaceOrView below;
        const std::vector<int64_t> s = ctx->saved_data["s"].toIntVector();
        const int64_t n = s[0], k = s[1], want = s[4];
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        int64_t ld;
        const Tensor dy = rows(grads[0], ld);
        const variable_list saved = n ? ctx->get_saved_variables() : variable_list{};
        const Plan p = saved_plan(ctx, n ? saved[1] : Tensor());
        Tensor dx, dw;
        if (need_x) dx = empty({s[3] ? p.slots() : p.tokens, k}, scalar_type(s[5]), dy);
        if (need_w) dw = empty({p.experts, n, k}, scalar_type(s[6]), dy);
        if (n && (need_x || need_w)) {
            On on(dy);
            const Tensor work = scratch(lib.mxfp4_expert_grad_workspace_bytes(p.slots(), p.max_tiles(), n, k, p.experts, s[6], s[2], s[3], (need_x ? 1 : 0) | (need_w ? 2 : 0)), dy);
            check(lib.mxfp4_expert_grad_stream(on.stream, dy.data_ptr(), s[5], ld, bytes(saved[0]), bytes(dx), bytes(dw), s[6], bytes(work), p.order(), p.positions(),
                                               p.scale_rows(), p.offsets(), p.tiles(), p.tokens, p.top, p.max_tiles(), n, k, p.experts, s[2], s[3], want),
                  "mxfp4_expert_grad");
        } else if (need_x) {
            dx.zero_();
        }
        return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, grads);
    }
};

// ------------------------------------------------------------------------ from and to Python objects

const Tensor &tensor(PyObject *o) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), "a tensor was expected");
    return THPVariable_Unpack(o);
}
Tensor tensor_or_none(PyObject *o) { return o == Py_None ? Tensor() : tensor(o); }
int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw py::error_already_set();
    return v;
}
bool flag(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw py::error_already_set();
    return v;
}
void *address(PyObject *o) {
    void *p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw py::error_already_set();
    return p;
}

// An MXFP4 matrix [r, k], or a stack of n: two objects from Python, its codes and its scales, or the buffer
// that holds both and where the scales begin.  Looked at on every call, never kept as addresses: who holds the
// tensors can give them other memory.
struct Matrix {
    const uint8_t *codes, *scales;
};
const uint8_t *held(const char *what, const Tensor &t, int64_t at, int64_t bytes, const Tensor &like) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kByte && t.is_contiguous() && t.device() == like.device() && t.numel() >= at + bytes &&
                          static_cast<int64_t>(t.storage().nbytes()) >= t.storage_offset() + at + bytes,
                      "the ", what, " of an MXFP4 matrix were changed: expected ", bytes, " contiguous bytes on ", like.device());
    return bytes ? static_cast<const uint8_t *>(t.data_ptr()) + at : nullptr;
}
Matrix matrix(PyObject *codes, PyObject *scales, int64_t n, int64_t r, int64_t k, const Tensor &like) {
    const int64_t code_bytes = n * r * ((k + 31) / 32) * 16, scale_bytes = n * ((r + 127) / 128) * ((k + 127) / 128) * 512;
    const Tensor &c = tensor(codes);
    if (PyLong_Check(scales)) return {held("codes", c, 0, code_bytes, like), held("scales", c, integer(scales), scale_bytes, like)};
    const Tensor &s = tensor(scales);
    TORCH_CHECK_VALUE(c.numel() == code_bytes && s.numel() == scale_bytes, "the codes or the scales of an MXFP4 matrix were changed: expected ", code_bytes, " and ",
                      scale_bytes, " bytes, got ", c.numel(), " and ", s.numel());
    return {held("codes", c, 0, code_bytes, like), held("scales", s, 0, scale_bytes, like)};
}

template <Tensor (*F)(PyObject *const *), Py_ssize_t N>
PyObject *wrapped(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_VALUE(n == N, "expected ", N, " arguments, got ", n);
    return THPVariable_Wrap(F(args));
    END_HANDLE_TH_ERRORS
}

Tensor py_quantize(PyObject *const *a) { return quantize(tensor(a[0]), flag(a[1]), flag(a[2])); }

// (codes, scales, type, shape)
Tensor py_dequantize(PyObject *const *a) {
    const Tensor &like = tensor(a[0]);
    const int64_t type = integer(a[2]);
    std::vector<int64_t> shape;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[3]); ++i) shape.push_back(integer(PyTuple_GET_ITEM(a[3], i)));
    const int64_t each = shape[shape.size() - 2], k = shape.back();
    Tensor out = empty(shape, scalar_type(type), like);
    const int64_t n = out.numel();
    if (n) {
        const Matrix q = matrix(a[0], a[1], n / k / each, each, k, like);
        On on(like);
        check(lib.mxfp4_dequantize_stream(on.stream, q.codes, q.scales, out.data_ptr(), type, n / k, k, each), "mxfp4_dequantize");
    }
    return out;
}

// (a codes, a scales, b codes, b scales, bias or None, type, m, n, k)
Tensor py_mm(PyObject *const *a) {
    const int64_t type = integer(a[5]), m = integer(a[6]), n = integer(a[7]), k = integer(a[8]);
    const Tensor &like = tensor(a[0]);
    Tensor out = empty({m, n}, scalar_type(type), like);
    if (m && n) {
        const Matrix p = matrix(a[0], a[1], 1, m, k, like), q = matrix(a[2], a[3], 1, n, k, like);
        On on(like);
        const Tensor bias = prepared_bias(tensor_or_none(a[4]), like);
        check(lib.mxfp4_mm_stream(on.stream, p.codes, p.scales, q.codes, q.scales, bias_of(bias), out.data_ptr(), type, n, m, n, k), "mxfp4_mm");
    }
    return out;
}

// In either mode; forward-mode tangents are refused by the nodes' apply, where they would be lost below it.
bool differentiates(const Tensor &x) {
    return x.defined() && ((x.requires_grad() && at::GradMode::is_enabled()) || torch::autograd::isFwGradDefined(x));
}

// A product over a weight held in 4 bits has no backward, but its result depends on what asks for a
// gradient.  So it joins the graph as a node that refuses: left out, a loss that reaches the same tensor by
// another way as well gets a wrong gradient without a word.
struct FrozenFn : torch::autograd::Function<FrozenFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &, const std::optional<Tensor> &, const std::function<Tensor()> &product, const std::string &refusal) {
        ctx->saved_data["refusal"] = refusal;
        return product();
    }
    static variable_list backward(AutogradContext *ctx, variable_list) { throw std::runtime_error(ctx->saved_data["refusal"].toStringRef()); }
};
Tensor frozen(const Tensor &x, const Tensor &bias, const std::function<Tensor()> &product, const char *refusal) {
    if (!differentiates(x) && !differentiates(bias)) return product();
    return FrozenFn::apply(x, bias.defined() ? std::optional<Tensor>(bias) : std::nullopt, product, std::string(refusal));
}

Tensor linear(const Tensor &x, const Matrix &w, int64_t n, const Tensor &bias_in, bool rotate) {
    const int64_t k = x.size(-1);
    at::AutoDispatchBelowADInplaceOrView below;
    int64_t ldx;
    const Tensor x2 = rows(x.dim() == 2 ? x : x.reshape({-1, k}), ldx);
    const int64_t m = x2.size(0);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = n;
    Tensor out = empty(shape, x.scalar_type(), x);
    if (m && n) {
        On on(x);
        // up to 8 rows of whole 16-byte words are quantised inside the product, without scratch
        Tensor work;
        if (m > 8 || reinterpret_cast<uintptr_t>(x2.data_ptr()) % 16 || ldx * x2.element_size() % 16) work = scratch(lib.mxfp4_linear_workspace_bytes(m, k), x);
        const Tensor bias = prepared_bias(bias_in, x);
        check(lib.mxfp4_linear_stream(on.stream, x2.data_ptr(), type_of(x), ldx, w.codes, w.scales, bias_of(bias), out.data_ptr(), bytes(work), m, n, k, rotate), "mxfp4_linear");
    }
    return out;
}

// (x, codes, scales, n, bias or None, rotate)
Tensor py_linear(PyObject *const *a) {
    const Tensor &x = tensor(a[0]);
    const Tensor bias = tensor_or_none(a[4]);
    const int64_t n = integer(a[3]);
    const Matrix w = matrix(a[1], a[2], 1, n, x.size(-1), x);
    const bool rotate = flag(a[5]);
    return frozen(x, bias, [&] { return linear(x, w, n, bias, rotate); },
                  "linear_mxfp4 has no backward, its weight is held in 4 bits: train with mxfp4_linear, or call it under torch.no_grad()");
}

// (x, w, bias or None, rotate)
Tensor py_train(PyObject *const *a) {
    const Tensor &x = tensor(a[0]), &w = tensor(a[1]);
    const int64_t want = at::GradMode::is_enabled() ? (x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0) : 0;
    const Tensor bias = tensor_or_none(a[2]);
    return LinearFn::apply(x, w, bias.defined() ? std::optional<Tensor>(bias) : std::nullopt, flag(a[3]), want);
}

Tensor py_sort(PyObject *const *a) { return sorted_plan(tensor(a[0]), integer(a[1])); }

// (x, buffer, tokens, top, experts)
Tensor py_gather(PyObject *const *a) {
    const Tensor &x = tensor(a[0]);
    const Plan p{tensor(a[1]), integer(a[2]), integer(a[3]), integer(a[4])};
    return differentiates(x) ? GatherFn::apply(x, p.buffer, p.tokens, p.top, p.experts) : gather(x, p);
}

// (y, weights, buffer, tokens, top, experts)
Tensor py_combine(PyObject *const *a) {
    const Tensor &y = tensor(a[0]), &w = tensor(a[1]);
    const Plan p{tensor(a[2]), integer(a[3]), integer(a[4]), integer(a[5])};
    return differentiates(y) || differentiates(w) ? CombineFn::apply(y, w, p.buffer, p.tokens, p.top, p.experts) : combine(y, w, p);
}

Tensor expert_linear(const Tensor &in, const Matrix &w, int64_t n, const Plan &p, bool rotate, bool sorted) {
    at::AutoDispatchBelowADInplaceOrView below;
    int64_t ldx;
    const Tensor x = rows(in, ldx);
    const int64_t k = x.size(1);
    Tensor out = empty({p.slots(), n}, x.scalar_type(), x);
    if (p.slots() && n) {
        On on(x);
        // up to 128 rows of whole 16-byte words are quantised inside the product, without scratch
        Tensor work;
        if (p.slots() > 128 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || ldx * x.element_size() % 16)
            work = scratch(lib.mxfp4_expert_linear_workspace_bytes(p.slots(), p.max_tiles(), k), x);
        check(lib.mxfp4_expert_linear_stream(on.stream, x.data_ptr(), type_of(x), ldx, w.codes, w.scales, out.data_ptr(), bytes(work), p.order(), p.positions(), p.scale_rows(),
                                             p.offsets(), p.tiles(), p.tokens, p.top, p.max_tiles(), n, k, p.experts, rotate, sorted),
              "mxfp4_expert_linear");
    }
    return out;
}

// (x, codes, scales, n, buffer, tokens, top, experts, rotate, sorted)
Tensor py_expert_linear(PyObject *const *a) {
    const Tensor &x = tensor(a[0]);
    const int64_t n = integer(a[3]);
    const Plan p{tensor(a[4]), integer(a[5]), integer(a[6]), integer(a[7])};
    const Matrix w = matrix(a[1], a[2], p.experts, n, x.size(1), x);
    const bool rotate = flag(a[8]), sorted = flag(a[9]);
    return frozen(x, Tensor(), [&] { return expert_linear(x, w, n, p, rotate, sorted); },
                  "expert_linear_mxfp4 has no backward, its weights are held in 4 bits: train with mxfp4_expert_linear, or call it under torch.no_grad()");
}

// (x, w, buffer, tokens, top, rotate, sorted)
Tensor py_expert_train(PyObject *const *a) {
    const Tensor &x = tensor(a[0]), &w = tensor(a[1]);
    const int64_t want = at::GradMode::is_enabled() ? (x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0) : 0;
    return ExpertLinearFn::apply(x, w, tensor(a[2]), integer(a[3]), integer(a[4]), flag(a[5]), flag(a[6]), want);
}

// {name: address} of the library's entries, without the xpuint8_ prefix
PyObject *py_bind(PyObject *, PyObject *dict) {
    HANDLE_TH_ERRORS
#define BIND(name)                                                                             \
    {                                                                                          \
        PyObject *v = PyDict_GetItemString(dict, #name);                                       \
        if (!v) throw std::runtime_error("the library has no entry " #name);                   \
        lib.name = reinterpret_cast<decltype(lib.name)>(address(v)); \
    }
    ENTRIES(BIND)
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject *py_names(PyObject *, PyObject *) {
    HANDLE_TH_ERRORS
    py::list names;
#define NAME(name) names.append(#name);
    ENTRIES(NAME)
    return names.release().ptr();
    END_HANDLE_TH_ERRORS
}

#define FAST(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&wrapped<py_##name, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(quantize, 3), FAST(dequantize, 4), FAST(mm, 9), FAST(linear, 6), FAST(train, 4), FAST(sort, 2), FAST(gather, 5), FAST(combine, 6),
                         FAST(expert_linear, 10), FAST(expert_train, 7), {"bind", py_bind, METH_O, nullptr}, {"names", py_names, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
