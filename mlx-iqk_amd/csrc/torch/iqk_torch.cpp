// The eager calls of the 4-bit modules and of the router on torch tensors: what
// an operator needs between its argument checks (in Python) and its launches --
// outputs, workspaces, the stream, and for the router the autograd nodes.  The
// kernels are libiqk_hip.so's, reached through its C ABI; nothing is computed here.
//
// In Python the allocations cost 1.7 us each and an autograd function 37 us a
// training step, more than the kernels of a small call.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include "iqk_hip.h"

#ifndef IQK_SOURCE_HASH
#define IQK_SOURCE_HASH "unset"
#endif
#ifndef IQK_BINDING_HASH
#define IQK_BINDING_HASH "unset"
#endif

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

Tensor empty(c10::IntArrayRef shape, at::ScalarType type, const Tensor &like) {
    return at::empty(shape, like.options().dtype(type).requires_grad(false));
}

int type_code(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return IQK_F32;
        case at::kHalf: return IQK_F16;
        default: return IQK_BF16;
    }
}

void check(int rc, const char *what) {
    TORCH_CHECK(rc == IQK_OK, what, ": code ", rc,
                rc == IQK_ERR_LAUNCH ? ", hipError " + std::to_string(iqk_hip_last_error()) : std::string());
}

template <typename T>
T *ptr(const Tensor &t) {
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

// A backward pass under a graph's capture has ended the process when the capture ended, for
// a reason that is not known; only the forward calls are for a graph.
void refuse_capture() {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    C10_HIP_CHECK(hipStreamIsCapturing(c10::hip::getCurrentHIPStream().stream(), &status));
    TORCH_CHECK(status == hipStreamCaptureStatusNone,
                "the router's gradients cannot be captured in a graph; run the backward pass eagerly");
}

// A gradient that is not differentiable again says so when asked.  It depends on what
// comes from above and on `saved`, the forward's tensor that the formula is of: the
// node that raises stands between it and them, so that a derivative in either meets it.
variable_list once(Tensor grad, const variable_list &above, const Tensor &saved) {
    if (!at::GradMode::is_enabled() || !(saved.requires_grad() || torch::autograd::any_variable_requires_grad(above)))
        return {grad};
    variable_list inputs{grad, saved};
    inputs.insert(inputs.end(), above.begin(), above.end());
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the router's gradients are not differentiable a second time", int64_t(inputs.size()));
    return {(*error)(std::move(inputs))[0]};
}

// ------------------------------------------------------------------- top k ---

std::pair<Tensor, Tensor> topk_forward(const Tensor &logits, int64_t k, bool normalize) {
    auto shape = logits.sizes().vec();
    const int64_t experts = shape.back(), rows = logits.numel() / experts;
    shape.back() = k;
    Tensor weights = empty(shape, at::kFloat, logits), ids = empty(shape, at::kInt, logits);
    check(iqk_router_topk(type_code(logits), logits.data_ptr(), rows, experts, k, normalize, ptr<float>(weights),
                          ptr<int32_t>(ids), stream_of(logits)),
          "iqk_router_topk");
    return {weights, ids};
}

struct TopK : torch::autograd::Function<TopK> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, int64_t k, bool normalize) {
        auto [weights, ids] = topk_forward(logits, k, normalize);
        ctx->mark_non_differentiable({ids});
        ctx->set_materialize_grads(false);
        ctx->saved_data["normalize"] = normalize;
        ctx->saved_data["type"] = int64_t(logits.scalar_type());
        ctx->saved_data["experts"] = logits.size(-1);
        ctx->save_for_backward({weights, ids, normalize ? Tensor() : logits});
        return {weights, ids};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_capture();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &weights = saved[0], &ids = saved[1], &logits = saved[2];
        const bool normalize = ctx->saved_data["normalize"].toBool();
        const int64_t experts = ctx->saved_data["experts"].toInt(), k = weights.size(-1);
        const Tensor dweights = grads[0].detach().to(at::kFloat).contiguous();
        auto shape = weights.sizes().vec();
        shape.back() = experts;
        Tensor dlogits = empty(shape, at::ScalarType(ctx->saved_data["type"].toInt()), weights);
        check(iqk_router_topk_grad(type_code(dlogits), ptr<void>(logits), ptr<float>(weights), ptr<int32_t>(ids),
                                   ptr<float>(dweights), weights.numel() / k, experts, k, normalize,
                                   dlogits.data_ptr(), stream_of(weights)),
              "iqk_router_topk_grad");
        auto out = once(dlogits, grads, normalize ? weights : logits);
        out.resize(3);
        return out;
    }
};

// ------------------------------------------------------------ balance loss ---

struct BalanceSums {
    Tensor loss, counts, kept;
};

BalanceSums balance_forward(const Tensor &logits, const Tensor &ids, const Tensor &mask) {
    auto lead = logits.sizes().vec();
    const int64_t experts = lead.back(), tokens = lead[lead.size() - 2], k = ids.size(-1);
    lead.resize(lead.size() - 2);
    int64_t groups = 1;
    for (const int64_t n : lead) groups *= n;
    BalanceSums s;
    s.loss = empty(lead, at::kFloat, logits);
    auto shape = lead;
    shape.push_back(experts);
    s.counts = empty(shape, at::kInt, logits);
    s.kept = empty(lead, at::kInt, logits);
    if (groups) {
        const int64_t words = iqk_balance_work(groups, tokens, experts);
        check(words < 0 ? IQK_ERR_GEOMETRY : IQK_OK, "iqk_balance_work");
        const Tensor work = empty({words}, at::kInt, logits);
        check(iqk_balance(type_code(logits), logits.data_ptr(), ptr<int32_t>(ids), ptr<uint8_t>(mask), groups, tokens,
                          experts, k, ptr<uint32_t>(work), ptr<float>(s.loss), ptr<int32_t>(s.counts),
                          ptr<int32_t>(s.kept), stream_of(logits)),
              "iqk_balance");
    }
    return s;
}

struct Balance : torch::autograd::Function<Balance> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &ids,
                                 const std::optional<Tensor> &given) {
        const Tensor mask = given.value_or(Tensor());
        const BalanceSums s = balance_forward(logits, ids, mask);
        ctx->mark_non_differentiable({s.counts});
        ctx->set_materialize_grads(false);
        ctx->saved_data["k"] = ids.size(-1);
        ctx->save_for_backward({logits, s.counts, s.kept, mask});
        return {s.loss, s.counts};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_capture();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &counts = saved[1], &kept = saved[2], &mask = saved[3];
        const Tensor dloss = grads[0].detach().to(at::kFloat).contiguous();
        const int64_t experts = logits.size(-1), tokens = logits.size(-2), groups = kept.numel();
        Tensor dlogits = empty(logits.sizes(), logits.scalar_type(), logits);
        check(iqk_balance_grad(type_code(logits), logits.data_ptr(), ptr<uint8_t>(mask), ptr<int32_t>(counts),
                               ptr<int32_t>(kept), ptr<float>(dloss), groups, tokens, experts,
                               ctx->saved_data["k"].toInt(), dlogits.data_ptr(), stream_of(logits)),
              "iqk_balance_grad");
        auto out = once(dlogits, grads, logits);
        out.resize(3);
        return out;
    }
};

// ------------------------------------------------------------ 4-bit modules ---

int64_t mx_scale_stride(int64_t cols) { return (cols + 127) / 128 * 4; }

// The module's outputs for n_pairs pairs: [n_pairs, ...] of `shape`.
Tensor mx_project(int64_t act, const Tensor &rows, const Tensor &scales, int64_t scale_stride, const Tensor &tiles,
                  const Tensor &tile_scales, const Tensor &row_exps, const Tensor &ids, c10::IntArrayRef shape,
                  int64_t in, int64_t pairs, int64_t rows_per_pair, int64_t per_row, bool grouped) {
    const int64_t experts = tiles.size(0), out = shape.back();
    Tensor y = empty(shape, act & 1 ? at::kBFloat16 : at::kHalf, rows);
    if (!y.numel()) return y;
    const int64_t n_x_rows = rows.numel() / rows.size(-1);
    const bool wide = ids.defined() && ids.scalar_type() == at::kLong;
    auto *const xs = ptr<uint8_t>(scales);
    auto *const ts = ptr<uint8_t>(tile_scales);
    auto *const ex = ptr<int32_t>(row_exps);
    void *const stream = stream_of(rows);
    if (!grouped) {
        check(iqk_mx_pairs(int(act), in, out, experts, rows.data_ptr(), n_x_rows, xs, scale_stride, tiles.data_ptr(),
                           ts, ex, ptr<void>(ids), wide, per_row, pairs, y.data_ptr(), stream),
              "iqk_mx_pairs");
    } else if (!ids.defined()) {
        check(iqk_mx_groups(int(act), in, out, experts, rows.data_ptr(), n_x_rows, xs, scale_stride, tiles.data_ptr(),
                            ts, ex, nullptr, nullptr, nullptr, pairs, y.data_ptr(), stream),
              "iqk_mx_groups");
    } else {
        const Tensor work = empty({2 * pairs * rows_per_pair + experts + 1}, at::kInt, rows);
        check(iqk_mx_prefill(int(act), in, out, experts, rows.data_ptr(), n_x_rows, xs, scale_stride,
                             tiles.data_ptr(), ts, ex, ids.data_ptr(), wide, pairs, rows_per_pair, per_row,
                             ptr<uint32_t>(work), y.data_ptr(), stream),
              "iqk_mx_prefill");
    }
    return y;
}

// ------------------------------------------------------------------ Python ---

const Tensor &tensor(PyObject *o) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a tensor");
    return THPVariable_Unpack(o);
}
Tensor tensor_or_none(PyObject *o) { return o == Py_None ? Tensor() : tensor(o); }
int64_t integer(PyObject *o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
void arguments(Py_ssize_t got, Py_ssize_t want) {
    TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got);
}
PyObject *pair(const Tensor &a, const Tensor &b) {
    PyObject *const x = THPVariable_Wrap(a), *const y = THPVariable_Wrap(b), *const t = PyTuple_New(2);
    PyTuple_SET_ITEM(t, 0, x);
    PyTuple_SET_ITEM(t, 1, y);
    return t;
}
bool wants_grad(const Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// The kernels carry no tangents, and a tensor that has one need not require a gradient.
void refuse_tangent(const Tensor &t, const char *name) {
    TORCH_CHECK(!t._fw_grad(0).defined(), name, " has a forward-mode derivative, which the kernels do not carry");
}

// topk(logits, k, normalize) -> (weights, ids); logits contiguous
PyObject *py_topk(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 3);
    const Tensor &logits = tensor(args[0]);
    const int64_t k = integer(args[1]);
    const bool normalize = integer(args[2]) != 0;
    refuse_tangent(logits, "logits");
    if (wants_grad(logits)) {
        const auto out = TopK::apply(logits, k, normalize);
        return pair(out[0], out[1]);
    }
    const auto [weights, ids] = topk_forward(logits, k, normalize);
    return pair(weights, ids);
    END_HANDLE_TH_ERRORS
}

// balance(logits, ids, mask) -> (loss, counts); all contiguous, mask may be None
PyObject *py_balance(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 3);
    const Tensor &logits = tensor(args[0]), &ids = tensor(args[1]);
    const Tensor mask = tensor_or_none(args[2]);
    refuse_tangent(logits, "logits");
    if (wants_grad(logits)) {
        const auto out = Balance::apply(logits, ids, mask.defined() ? std::optional<Tensor>(mask) : std::nullopt);
        return pair(out[0], out[1]);
    }
    const BalanceSums s = balance_forward(logits, ids, mask);
    return pair(s.loss, s.counts);
    END_HANDLE_TH_ERRORS
}

// Whether the kernels take t as it is: on a GPU, dense, at a 16-byte boundary, not empty.
bool ready(const Tensor &t) {
    return t.is_cuda() && t.is_contiguous() && t.dim() && t.numel() &&
           (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0;
}

// mx_quantize(x, row_stride) -> (codes, scales); with a row_stride of 0 x is looked
// at first, and the answer is None where it is no such tensor
PyObject *py_mx_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 2);
    const Tensor &x = tensor(args[0]);
    int64_t row_stride = integer(args[1]);
    if (row_stride == 0) {
        const auto type = x.scalar_type();
        if ((type != at::kFloat && type != at::kHalf && type != at::kBFloat16) || !ready(x) || x.size(-1) % 32 ||
            wants_grad(x))
            Py_RETURN_NONE;
        row_stride = x.size(-1);
    }
    refuse_tangent(x, "x");
    const int64_t cols = x.size(-1), stride = mx_scale_stride(cols);
    auto shape = x.sizes().vec();
    shape.back() = cols / 2;
    const Tensor codes = empty(shape, at::kByte, x);
    shape.back() = stride;
    Tensor scales = empty(shape, at::kByte, x);
    if (x.numel())
        check(iqk_mx_quantize(type_code(x), x.data_ptr(), x.numel() / cols, cols, row_stride, ptr<uint8_t>(codes),
                              ptr<uint8_t>(scales), stride, stream_of(x)),
              "iqk_mx_quantize");
    if (stride * 32 != cols) scales = scales.narrow(-1, 0, cols / 32);
    return pair(codes, scales);
    END_HANDLE_TH_ERRORS
}

// mx_dequantize(codes, scales, scale_stride, like) -> values of the type of
// IQK_* code `like`; with a scale_stride of 0 codes and scales are looked at first, and
// the answer is None where they are not ready or scales' rows not evenly spaced
PyObject *py_mx_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 4);
    const Tensor &codes = tensor(args[0]), &scales = tensor(args[1]);
    int64_t stride = integer(args[2]);
    const int64_t type = integer(args[3]);
    if (stride == 0) {
        const int64_t dim = scales.dim();
        if (!ready(codes) || scales.stride(-1) != 1) Py_RETURN_NONE;
        stride = dim > 1 ? scales.stride(-2) : scales.size(-1);
        for (int64_t i = dim - 3; i >= 0; --i)
            if (scales.stride(i) != scales.stride(i + 1) * scales.size(i + 1)) Py_RETURN_NONE;
        if (stride < scales.size(-1)) Py_RETURN_NONE;
    }
    auto shape = codes.sizes().vec();
    const int64_t cols = shape.back() *= 2;
    const Tensor y = empty(shape, type == IQK_F32 ? at::kFloat : type == IQK_F16 ? at::kHalf : at::kBFloat16, codes);
    if (y.numel())
        check(iqk_mx_dequantize(int(type), ptr<uint8_t>(codes), ptr<uint8_t>(scales), y.numel() / cols, cols, stride,
                                y.data_ptr(), stream_of(codes)),
              "iqk_mx_dequantize");
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// mx_project(act, rows, scales | None, scale_stride, tiles, tile_scales, row_exps,
//            ids | None, shape, in_features, pairs, rows_per_pair, pairs_per_x_row, grouped) -> y
PyObject *py_mx_project(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 14);
    refuse_tangent(tensor(args[1]), "x");
    c10::SmallVector<int64_t, 8> shape;
    TORCH_CHECK_TYPE(PyTuple_Check(args[8]), "the shape is a tuple");
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[8]); ++i) shape.push_back(integer(PyTuple_GET_ITEM(args[8], i)));
    return THPVariable_Wrap(mx_project(integer(args[0]), tensor(args[1]), tensor_or_none(args[2]), integer(args[3]),
                                       tensor(args[4]), tensor(args[5]), tensor(args[6]), tensor_or_none(args[7]),
                                       shape, integer(args[9]), integer(args[10]), integer(args[11]),
                                       integer(args[12]), integer(args[13]) != 0));
    END_HANDLE_TH_ERRORS
}

PyObject *source_hash(PyObject *, PyObject *) { return PyUnicode_FromString(IQK_SOURCE_HASH); }
PyObject *binding_hash(PyObject *, PyObject *) { return PyUnicode_FromString(IQK_BINDING_HASH); }

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    METHOD(topk), METHOD(balance), METHOD(mx_quantize), METHOD(mx_dequantize), METHOD(mx_project),
    {"source_hash", source_hash, METH_NOARGS, "digest of the kernel sources this binding was built with"},
    {"binding_hash", binding_hash, METH_NOARGS, "digest of this binding's own source and torch's version"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_iqk_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__iqk_torch(void) { return PyModule_Create(&module); }
