// The eager calls of the 4-bit modules, the router and the adapters on torch tensors: what
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
#include <c10/core/DeviceGuard.h>
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
// comes from above and on `saved`, the forward's tensor that the formula is of (if any): the
// node that raises stands between it and them, so that a derivative in either meets it.
variable_list once(Tensor grad, const variable_list &above, const Tensor &saved) {
    const bool of_saved = saved.defined() && saved.requires_grad();
    if (!at::GradMode::is_enabled() || !(of_saved || torch::autograd::any_variable_requires_grad(above))) return {grad};
    variable_list inputs{grad};
    if (saved.defined()) inputs.push_back(saved);
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

// ---------------------------------------------------- sort, dispatch, combine ---

struct Sorted {
    Tensor offsets, ids, tokens, slots;
};

// A tensor of its own in a part of base's storage.  (An allocation takes 1 us, this a tenth.)
Tensor part_of(const Tensor &base, int64_t offset, c10::IntArrayRef shape) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
}

// The lists of ids [..., k], each at 16 bytes of one allocation.
Sorted empty_lists(const Tensor &ids, int64_t experts) {
    const int64_t pairs = ids.numel();
    const auto whole = [](int64_t n) { return (n + 3) / 4 * 4; };
    const int64_t ids_at = whole(experts + 1), tokens_at = ids_at + whole(pairs), slots_at = tokens_at + whole(pairs);
    const Tensor all = empty({slots_at + whole(pairs)}, at::kInt, ids);
    return {part_of(all, 0, {experts + 1}), part_of(all, ids_at, {pairs}), part_of(all, tokens_at, {pairs}),
            part_of(all, slots_at, ids.sizes())};
}

Tensor sort_work(const Tensor &ids, int64_t experts) {
    const int64_t k = ids.size(-1), words = iqk_sort_work(ids.numel() / k, k, experts);
    check(words < 0 ? IQK_ERR_GEOMETRY : IQK_OK, "iqk_sort_work");
    return words > 0 ? empty({words}, at::kInt, ids) : Tensor();
}

// ids [..., k], contiguous, i32 or i64
Sorted sort_pairs(const Tensor &ids, int64_t experts) {
    const int64_t k = ids.size(-1), tokens = ids.numel() / k;
    const Sorted s = empty_lists(ids, experts);
    const Tensor work = sort_work(ids, experts);
    check(iqk_sort(ids.data_ptr(), ids.scalar_type() == at::kLong, tokens, k, experts, ptr<uint32_t>(work),
                   ptr<int32_t>(s.offsets), ptr<int32_t>(s.ids), ptr<int32_t>(s.tokens), ptr<int32_t>(s.slots),
                   stream_of(ids)),
          "iqk_sort");
    return s;
}

// The number of slots that have an expert, the last of the offsets.
const int32_t *kept(const Tensor &offsets) {
    return offsets.defined() ? ptr<int32_t>(offsets) + offsets.numel() - 1 : nullptr;
}

// x [tokens, cols] by ids [tokens, k]: the rows, and the lists in `s`.
Tensor dispatch_forward(const Tensor &x, const Tensor &ids, int64_t experts, const Sorted &s) {
    const int64_t k = ids.size(-1), tokens = ids.numel() / k, cols = x.size(-1);
    Tensor rows = empty({tokens * k, cols}, x.scalar_type(), x);
    const Tensor work = sort_work(ids, experts);
    check(iqk_dispatch(type_code(x), x.data_ptr(), ids.data_ptr(), ids.scalar_type() == at::kLong, tokens, k, experts,
                       cols, ptr<uint32_t>(work), ptr<int32_t>(s.offsets), ptr<int32_t>(s.ids), ptr<int32_t>(s.tokens),
                       ptr<int32_t>(s.slots), rows.data_ptr(), stream_of(x)),
          "iqk_dispatch");
    return rows;
}

// The sum of a token's rows: [..., cols], weights' leading shape (slots' without weights).
Tensor combine_forward(const Tensor &y, const Tensor &weights, const Tensor &slots, const Tensor &offsets,
                       const Tensor &add) {
    const Tensor &pairs = weights.defined() ? weights : slots;
    auto shape = pairs.sizes().vec();
    const int64_t k = shape.back(), cols = y.size(-1);
    shape.back() = cols;
    Tensor out = empty(shape, y.scalar_type(), y);
    check(iqk_combine(type_code(y), y.data_ptr(), ptr<int32_t>(slots), kept(offsets), ptr<float>(weights),
                      ptr<void>(add), pairs.numel() / k, k, cols, out.data_ptr(), stream_of(y)),
          "iqk_combine");
    return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    // the lists are written here, and the caller's
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &ids, int64_t experts,
                                 const Tensor &offsets, const Tensor &sorted_ids, const Tensor &tokens,
                                 const Tensor &slots) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({slots, offsets});
        return {dispatch_forward(x, ids, experts, {offsets, sorted_ids, tokens, slots})};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_capture();
        if (!grads[0].defined()) return variable_list(7);
        const auto saved = ctx->get_saved_variables();
        const c10::DeviceGuard guard(grads[0].device());
        const Tensor dx = combine_forward(grads[0].detach().contiguous(), Tensor(), saved[0], saved[1], Tensor());
        auto out = once(dx, grads, Tensor());
        out.resize(7);
        return out;
    }
};

struct Combine : torch::autograd::Function<Combine> {
    static variable_list forward(AutogradContext *ctx, const Tensor &y, const Tensor &weights,
                                 const std::optional<Tensor> &slots, const std::optional<Tensor> &offsets,
                                 const std::optional<Tensor> &add, bool permutation) {
        ctx->set_materialize_grads(false);
        const bool dy = y.requires_grad(), dw = weights.requires_grad();
        ctx->saved_data["dy"] = dy;
        ctx->saved_data["dw"] = dw;
        ctx->saved_data["dadd"] = add && add->requires_grad();
        ctx->saved_data["permutation"] = permutation;  // of the slots: each row has one pair, which writes its gradient
        ctx->saved_data["shape"] = y.sizes().vec();
        const Tensor s = slots.value_or(Tensor()), o = offsets.value_or(Tensor());
        // y for the weights' gradient only, which is the larger by far
        ctx->save_for_backward({dw ? y : Tensor(), dy || dw ? weights : Tensor(), s, o});
        return {combine_forward(y, weights, s, o, add.value_or(Tensor()))};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        refuse_capture();
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const Tensor &y = saved[0], &weights = saved[1], &slots = saved[2], &offsets = saved[3];
        const c10::DeviceGuard guard(grads[0].device());
        const Tensor dout = grads[0].detach().contiguous();
        Tensor dy, dweights;
        if (ctx->saved_data["dy"].toBool()) dy = empty(ctx->saved_data["shape"].toIntVector(), dout.scalar_type(), dout);
        if (ctx->saved_data["dw"].toBool()) dweights = empty(weights.sizes(), at::kFloat, dout);
        if (dy.defined() || dweights.defined()) {
            const int64_t k = weights.size(-1), tokens = weights.numel() / k;
            const bool rows_apart = dy.defined() && !ctx->saved_data["permutation"].toBool();
            if (rows_apart) {
                const Tensor work = empty({2 * weights.numel()}, at::kInt, dout);
                check(iqk_combine_grad_rows(type_code(dout), dout.data_ptr(), ptr<int32_t>(slots), kept(offsets),
                                            ptr<float>(weights), tokens, k, dout.size(-1), ptr<uint32_t>(work),
                                            dy.data_ptr(), stream_of(dout)),
                      "iqk_combine_grad_rows");
            }
            check(iqk_combine_grad(type_code(dout), dout.data_ptr(), ptr<void>(y), ptr<int32_t>(slots), kept(offsets),
                                   ptr<float>(weights), tokens, k, dout.size(-1), rows_apart ? nullptr : ptr<void>(dy),
                                   ptr<float>(dweights), stream_of(dout)),
                  "iqk_combine_grad");
            if (dy.defined()) out[0] = once(dy, grads, weights)[0];
            if (dweights.defined()) out[1] = once(dweights, grads, y)[0];
        }
        if (ctx->saved_data["dadd"].toBool()) out[4] = grads[0];
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

PyObject *tuple(std::initializer_list<Tensor> tensors) {
    PyObject *const t = PyTuple_New(Py_ssize_t(tensors.size()));
    Py_ssize_t i = 0;
    for (const Tensor &x : tensors) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
    return t;
}

// Whether the sort and row calls take t as it is: dense, on a GPU (of like's device).
bool dense(const Tensor &t) { return t.is_cuda() && t.dim() && t.is_contiguous(); }
bool dense(const Tensor &t, const Tensor &like) { return dense(t) && t.get_device() == like.get_device(); }

bool rows_type(const Tensor &t) {
    const auto type = t.scalar_type();
    return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

constexpr int64_t kPairs = int64_t(1) << 31;  // fewer than these
constexpr int64_t kMaxK = 64, kMaxExperts = 1024, kMaxCols = int64_t(1) << 28;

bool ids_ready(const Tensor &ids, int64_t experts) {
    const auto type = ids.scalar_type();
    return (type == at::kInt || type == at::kLong) && dense(ids) && ids.size(-1) > 0 && ids.size(-1) <= kMaxK &&
           ids.numel() < kPairs && experts > 0 && experts <= kMaxExperts;
}

// Whether t is [..., cols] with the leading shape of pairs [..., k].
bool of_tokens(const Tensor &t, const Tensor &pairs, int64_t cols) {
    return t.dim() == pairs.dim() && t.size(-1) == cols && t.sizes().slice(0, t.dim() - 1) == pairs.sizes().slice(0, t.dim() - 1);
}

// The calls below answer None where an operand is not one that the kernels take as it is,
// with nothing launched: the caller says what is wrong with it, or copies it.

// sort(ids, experts) -> (offsets, ids, tokens, slots)
PyObject *py_sort(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 2);
    if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
    const Tensor &ids = tensor(args[0]);
    const int64_t experts = integer(args[1]);
    if (!ids_ready(ids, experts)) Py_RETURN_NONE;
    const c10::DeviceGuard guard(ids.device());
    const Sorted s = sort_pairs(ids, experts);
    return tuple({s.offsets, s.ids, s.tokens, s.slots});
    END_HANDLE_TH_ERRORS
}

// dispatch(x, ids, experts) -> (rows, offsets, ids, tokens, slots)
PyObject *py_dispatch(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 3);
    if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_NONE;
    const Tensor &x = tensor(args[0]), &ids = tensor(args[1]);
    const int64_t experts = integer(args[2]);
    if (!ids_ready(ids, experts) || !dense(x, ids) || !rows_type(x) || x.size(-1) <= 0 || x.size(-1) >= kMaxCols ||
        !of_tokens(x, ids, x.size(-1)))
        Py_RETURN_NONE;
    refuse_tangent(x, "x");
    const c10::DeviceGuard guard(x.device());
    const Sorted s = empty_lists(ids, experts);
    const Tensor rows = wants_grad(x) ? Dispatch::apply(x, ids, experts, s.offsets, s.ids, s.tokens, s.slots)[0]
                                      : dispatch_forward(x, ids, experts, s);
    return tuple({rows, s.offsets, s.ids, s.tokens, s.slots});
    END_HANDLE_TH_ERRORS
}

// combine(y, weights, slots | None, offsets | None, add | None, whether sort gave the slots) -> out
PyObject *py_combine(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 6);
    for (int i = 0; i < 5; ++i)
        if (!THPVariable_Check(args[i]) && (i < 2 || args[i] != Py_None)) Py_RETURN_NONE;
    const Tensor &y = tensor(args[0]), &weights = tensor(args[1]);
    const Tensor slots = tensor_or_none(args[2]), offsets = tensor_or_none(args[3]), add = tensor_or_none(args[4]);
    if (!dense(y) || !rows_type(y) || y.size(-1) <= 0 || y.size(-1) >= kMaxCols || !dense(weights, y) ||
        weights.scalar_type() != at::kFloat || weights.size(-1) <= 0 || weights.size(-1) > kMaxK ||
        weights.numel() >= kPairs || slots.defined() != offsets.defined())
        Py_RETURN_NONE;
    const int64_t cols = y.size(-1);
    if (slots.defined()) {
        if (!dense(slots, y) || slots.scalar_type() != at::kInt || slots.sizes() != weights.sizes() || !dense(offsets, y) ||
            offsets.scalar_type() != at::kInt || !offsets.numel() || y.dim() != 2 || y.size(0) != weights.numel())
            Py_RETURN_NONE;
    } else if (y.dim() != weights.dim() + 1 || y.sizes().slice(0, weights.dim()) != weights.sizes()) {
        Py_RETURN_NONE;
    }
    if (add.defined() && (!dense(add, y) || add.scalar_type() != y.scalar_type() || !of_tokens(add, weights, cols)))
        Py_RETURN_NONE;
    refuse_tangent(y, "y");
    refuse_tangent(weights, "weights");
    if (add.defined()) refuse_tangent(add, "add");
    const c10::DeviceGuard guard(y.device());
    if (wants_grad(y) || wants_grad(weights) || (add.defined() && wants_grad(add))) {
        const auto given = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
        // what sort gave is a permutation until it is written to
        const bool permutation = !slots.defined() || (args[5] == Py_True && !slots.is_inference() && slots._version() == 0);
        return THPVariable_Wrap(Combine::apply(y, weights, given(slots), given(offsets), given(add), permutation)[0]);
    }
    return THPVariable_Wrap(combine_forward(y, weights, slots, offsets, add));
    END_HANDLE_TH_ERRORS
}

// adapters(x, ids, y, down, up, scales, out | None) -> out; out may be y
PyObject *py_adapters(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arguments(n, 7);
    for (int i = 0; i < 6; ++i)
        if (!THPVariable_Check(args[i])) Py_RETURN_NONE;
    const Tensor &x = tensor(args[0]), &ids = tensor(args[1]), &y = tensor(args[2]), &down = tensor(args[3]),
                 &up = tensor(args[4]), &scales = tensor(args[5]);
    const auto type = down.scalar_type(), id_type = ids.scalar_type();
    if ((type != at::kHalf && type != at::kBFloat16) || up.scalar_type() != type || scales.scalar_type() != at::kFloat ||
        x.scalar_type() != type || y.scalar_type() != type || (id_type != at::kInt && id_type != at::kLong) ||
        !dense(down) || !dense(up, down) || !dense(scales, down) || !dense(x, down) || !dense(y, down) ||
        !ids.is_cuda() || ids.get_device() != down.get_device() || !ids.is_contiguous())
        Py_RETURN_NONE;
    TORCH_CHECK(down.dim() == 4 && up.dim() == 4 && up.size(0) == down.size(0) && 8 * up.size(1) == down.size(2) &&
                    down.size(3) == 8 && up.size(3) == 8 && scales.numel() == down.size(0),
                "the bank's tensors do not belong together: down ", down.sizes(), ", up ", up.sizes(), ", scales ",
                scales.sizes());
    const int64_t adapters = down.size(0), rank = down.size(2), in = 8 * down.size(1), out = up.size(2), lead = x.dim() - 1;
    if (x.size(-1) != in || y.size(-1) != out || y.dim() != x.dim() || ids.dim() != lead || !x.numel() ||
        x.sizes().slice(0, lead) != y.sizes().slice(0, lead) || wants_grad(x) || wants_grad(y))
        Py_RETURN_NONE;
    int64_t same = 0, rows_per_id = 1;  // the rows' shape up to some dimension, 1 from there on
    while (same < lead && ids.size(same) == x.size(same)) ++same;
    for (int64_t i = same; i < lead; ++i) {
        if (ids.size(i) != 1) Py_RETURN_NONE;
        rows_per_id *= x.size(i);
    }
    refuse_tangent(x, "x");
    refuse_tangent(y, "y");
    const c10::DeviceGuard guard(x.device());
    const int64_t rows = x.numel() / in, words = iqk_adapters_work(in, out, rank, adapters, rows);
    check(words < 0 ? IQK_ERR_GEOMETRY : IQK_OK, "iqk_adapters_work");
    const Tensor sum = args[6] == Py_None ? empty(y.sizes(), type, y) : tensor(args[6]);
    const Tensor work = words ? empty({words}, at::kInt, x) : Tensor();
    check(iqk_adapters(type_code(x), in, out, rank, adapters, x.data_ptr(), rows, ids.data_ptr(), id_type == at::kLong,
                       rows_per_id, down.data_ptr(), up.data_ptr(), ptr<float>(scales), ptr<uint32_t>(work),
                       y.data_ptr(), sum.data_ptr(), stream_of(x)),
          "iqk_adapters");
    return THPVariable_Wrap(sum);
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
    METHOD(topk), METHOD(balance), METHOD(sort), METHOD(dispatch), METHOD(combine), METHOD(adapters), METHOD(mx_quantize), METHOD(mx_dequantize), METHOD(mx_project),
    {"source_hash", source_hash, METH_NOARGS, "digest of the kernel sources this binding was built with"},
    {"binding_hash", binding_hash, METH_NOARGS, "digest of this binding's own source and torch's version"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_iqk_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__iqk_torch(void) { return PyModule_Create(&module); }
