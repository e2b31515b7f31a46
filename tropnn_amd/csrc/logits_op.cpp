// torch.ops.tropnn_hip.distill: the autograd operator behind
// tropnn_amd.distillation_loss, in C++ for the reason that the pairwise
// operator is (autograd_op.cpp): an eager training step then pays Python
// neither for the backward node nor for autograd's calls around it. Host code
// only: every launch goes through the C ABI of libtropnn_hip.so
// (include/tropnn_hip_logits.h), whose addresses the Python package hands over.
//
// The forward's launch writes the gradient too. The backward hands it over and
// gives it up, so that autograd can keep it as the logits' grad without a copy.
// An incoming gradient that the host does not know to be one is read by a
// kernel, which leaves the gradient alone where it is one after all. Otherwise
// an f32 gradient is scaled in place, and a 16-bit one is computed again with
// the factor before its rounding: a loss scaled against f16's underflow needs
// the bits that the unscaled gradient does not have. Either moves as many bytes
// (a read and a write of the gradient's size). A second backward through the
// same node computes the gradient again from the saved inputs. The gradient has
// no derivative of its own: where a graph of the backward is made, it hangs on a
// node that raises.

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <atomic>
#include <cstdint>
#include <optional>
#include <tuple>

#include "tropnn_hip_logits.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct LogitsAbi {
    decltype(&tropnn_hip_distill) distill = nullptr;
    decltype(&tropnn_hip_distill_workspace_size) distill_workspace_size = nullptr;
    decltype(&tropnn_hip_distill_grad) distill_grad = nullptr;
    decltype(&tropnn_hip_scale_in_place) scale_in_place = nullptr;
    decltype(&tropnn_hip_last_error) last_error = nullptr;
};
LogitsAbi g_logits_abi;
std::atomic<bool> g_logits_bound{false};

void bind_logits_abi(int64_t distill, int64_t distill_workspace_size, int64_t distill_grad, int64_t scale_in_place,
                     int64_t last_error, int64_t abi_version) {
    TORCH_CHECK(abi_version == TROPNN_HIP_LOGITS_ABI_VERSION, "libtropnn_hip.so has logits ABI version ", abi_version,
                ", the autograd operator was built for ", TROPNN_HIP_LOGITS_ABI_VERSION);
    TORCH_CHECK(distill != 0 && distill_workspace_size != 0 && distill_grad != 0 && scale_in_place != 0 && last_error != 0,
                "bind_logits_abi: NULL entry point");
    auto set = [](auto &f, int64_t address) { f = reinterpret_cast<std::decay_t<decltype(f)>>(static_cast<intptr_t>(address)); };
    set(g_logits_abi.distill, distill);
    set(g_logits_abi.distill_workspace_size, distill_workspace_size);
    set(g_logits_abi.distill_grad, distill_grad);
    set(g_logits_abi.scale_in_place, scale_in_place);
    set(g_logits_abi.last_error, last_error);
    g_logits_bound.store(true, std::memory_order_release);
}

// Status codes of the C ABI to exception types, as the ctypes bindings have them.
void check(int rc, const char *what) {
    if (rc == TROPNN_OK) return;
    const char *msg = g_logits_abi.last_error();
    TORCH_CHECK_VALUE(rc != TROPNN_ERR_INVALID_ARGUMENT, what, ": ", msg);
    TORCH_CHECK_NOT_IMPLEMENTED(rc != TROPNN_ERR_UNSUPPORTED, what, ": ", msg);
    TORCH_CHECK(false, what, ": HIP error: ", msg);
}

int logit_type(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TROPNN_LOGITS_F32;
        case at::kHalf: return TROPNN_LOGITS_F16;
        case at::kBFloat16: return TROPNN_LOGITS_BF16;
        default: TORCH_CHECK_TYPE(false, "expected f32, f16 or bf16, got ", t.scalar_type());
    }
}

// logits [..., vocab] as evenly spaced rows: where they are if they are that,
// else a copy.
struct Rows {
    Tensor t;
    int64_t rows, vocab, stride;
};
Rows as_rows(const Tensor &logits) {
    const int64_t dim = logits.dim(), vocab = logits.size(-1), rows = vocab > 0 ? logits.numel() / vocab : 0;
    if (logits.is_contiguous()) return {logits, rows, vocab, vocab};
    std::optional<int64_t> stride;  // of a row, from the innermost dimension that has more than one
    int64_t span = 1;               // rows in the dimensions seen so far
    bool even = logits.stride(-1) == 1 || vocab == 1;
    for (int64_t i = dim - 2; even && i >= 0; --i) {
        if (logits.size(i) == 1) continue;
        if (!stride) stride = logits.stride(i);
        // rows on top of each other (a broadcast dimension) are no rows of a matrix
        even = *stride >= vocab && logits.stride(i) == *stride * span;
        span *= logits.size(i);
    }
    if (even) return {logits, rows, vocab, stride.value_or(vocab)};
    return {logits.contiguous(), rows, vocab, vocab};
}

// An operator's inputs as the entry points take them.
struct Inputs {
    Rows x;
    Tensor values, indices, log_rest, weights;
    int64_t k;
    int dtype, values_dtype;
    double temperature, scale;
    bool mean;

    Inputs(const Tensor &logits, const Tensor &v, const Tensor &at, const std::optional<Tensor> &rest,
           const std::optional<Tensor> &w, double t, double s, bool m)
        : x(as_rows(logits)), values(v.contiguous()), indices(at.contiguous()),
          log_rest(rest.has_value() ? rest->contiguous() : Tensor()), weights(w.has_value() ? w->contiguous() : Tensor()),
          k(v.size(-1)), dtype(logit_type(logits)), values_dtype(logit_type(v)), temperature(t), scale(s), mean(m) {
        TORCH_CHECK(g_logits_bound.load(std::memory_order_acquire), "tropnn_hip.distill: the C ABI is not bound");
    }
    Tensor workspace() const {
        const size_t bytes = g_logits_abi.distill_workspace_size(x.rows, x.vocab, dtype, k, 1);
        return at::empty({static_cast<int64_t>(bytes)}, x.t.options().dtype(at::kByte));
    }
    // Calls `entry` with the inputs, `out...`, the workspace and the stream.
    template <typename F, typename... Out>
    void call(const char *what, F entry, const Tensor &ws, Out... out) const {
        check(entry(x.rows, x.vocab, x.stride, x.t.const_data_ptr(), dtype, k, values.const_data_ptr(), values_dtype,
                    indices.const_data_ptr<int64_t>(), log_rest.defined() ? log_rest.const_data_ptr<float>() : nullptr,
                    weights.defined() ? weights.const_data_ptr<float>() : nullptr, static_cast<float>(temperature),
                    static_cast<float>(scale), mean, out..., ws.mutable_data_ptr(), ws.nbytes(),
                    c10::hip::getCurrentHIPStream(x.t.device().index()).stream()),
              what);
    }
};

struct Loss {
    Tensor loss, grad, workspace;
};

Loss run_distill(const Tensor &logits, const Inputs &in, bool want_grad) {
    Loss out;
    out.loss = at::empty({}, logits.options().dtype(at::kFloat));
    if (want_grad) out.grad = at::empty(logits.sizes(), logits.options());
    out.workspace = in.workspace();
    in.call("tropnn_hip_distill", g_logits_abi.distill, out.workspace, out.loss.mutable_data_ptr<float>(),
            want_grad ? out.grad.mutable_data_ptr() : nullptr);
    return out;
}

std::optional<Tensor> some(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// What a backward needs beside the saved inputs, in one value: each entry of a
// context's dictionary costs a step about a microsecond of host time.
struct State : public torch::CustomClassHolder {
    Tensor grad;       // undefined once a backward has handed it over
    Tensor workspace;  // of the call that wrote grad, where tropnn_hip_distill_grad asks for it
    Tensor unit;
    double temperature = 1.0, scale = 1.0;
    bool mean = true;
};

struct DistillFunction : public torch::autograd::Function<DistillFunction> {
    // unit: the tensor of one that a training loop may start its backward with
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &values, const Tensor &indices,
                          const std::optional<Tensor> &log_rest, const std::optional<Tensor> &weights, double temperature,
                          double scale, bool mean, const std::optional<Tensor> &unit) {
        const c10::DeviceGuard guard(logits.device());
        const Inputs in(logits, values, indices, log_rest, weights, temperature, scale, mean);
        Loss out = run_distill(logits, in, true);
        ctx->save_for_backward({logits, values, indices, log_rest.value_or(Tensor()), weights.value_or(Tensor())});
        auto state = c10::make_intrusive<State>();
        state->grad = std::move(out.grad);
        if (in.dtype != TROPNN_LOGITS_F32 && mean && weights.has_value()) state->workspace = std::move(out.workspace);
        if (unit.has_value()) state->unit = *unit;
        state->temperature = temperature;
        state->scale = scale;
        state->mean = mean;
        ctx->saved_data["state"] = c10::IValue::make_capsule(std::move(state));
        return out.loss;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grad_outputs) {
        variable_list grads(9);  // one per forward argument
        const Tensor &incoming = grad_outputs[0];
        if (!incoming.defined()) return grads;
        const bool graph = at::GradMode::is_enabled();  // of this backward (create_graph)
        const at::NoGradGuard no_grad;
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0];
        const c10::DeviceGuard guard(logits.device());
        const auto state = c10::static_intrusive_pointer_cast<State>(ctx->saved_data["state"].toCapsule());
        const Tensor &unit = state->unit;
        const bool one = unit.defined() && unit._version() == 0 && unit.const_data_ptr() == incoming.const_data_ptr();
        Tensor grad = std::move(state->grad), workspace = std::move(state->workspace);
        if (!(grad.defined() && one)) {
            const Tensor factor = incoming.to(at::kFloat).contiguous();
            const float *f = factor.const_data_ptr<float>();
            if (grad.defined() && logit_type(grad) == TROPNN_LOGITS_F32) {
                check(g_logits_abi.scale_in_place(grad.numel(), grad.mutable_data_ptr(), TROPNN_LOGITS_F32, f,
                                                  c10::hip::getCurrentHIPStream(grad.device().index()).stream()),
                      "tropnn_hip_scale_in_place");
            } else {
                const Inputs in(logits, saved[1], saved[2], some(saved[3]), some(saved[4]),
                                state->temperature, state->scale, state->mean);
                const bool holds = grad.defined();
                if (!holds) grad = at::empty(logits.sizes(), logits.options());
                if (!workspace.defined()) workspace = in.workspace();
                in.call("tropnn_hip_distill_grad", g_logits_abi.distill_grad, workspace, f, static_cast<int>(holds),
                        grad.mutable_data_ptr());
            }
        }
        if (graph)
            torch::autograd::set_history(
                grad, std::make_shared<torch::autograd::Error>(
                          "distillation_loss: a derivative of its gradient was asked for, which it does not have "
                          "(the operator can be differentiated once)",
                          torch::autograd::collect_next_edges(logits, incoming)));
        grads[0] = std::move(grad);
        return grads;
    }
};

Tensor distill(const Tensor &logits, const Tensor &values, const Tensor &indices, const std::optional<Tensor> &log_rest,
               const std::optional<Tensor> &weights, double temperature, double scale, bool mean,
               const std::optional<Tensor> &unit) {
    TORCH_CHECK_NOT_IMPLEMENTED(!logits._fw_grad(/*level=*/0).defined(),
                                "distillation_loss: forward-mode differentiation is not supported");
    if (at::GradMode::is_enabled() && logits.requires_grad())
        return DistillFunction::apply(logits, values, indices, log_rest, weights, temperature, scale, mean, unit);
    const c10::DeviceGuard guard(logits.device());
    return run_distill(logits, Inputs(logits, values, indices, log_rest, weights, temperature, scale, mean), false).loss;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tropnn_hip, m) {
    m.def("bind_logits_abi(int distill, int distill_workspace_size, int distill_grad, int scale_in_place, "
          "int last_error, int abi_version) -> ()",
          &bind_logits_abi);
    // the layout that distill reads logits in, for any device: (tensor, rows, vocab, row stride)
    m.def("logit_rows(Tensor logits) -> (Tensor, int, int, int)", [](const Tensor &logits) {
        const Rows x = as_rows(logits);
        return std::make_tuple(x.t, x.rows, x.vocab, x.stride);
    });
    m.def("distill(Tensor logits, Tensor values, Tensor indices, Tensor? log_rest, Tensor? weights, "
          "float temperature, float scale, bool mean, Tensor? unit) -> Tensor",
          &distill);
}
