// torch.ops.tropnn_hip.distill: the autograd operator behind
// tropnn_amd.distillation_loss, in C++ for the reason that the pairwise
// operator is (autograd_op.cpp): an eager training step then pays Python
// neither for the backward node nor for autograd's calls around it. Host code
// only: every launch goes through the C ABI of libtropnn_hip.so
// (include/tropnn_hip_logits.h), whose addresses the Python package hands over.
//
// The forward's launch writes the gradient too. The backward hands it over,
// scaled in place by the incoming gradient (a kernel reads that, and leaves the
// gradient alone where it is one), and gives it up, so that autograd can keep
// it as the logits' grad without a copy. A second backward through the same
// node computes it again from the saved inputs.

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
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
    decltype(&tropnn_hip_scale_in_place) scale_in_place = nullptr;
    decltype(&tropnn_hip_last_error) last_error = nullptr;
};
LogitsAbi g_logits_abi;
std::atomic<bool> g_logits_bound{false};

void bind_logits_abi(int64_t distill, int64_t distill_workspace_size, int64_t scale_in_place, int64_t last_error,
                     int64_t abi_version) {
    TORCH_CHECK(abi_version == TROPNN_HIP_LOGITS_ABI_VERSION, "libtropnn_hip.so has logits ABI version ", abi_version,
                ", the autograd operator was built for ", TROPNN_HIP_LOGITS_ABI_VERSION);
    TORCH_CHECK(distill != 0 && distill_workspace_size != 0 && scale_in_place != 0 && last_error != 0,
                "bind_logits_abi: NULL entry point");
    auto set = [](auto &f, int64_t address) { f = reinterpret_cast<std::decay_t<decltype(f)>>(static_cast<intptr_t>(address)); };
    set(g_logits_abi.distill, distill);
    set(g_logits_abi.distill_workspace_size, distill_workspace_size);
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

struct Loss {
    Tensor loss, grad;
};

Loss run_distill(const Tensor &logits, const Tensor &values, const Tensor &indices, const std::optional<Tensor> &log_rest,
                 const std::optional<Tensor> &weights, double temperature, double scale, bool mean, bool want_grad) {
    TORCH_CHECK(g_logits_bound.load(std::memory_order_acquire), "tropnn_hip.distill: the C ABI is not bound");
    const c10::DeviceGuard guard(logits.device());
    const Rows x = as_rows(logits);
    const Tensor v = values.contiguous(), at = indices.contiguous();
    const Tensor rest = log_rest.has_value() ? log_rest->contiguous() : Tensor();
    const Tensor w = weights.has_value() ? weights->contiguous() : Tensor();
    const auto f32 = logits.options().dtype(at::kFloat);
    Loss out;
    out.loss = at::empty({}, f32);
    if (want_grad) out.grad = at::empty(logits.sizes(), logits.options());
    const int dtype = logit_type(logits);
    const int64_t k = values.size(-1);
    const size_t bytes = g_logits_abi.distill_workspace_size(x.rows, x.vocab, dtype, k, want_grad);
    const Tensor ws = at::empty({static_cast<int64_t>(bytes)}, f32.dtype(at::kByte));
    check(g_logits_abi.distill(x.rows, x.vocab, x.stride, x.t.const_data_ptr(), dtype, k, v.const_data_ptr(),
                               logit_type(v), at.const_data_ptr<int64_t>(),
                               rest.defined() ? rest.const_data_ptr<float>() : nullptr,
                               w.defined() ? w.const_data_ptr<float>() : nullptr, static_cast<float>(temperature),
                               static_cast<float>(scale), mean, out.loss.mutable_data_ptr<float>(),
                               want_grad ? out.grad.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), bytes,
                               c10::hip::getCurrentHIPStream(logits.device().index()).stream()),
          "tropnn_hip_distill");
    return out;
}

std::optional<Tensor> some(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

struct DistillFunction : public torch::autograd::Function<DistillFunction> {
    // unit: the tensor of one that a training loop may start its backward with
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &values, const Tensor &indices,
                          const std::optional<Tensor> &log_rest, const std::optional<Tensor> &weights, double temperature,
                          double scale, bool mean, const std::optional<Tensor> &unit) {
        Loss out = run_distill(logits, values, indices, log_rest, weights, temperature, scale, mean, true);
        ctx->save_for_backward({logits, values, indices, log_rest.value_or(Tensor()), weights.value_or(Tensor())});
        ctx->saved_data["grad"] = std::move(out.grad);
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["mean"] = mean;
        if (unit.has_value()) ctx->saved_data["unit"] = *unit;
        return out.loss;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grad_outputs) {
        variable_list grads(9);  // one per forward argument
        const Tensor &incoming = grad_outputs[0];
        if (!incoming.defined()) return grads;
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0];
        const c10::DeviceGuard guard(logits.device());
        Tensor grad;
        if (auto it = ctx->saved_data.find("grad"); it != ctx->saved_data.end()) {
            grad = it->second.toTensor();
            ctx->saved_data.erase(it);
        } else {
            grad = run_distill(logits, saved[1], saved[2], some(saved[3]), some(saved[4]),
                               ctx->saved_data["temperature"].toDouble(), ctx->saved_data["scale"].toDouble(),
                               ctx->saved_data["mean"].toBool(), true)
                       .grad;
        }
        bool one = false;  // known on the host
        if (auto it = ctx->saved_data.find("unit"); it != ctx->saved_data.end()) {
            const Tensor unit = it->second.toTensor();
            one = unit._version() == 0 && unit.const_data_ptr() == incoming.const_data_ptr();
        }
        if (!one) {
            const Tensor factor = incoming.to(at::kFloat).contiguous();
            check(g_logits_abi.scale_in_place(grad.numel(), grad.mutable_data_ptr(), logit_type(grad),
                                              factor.const_data_ptr<float>(),
                                              c10::hip::getCurrentHIPStream(grad.device().index()).stream()),
                  "tropnn_hip_scale_in_place");
        }
        grads[0] = std::move(grad);
        return grads;
    }
};

Tensor distill(const Tensor &logits, const Tensor &values, const Tensor &indices, const std::optional<Tensor> &log_rest,
               const std::optional<Tensor> &weights, double temperature, double scale, bool mean,
               const std::optional<Tensor> &unit) {
    if (at::GradMode::is_enabled() && logits.requires_grad())
        return DistillFunction::apply(logits, values, indices, log_rest, weights, temperature, scale, mean, unit);
    return run_distill(logits, values, indices, log_rest, weights, temperature, scale, mean, false).loss;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tropnn_hip, m) {
    m.def("bind_logits_abi(int distill, int distill_workspace_size, int scale_in_place, int last_error, "
          "int abi_version) -> ()",
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
