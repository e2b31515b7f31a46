// C ABI of the operators on rows of logits (declared in
// include/tropnn_hip_logits.h): argument validation and dispatch. Errors go
// to the per-thread channel of abi.hip. Nothing here allocates memory or
// synchronises the device.
#include <limits>

#include "logits.hpp"

namespace {

using tropnn::abi_fail;
using tropnn::abi_hip_fail;
using tropnn::abi_ok;

bool misaligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

bool is_logit_type(int dtype) {
    return dtype == TROPNN_LOGITS_F32 || dtype == TROPNN_LOGITS_F16 || dtype == TROPNN_LOGITS_BF16;
}

size_t element_size(int dtype) { return dtype == TROPNN_LOGITS_F32 ? 4 : 2; }

int check_type(const char *name, int dtype) {
    if (!is_logit_type(dtype))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "%s must be a TROPNN_LOGITS_* type, got %d", name, dtype);
    return TROPNN_OK;
}

int check_sizes(int64_t rows, int64_t vocab, int dtype, tropnn::LogitRows &x) {
    if (rows < 0 || rows > std::numeric_limits<int>::max())
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "rows must be in [0, 2^31), got %lld", (long long)rows);
    if (vocab < 1) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "vocab must be >= 1, got %lld", (long long)vocab);
    if (vocab > TROPNN_MAX_VOCAB)
        return abi_fail(TROPNN_ERR_UNSUPPORTED, "vocab=%lld exceeds the supported maximum %d", (long long)vocab,
                        TROPNN_MAX_VOCAB);
    if (int rc = check_type("dtype", dtype)) return rc;
    x = tropnn::LogitRows{nullptr, rows, vocab, static_cast<int>(vocab), dtype};
    return TROPNN_OK;
}

int check_rows(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, tropnn::LogitRows &x) {
    if (int rc = check_sizes(rows, vocab, dtype, x)) return rc;
    if (rows > 1 && row_stride < vocab)
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "row_stride must be >= vocab, got %lld", (long long)row_stride);
    if (rows > 0 && !logits) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "logits must be non-NULL");
    if (misaligned(logits, element_size(dtype)))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "logits must be aligned to their elements");
    x.p = logits;
    x.stride = row_stride;
    return TROPNN_OK;
}

int check_top(int64_t k) {
    if (k < 1) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "k must be >= 1, got %lld", (long long)k);
    if (k > TROPNN_MAX_TOP)
        return abi_fail(TROPNN_ERR_UNSUPPORTED, "k=%lld exceeds the supported maximum %d", (long long)k, TROPNN_MAX_TOP);
    return TROPNN_OK;
}

int check_temperature(float t) {
    if (!(t > 0.f) || t > std::numeric_limits<float>::max())
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "temperature must be positive and finite, got %g",
                        static_cast<double>(t));
    return TROPNN_OK;
}

int check_workspace(const void *workspace, size_t bytes, size_t need) {
    if (need > 0 && (!workspace || bytes < need || misaligned(workspace, 16)))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned and hold %zu bytes, got %zu", need,
                        workspace ? bytes : static_cast<size_t>(0));
    return TROPNN_OK;
}

// What tropnn_hip_distill and tropnn_hip_distill_grad have in common; x is
// filled in.
int check_distill(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                  const void *values, int values_dtype, const int64_t *indices, const float *log_rest,
                  const float *weights, float temperature, const void *grad, const void *workspace,
                  size_t workspace_bytes, tropnn::LogitRows &x) {
    if (int rc = check_rows(rows, vocab, row_stride, logits, dtype, x)) return rc;
    if (int rc = check_top(k)) return rc;
    if (int rc = check_temperature(temperature)) return rc;
    if (int rc = check_type("values_dtype", values_dtype)) return rc;
    if (rows > 0 && (!values || !indices))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "values and indices must be non-NULL");
    if (misaligned(values, element_size(values_dtype)) || misaligned(indices, 8) || misaligned(log_rest, 4) ||
        misaligned(weights, 4) || misaligned(grad, element_size(dtype)))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT,
                        "values, indices, log_rest, weights and grad must be aligned to their elements");
    return check_workspace(workspace, workspace_bytes, tropnn::distill_workspace(x, static_cast<int>(k), grad != nullptr));
}

int launched(const char *what, hipError_t e) { return e == hipSuccess ? abi_ok() : abi_hip_fail(what, e); }

}  // namespace

extern "C" {

int tropnn_hip_logits_abi_version(void) { return TROPNN_HIP_LOGITS_ABI_VERSION; }

size_t tropnn_hip_top_logits_workspace_size(int64_t rows, int64_t vocab, int dtype, int64_t k) {
    tropnn::LogitRows x{};
    if (check_sizes(rows, vocab, dtype, x) || check_top(k)) return 0;
    abi_ok();
    return tropnn::top_logits_workspace(x, static_cast<int>(k));
}

int tropnn_hip_top_logits(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                          float temperature, void *values, int64_t *indices, float *log_rest, void *workspace,
                          size_t workspace_bytes, tropnn_stream_t stream) {
    tropnn::LogitRows x{};
    if (int rc = check_rows(rows, vocab, row_stride, logits, dtype, x)) return rc;
    if (int rc = check_top(k)) return rc;
    if (int rc = check_temperature(temperature)) return rc;
    if (k > vocab)
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "k must be <= vocab, got %lld of %lld", (long long)k, (long long)vocab);
    if (rows == 0) return abi_ok();
    if (!values || !indices || !log_rest)
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "values, indices and log_rest must be non-NULL");
    if (misaligned(values, element_size(dtype)) || misaligned(indices, 8) || misaligned(log_rest, 4))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "values, indices and log_rest must be aligned to their elements");
    if (int rc = check_workspace(workspace, workspace_bytes, tropnn::top_logits_workspace(x, static_cast<int>(k)))) return rc;
    const tropnn::TopArgs a{x, static_cast<int>(k), temperature, values, indices, log_rest};
    return launched("top logits launch", tropnn::launch_top_logits(a, workspace, static_cast<hipStream_t>(stream)));
}

size_t tropnn_hip_distill_workspace_size(int64_t rows, int64_t vocab, int dtype, int64_t k, int want_grad) {
    tropnn::LogitRows x{};
    if (check_sizes(rows, vocab, dtype, x) || check_top(k)) return 0;
    abi_ok();
    return tropnn::distill_workspace(x, static_cast<int>(k), want_grad != 0);
}

int tropnn_hip_distill(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                       const void *values, int values_dtype, const int64_t *indices, const float *log_rest,
                       const float *weights, float temperature, float scale, int mean, float *loss, void *grad,
                       void *workspace, size_t workspace_bytes, tropnn_stream_t stream) {
    if (!loss) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "loss must be non-NULL");
    if (misaligned(loss, 4)) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "loss must be aligned to its elements");
    tropnn::LogitRows x{};
    if (int rc = check_distill(rows, vocab, row_stride, logits, dtype, k, values, values_dtype, indices, log_rest, weights,
                               temperature, grad, workspace, workspace_bytes, x))
        return rc;
    const tropnn::DistillArgs a{x, values, indices, log_rest, weights, static_cast<int>(k), values_dtype, mean != 0,
                                temperature, scale, loss, grad, nullptr, false};
    return launched("distillation launch", tropnn::launch_distill(a, workspace, static_cast<hipStream_t>(stream)));
}

int tropnn_hip_distill_grad(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                            const void *values, int values_dtype, const int64_t *indices, const float *log_rest,
                            const float *weights, float temperature, float scale, int mean, const float *factor,
                            int holds, void *grad, void *workspace, size_t workspace_bytes, tropnn_stream_t stream) {
    tropnn::LogitRows x{};
    if (int rc = check_distill(rows, vocab, row_stride, logits, dtype, k, values, values_dtype, indices, log_rest, weights,
                               temperature, grad, workspace, workspace_bytes, x))
        return rc;
    if (rows == 0) return abi_ok();
    if (!factor || !grad) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "factor and grad must be non-NULL");
    if (misaligned(factor, 4)) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "factor must be aligned to its elements");
    const tropnn::DistillArgs a{x, values, indices, log_rest, weights, static_cast<int>(k), values_dtype, mean != 0,
                                temperature, scale, nullptr, grad, factor, holds != 0};
    return launched("distillation gradient launch", tropnn::launch_distill(a, workspace, static_cast<hipStream_t>(stream)));
}

int tropnn_hip_scale_in_place(int64_t n, void *x, int dtype, const float *factor, tropnn_stream_t stream) {
    if (n < 0) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "n must be >= 0, got %lld", (long long)n);
    if (int rc = check_type("dtype", dtype)) return rc;
    if (n == 0) return abi_ok();
    if (!x || !factor) return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "x and factor must be non-NULL");
    if (misaligned(x, element_size(dtype)) || misaligned(factor, 4))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "x and factor must be aligned to their elements");
    return launched("scale launch", tropnn::launch_scale_in_place(n, x, dtype, factor, static_cast<hipStream_t>(stream)));
}

size_t tropnn_hip_sample_workspace_size(int64_t rows, int64_t vocab, int dtype) {
    tropnn::LogitRows x{};
    if (check_sizes(rows, vocab, dtype, x)) return 0;
    abi_ok();
    return tropnn::sample_workspace(x);
}

int tropnn_hip_sample(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype,
                      const float *uniforms, const float *temperatures, float temperature, const int32_t *top_ks,
                      int32_t top_k, const float *top_ps, float top_p, const float *min_ps, float min_p,
                      int64_t *tokens, float *log_probs, void *workspace, size_t workspace_bytes,
                      tropnn_stream_t stream) {
    tropnn::LogitRows x{};
    if (int rc = check_rows(rows, vocab, row_stride, logits, dtype, x)) return rc;
    if (rows == 0) return abi_ok();
    if (!uniforms || !tokens || !log_probs)
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "uniforms, tokens and log_probs must be non-NULL");
    if (misaligned(uniforms, 4) || misaligned(temperatures, 4) || misaligned(top_ks, 4) || misaligned(top_ps, 4) ||
        misaligned(min_ps, 4) || misaligned(tokens, 8) || misaligned(log_probs, 4))
        return abi_fail(TROPNN_ERR_INVALID_ARGUMENT, "arrays must be aligned to their elements");
    if (int rc = check_workspace(workspace, workspace_bytes, tropnn::sample_workspace(x))) return rc;
    const tropnn::SampleArgs a{x, uniforms, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k,
                               tokens, log_probs};
    return launched("sampling launch", tropnn::launch_sample(a, workspace, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
