// Distillation from a teacher's top logits (tropnn_hip_distill): the loss of
// every row and, in the same pass through the GPU, its gradient.
//
// All exponentials are powers of two: with c = log2(e) / temperature, a row of
// largest logit m has s = sum 2^(c (x - m)), l = log2 s and q = 2^(c (x - m) - l).
// The classes outside the list are summed by themselves (m_0, l_0; a bitmap in
// LDS marks the listed ones): q_0 then has the relative precision of a sum,
// where 1 - sum of the listed q would lose it as the list nears the whole
// mass, and the gradient of an unlisted class,
//   t (q_0 - p_0) / q_0 q_i = t (q_0 - p_0) 2^(c (x_i - m_0) - l_0),
// never divides by a small q_0. Sums, log-sums and the gradient are f32 (the
// sums over rows f64); the gradient is rounded once, when it is stored.
#include "logits.hpp"

namespace tropnn {
namespace {

constexpr int kListed = 3;  // log-sums a row needs: unlisted classes, listed classes, teacher

struct DistillKernelArgs {
    const void *x;
    int64_t stride;
    int vocab, k, values_dtype;
    const void *values;
    const int64_t *indices;
    const float *log_rest, *weights;
    const float *norm;  // sum of the weights, or NULL: norm_value
    float norm_value;
    float temperature, scale;
    float *row_loss;
    void *grad;
};

__device__ __forceinline__ float any_value(const void *p, int dtype, int64_t i) {
    if (dtype == TROPNN_LOGITS_F32) return static_cast<const float *>(p)[i];
    if (dtype == TROPNN_LOGITS_F16) return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
    return static_cast<float>(static_cast<const __bf16 *>(p)[i]);
}

// One list entry: its class (-1: none), the teacher's and the student's
// logits.
struct Entry {
    int at;
    float v, y;
};

// p log2(p / q) from the two logarithms, 0 where p is 0.
__device__ __forceinline__ float kl_term(float log_p, float log_q) {
    const float p = fast_exp2(log_p);
    return p == 0.f ? 0.f : p * (log_p - log_q);
}

// Joins the workgroup's sums: every lane gives its three, every thread gets
// the three totals (the same bits in every thread: each wave joins the
// waves' sums in the same tree).
template <int THREADS>
__device__ __forceinline__ void block_join(ExpSum (&v)[kListed], int &entries, float c,
                                           float (*red)[2 * kListed + 1]) {
    constexpr int kWaves = THREADS / kWave;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
    for (int i = 0; i < kListed; ++i) v[i] = wave_join(v[i], c);
    entries = wave_add(entries);
    if constexpr (kWaves > 1) {
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < kListed; ++i) {
                red[wave][2 * i] = v[i].m;
                red[wave][2 * i + 1] = v[i].s;
            }
            red[wave][2 * kListed] = static_cast<float>(entries);
        }
        __syncthreads();
        const int from = lane & (kWaves - 1);
#pragma unroll
        for (int i = 0; i < kListed; ++i) {
            v[i].m = red[from][2 * i];
            v[i].s = red[from][2 * i + 1];
        }
        float n = red[from][2 * kListed];
#pragma unroll
        for (int d = 1; d < kWaves; d <<= 1) {
#pragma unroll
            for (int i = 0; i < kListed; ++i) v[i] = lane_join(v[i], d, c);
            n += __shfl_xor(n, d, kWave);
        }
        entries = static_cast<int>(n);
    }
}

// One workgroup per row: the row is read once for its log-sums and, for the
// gradient, once more (from the caches: the rows in flight fit them).
template <typename T, int THREADS, bool REST, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(DistillKernelArgs a) {
    constexpr int N = kPerLoad<T>, kWaves = THREADS / kWave, U = 4;
    extern __shared__ uint32_t listed_bits[];  // REST: bit i: class i is in the list
    __shared__ float red[kWaves][2 * kListed + 1];
    __shared__ float loss_part[kWaves];
    const int tid = threadIdx.x, vocab = a.vocab;
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.stride;
    T *grad = GRAD ? static_cast<T *>(a.grad) + row * vocab : nullptr;
    const float weight = a.weights ? a.weights[row] : 1.f;

    auto write_zeros = [&] {
        const words4 zero = {0, 0, 0, 0};
        for (int at = tid * N; at < vocab; at += THREADS * N) {
            if (at + N <= vocab)
                store_piece(grad + at, zero);
            else
                for (int i = at; i < vocab; ++i) grad[i] = static_cast<T>(0.f);
        }
    };
    if (weight == 0.f) {
        if (GRAD) write_zeros();
        if (tid == 0) a.row_loss[row] = 0.f;
        return;
    }

    const float c = kLog2e / a.temperature;
    auto entry = [&](int j) {
        Entry e{-1, -INFINITY, -INFINITY};
        const int64_t at = a.indices[row * a.k + j];
        if (at >= 0) {
            e.v = any_value(a.values, a.values_dtype, row * a.k + j);
            if (at < vocab) {
                e.at = static_cast<int>(at);
                e.y = static_cast<float>(x[at]);
            } else {
                e.at = vocab;
                e.v = e.y = NAN;  // no such class: the row's loss and gradient are NaN
            }
        }
        return e;
    };
    const float rest = REST ? a.log_rest[row] * a.temperature : 0.f;  // as a logit
    if (REST) {
        for (int i = tid; i < (vocab + 31) / 32; i += THREADS) listed_bits[i] = 0;
        __syncthreads();
    }
    // sums[0]: classes outside the list (REST) or all classes; [1]: classes
    // in the list (REST); [2]: the teacher's mass
    ExpSum sums[kListed];
    int entries = 0;
    Entry first{-1, 0.f, 0.f};
    for (int j = tid; j < a.k; j += THREADS) {
        const Entry e = entry(j);
        if (j == tid) first = e;
        if (e.at < 0) continue;
        ++entries;
        sums[2].join(ExpSum::of(e.v), c);
        if (REST && e.at < vocab) {
            atomicOr(&listed_bits[e.at >> 5], 1u << (e.at & 31));
            sums[1].join(ExpSum::of(e.y), c);
        }
    }
    if (REST) {
        if (tid == 0) sums[2].join(ExpSum::of(rest), c);
        __syncthreads();
    }

    // log-sum of the row
    float m = -INFINITY, s = 0.f;
    auto add = [&](const words4 &w, int at) {
        float y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<T>(w, i);
        if (REST) {
            const uint32_t bits = listed_bits[at >> 5] >> (at & 31);
            if (bits & ((1u << N) - 1)) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (bits & (1u << i)) y[i] = -INFINITY;
            }
        }
        float top = y[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, y[i]);
        const float next = fmaxf(m, top);
        const float r = next == -INFINITY ? 0.f : next;  // nothing above -inf yet: the terms are 2^-inf
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) part += fast_exp2((y[i] - r) * c);
        s = s * fast_exp2((m - r) * c) + part;
        m = next;
    };
    for (int at = tid * N; at < vocab; at += U * THREADS * N) {
        words4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + u * THREADS * N < vocab) w[u] = load_piece_to(x, at + u * THREADS * N, vocab);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + u * THREADS * N < vocab) add(w[u], at + u * THREADS * N);
    }
    sums[0].m = m;
    sums[0].s = s;
    block_join<THREADS>(sums, entries, c, red);

    if (entries == 0) {  // no list: nothing to learn from this row
        if (GRAD) write_zeros();
        if (tid == 0) a.row_loss[row] = 0.f;
        return;
    }
    const ExpSum unlisted = sums[0];
    ExpSum all = sums[0];
    if (REST) all.join(sums[1], c);
    const float l = log2f(all.s), l_rest = REST ? log2f(unlisted.s) : l, l_teacher = log2f(sums[2].s);
    auto log_q = [&](float y) { return fmaf(y - all.m, c, -l); };
    auto log_p = [&](float v) { return fmaf(v - sums[2].m, c, -l_teacher); };

    float part = 0.f;
    for (int j = tid; j < a.k; j += THREADS) {
        const Entry e = j == tid ? first : entry(j);
        if (e.at >= 0) part += kl_term(log_p(e.v), log_q(e.y));
    }
    float p0 = 0.f, q0 = 1.f;
    if (REST) {
        const float log_q0 = fmaf(unlisted.m - all.m, c, l_rest - l);
        p0 = fast_exp2(log_p(rest));
        q0 = fast_exp2(log_q0);
        if (tid == 0) part += kl_term(log_p(rest), log_q0);
    }
    part = wave_sum(part);
    if ((tid & (kWave - 1)) == 0) loss_part[tid / kWave] = part;

    const float norm = a.norm ? *a.norm : a.norm_value;
    const float scale = a.temperature * a.scale * weight / norm;
    if (GRAD) {
        // where every unlisted class is -inf, theirs is 0
        const bool none = REST && unlisted.m == -INFINITY && unlisted.s == 0.f;
        const float outer = none ? 0.f : REST ? scale * (q0 - p0) : scale;
        const float ref = none ? 0.f : unlisted.m, l_ref = none ? 0.f : l_rest;
        for (int at = tid * N; at < vocab; at += THREADS * N) {
            const words4 w = load_piece_to(x, at, vocab);
            float g[N];
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = outer * fast_exp2(fmaf(piece_value<T>(w, i) - ref, c, -l_ref));
            const words4 o = make_piece<T>(g);
            if (at + N <= vocab) {
                store_piece(grad + at, o);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (at + i < vocab) grad[at + i] = static_cast<T>(g[i]);
            }
        }
    }
    __syncthreads();  // the row's stores come before the listed classes'
    if (GRAD) {
        for (int j = tid; j < a.k; j += THREADS) {
            const Entry e = j == tid ? first : entry(j);
            if (e.at >= 0 && e.at < vocab)
                grad[e.at] = static_cast<T>(scale * (fast_exp2(log_q(e.y)) - fast_exp2(log_p(e.v))));
        }
    }
    if (tid == 0) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += loss_part[w];
        a.row_loss[row] = weight * a.temperature * a.temperature * kLn2 * sum;
    }
}

constexpr int kSumThreads = 1024;

__device__ double block_sum_f64(double v, double *red) {
    v = wave_add(v);
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kSumThreads / kWave; ++w) s += red[w];
    return s;
}

// out[0] = scale * sum of v (n values, in a fixed order) / (norm[0], or
// norm_value where norm is NULL)
__global__ __launch_bounds__(kSumThreads) void distill_sum_kernel(const float *v, int64_t n, float scale,
                                                                  const float *norm, float norm_value, float *out) {
    __shared__ double red[kSumThreads / kWave];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kSumThreads) s += static_cast<double>(v[i]);
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) *out = static_cast<float>(static_cast<double>(scale) * s / static_cast<double>(norm ? *norm : norm_value));
}

template <typename T>
__global__ __launch_bounds__(256) void scale_in_place_kernel(T *x, int64_t n, const float *factor) {
    constexpr int N = kPerLoad<T>;
    const float f = *factor;
    if (f == 1.f) return;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * N;
    for (int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * N; at < n; at += step) {
        if (at + N <= n) {
            const words4 w = load_piece(x + at);
            float v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = piece_value<T>(w, i) * f;
            store_piece(x + at, make_piece<T>(v));
        } else {
            for (int64_t i = at; i < n; ++i) x[i] = static_cast<T>(static_cast<float>(x[i]) * f);
        }
    }
}

template <typename T, int THREADS>
hipError_t launch_rows(const DistillKernelArgs &k, int64_t rows, int lds, hipStream_t stream) {
    auto go = [&](auto kernel) -> hipError_t {
        if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void *>(kernel), lds); e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(rows)), dim3(THREADS), lds, stream, k);
        return hipGetLastError();
    };
    if (k.log_rest)
        return k.grad ? go(distill_row_kernel<T, THREADS, true, true>) : go(distill_row_kernel<T, THREADS, true, false>);
    return k.grad ? go(distill_row_kernel<T, THREADS, false, true>) : go(distill_row_kernel<T, THREADS, false, false>);
}

}  // namespace

// 16 bytes for the sum of the weights, then a loss per row.
size_t distill_workspace(const LogitRows &x, int, bool) { return 16 + sizeof(float) * static_cast<size_t>(x.rows); }

hipError_t launch_distill(const DistillArgs &a, void *workspace, hipStream_t stream) {
    float *norm = static_cast<float *>(workspace), *row_loss = norm + 4;
    const bool sum_weights = a.mean && a.weights;
    DistillKernelArgs k{a.x.p, a.x.stride, a.x.vocab, a.k, a.values_dtype, a.values, a.indices, a.log_rest, a.weights,
                        sum_weights ? norm : nullptr, a.mean ? static_cast<float>(a.x.rows) : 1.f, a.temperature,
                        a.scale, row_loss, a.grad};
    if (sum_weights) {
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kSumThreads), 0, stream, a.weights, a.x.rows, 1.f,
                           static_cast<const float *>(nullptr), 1.f, norm);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (a.x.rows > 0) {
        const int lds = a.log_rest ? (a.x.vocab + 31) / 32 * 4 : 0;
        hipError_t e = with_logit_type(a.x.dtype, [&](auto t) {
            using T = decltype(t);
            const int pieces = (a.x.vocab + kPerLoad<T> - 1) / kPerLoad<T>;
            if (pieces <= 256) return launch_rows<T, 64>(k, a.x.rows, lds, stream);
            if (pieces <= 2048) return launch_rows<T, 256>(k, a.x.rows, lds, stream);
            return launch_rows<T, 1024>(k, a.x.rows, lds, stream);
        });
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kSumThreads), 0, stream, static_cast<const float *>(row_loss),
                       a.x.rows, a.scale, static_cast<const float *>(k.norm), k.norm_value, a.loss);
    return hipGetLastError();
}

hipError_t launch_scale_in_place(int64_t n, void *x, int dtype, const float *factor, hipStream_t stream) {
    return with_logit_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int64_t pieces = (n + kPerLoad<T> - 1) / kPerLoad<T>;
        const int64_t blocks = (pieces + 255) / 256;
        hipLaunchKernelGGL(scale_in_place_kernel<T>, dim3(static_cast<uint32_t>(blocks < 8192 ? blocks : 8192)), dim3(256), 0,
                           stream, static_cast<T *>(x), n, factor);
        return hipGetLastError();
    });
}

}  // namespace tropnn
