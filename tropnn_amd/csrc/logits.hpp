// Shared by the operators on rows of logits (distill.hip, select.hip): the
// launch API that the C ABI calls, and device helpers for reading rows,
// ordering logits and reducing over a workgroup.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "device.hpp"
#include "launch.hpp"
#include "tropnn_hip_logits.h"

namespace tropnn {

// The C ABI's error channel (abi.hip), for its other translation unit.
int abi_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int abi_ok();
int abi_hip_fail(const char *where, hipError_t e);

// Rows of logits as the entry points take them.
struct LogitRows {
    const void *p;
    int64_t rows, stride;
    int vocab, dtype;
};

struct DistillArgs {
    LogitRows x;
    const void *values;
    const int64_t *indices;
    const float *log_rest, *weights;
    int k, values_dtype, mean;
    float temperature, scale;
    float *loss;  // NULL: the gradient alone
    void *grad;
    const float *factor;  // of the gradient, or NULL: 1
    bool holds;           // grad and the workspace are as a call without a factor left them
};
size_t distill_workspace(const LogitRows &x, int k, bool want_grad);
hipError_t launch_distill(const DistillArgs &a, void *workspace, hipStream_t stream);
hipError_t launch_scale_in_place(int64_t n, void *x, int dtype, const float *factor, hipStream_t stream);

struct TopArgs {
    LogitRows x;
    int k;
    float temperature;
    void *values;
    int64_t *indices;
    float *log_rest;
};
size_t top_logits_workspace(const LogitRows &x, int k);
hipError_t launch_top_logits(const TopArgs &a, void *workspace, hipStream_t stream);

struct SampleArgs {
    LogitRows x;
    const float *uniforms, *temperatures, *top_ps, *min_ps;
    const int32_t *top_ks;
    float temperature, top_p, min_p;
    int top_k;
    int64_t *tokens;
    float *log_probs;
};
size_t sample_workspace(const LogitRows &x);
hipError_t launch_sample(const SampleArgs &a, void *workspace, hipStream_t stream);

// Calls f with a value of the element type of `dtype`.
template <typename F>
auto with_logit_type(int dtype, F &&f) {
    if (dtype == TROPNN_LOGITS_F32) return f(float{});
    if (dtype == TROPNN_LOGITS_F16) return f(_Float16{});
    return f(__bf16{});
}

// A launch of a workgroup per row, in as many grids as the runtime's limit of
// 2^32 threads a grid asks for: launch(first row, rows).
template <typename F>
hipError_t by_grids(int64_t rows, F &&launch) {
    constexpr int64_t kMost = 1 << 21;  // of up to 1024 threads
    for (int64_t first = 0; first < rows; first += kMost) {
        launch(first, static_cast<uint32_t>(rows - first < kMost ? rows - first : kMost));
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

#if defined(__HIPCC__)

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;

// N = 16 / sizeof(T) consecutive elements: one 16-byte load or store. Rows
// start at any element, so the type is aligned like one element; gfx950
// takes such accesses whole.
template <typename T>
constexpr int kPerLoad = 16 / static_cast<int>(sizeof(T));
using words4 = vec_t<uint32_t, 4>;
typedef words4 __attribute__((aligned(2))) words4_at2;
typedef words4 __attribute__((aligned(4))) words4_at4;

template <typename T>
__device__ __forceinline__ words4 load_piece(const T *p) {
    if constexpr (sizeof(T) == 2)
        return *reinterpret_cast<const words4_at2 *>(p);
    else
        return *reinterpret_cast<const words4_at4 *>(p);
}

template <typename T>
__device__ __forceinline__ void store_piece(T *p, words4 w) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<words4_at2 *>(p) = w;
    else
        *reinterpret_cast<words4_at4 *>(p) = w;
}

// Element i of a piece as f32.
template <typename T>
__device__ __forceinline__ float piece_value(const words4 &w, int i) {
    // a copy of the word first: a bit cast of w[j] itself takes the bits of w[0]
    if constexpr (sizeof(T) == 4) {
        const uint32_t u = w[i];
        return __builtin_bit_cast(float, u);
    } else if constexpr (__is_same(T, __bf16)) {
        const uint32_t u = w[i >> 1];
        return __builtin_bit_cast(float, (i & 1) ? (u & 0xffff0000u) : (u << 16));
    } else {
        const uint32_t u = w[i >> 1];
        const vec_t<_Float16, 2> h = __builtin_bit_cast(vec_t<_Float16, 2>, u);
        return static_cast<float>(h[i & 1]);
    }
}

// kPerLoad f32 values rounded (to nearest even) into a piece.
template <typename T>
__device__ __forceinline__ words4 make_piece(const float (&v)[kPerLoad<T>]) {
    if constexpr (sizeof(T) == 4) {
        return words4{__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]),
                      __builtin_bit_cast(uint32_t, v[2]), __builtin_bit_cast(uint32_t, v[3])};
    } else {
        words4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            vec_t<T, 2> h;
            h[0] = static_cast<T>(v[2 * i]);
            h[1] = static_cast<T>(v[2 * i + 1]);
            w[i] = __builtin_bit_cast(uint32_t, h);
        }
        return w;
    }
}

// The piece of elements [at, at + kPerLoad) of a row of n, those past its end
// read as -inf. `at` < n.
template <typename T>
__device__ __forceinline__ words4 load_piece_to(const T *row, int at, int n) {
    constexpr int N = kPerLoad<T>;
    if (at + N <= n) return load_piece(row + at);
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = at + i < n ? static_cast<float>(row[at + i]) : -INFINITY;
    return make_piece<T>(v);
}

// The position of a logit in the order, as an integer: larger comes first.
// NaN 0xffffffff, +inf 0xff800000, -inf 0x007fffff; 0 is no logit's. 16-bit
// types convert to f32 exactly, so one key serves all three.
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 becomes +0
    const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return x != x ? 0xffffffffu : k;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;
constexpr uint32_t kKeyNan = 0xffffffffu;

// exp2 of an f32, one instruction (about one unit in the last place; results
// below the smallest normal number become 0).
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// A sum of exponentials 2^(c x) with its largest x apart: 2^(c m) s, s in
// units of the largest term. Differences x - m are taken before the product
// with c, so rows masked with the lowest finite value, all of them too, have
// the softmax of any other row. Empty: m = -inf, s = 0. A NaN term makes s
// NaN for good.
struct ExpSum {
    float m = -INFINITY, s = 0.f;
    static __device__ __forceinline__ ExpSum of(float x) {
        ExpSum t;
        t.m = x != x ? -INFINITY : x;
        t.s = x != x ? NAN : x == -INFINITY ? 0.f : 1.f;
        return t;
    }
    static __device__ __forceinline__ float rel(float x, float r, float c) { return x == r ? 1.f : fast_exp2((x - r) * c); }
    __device__ __forceinline__ void join(ExpSum o, float c) {
        const float r = fmaxf(m, o.m);
        s = r == -INFINITY ? s + o.s : s * rel(m, r, c) + o.s * rel(o.m, r, c);
        m = r;
    }
};

__device__ __forceinline__ ExpSum wave_join(ExpSum v, float c) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        ExpSum o;
        o.m = __shfl_xor(v.m, d, kWave);
        o.s = __shfl_xor(v.s, d, kWave);
        v.join(o, c);
    }
    return v;
}

// Lane l gets lane l - n's value within its row of 16 (CTRL row_shr:n), or the
// last of the row or the two rows before it (row_bcast, to the ROWS given), else
// `none`. Six of them fold a wave into its last lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_from(uint32_t v, uint32_t none = 0) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_from(float v, float none) {
    return __builtin_bit_cast(float, dpp_from<CTRL, ROWS>(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, none)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp_from(unsigned long long v) {
    const uint32_t low = dpp_from<CTRL, ROWS>(static_cast<uint32_t>(v)), high = dpp_from<CTRL, ROWS>(static_cast<uint32_t>(v >> 32));
    return static_cast<unsigned long long>(high) << 32 | low;
}
template <typename F>
__device__ __forceinline__ float wave_fold(float v, float none, F &&f) {
    v = f(v, dpp_from<0x111, 0xF>(v, none));
    v = f(v, dpp_from<0x112, 0xF>(v, none));
    v = f(v, dpp_from<0x114, 0xF>(v, none));
    v = f(v, dpp_from<0x118, 0xF>(v, none));
    v = f(v, dpp_from<0x142, 0xA>(v, none));
    v = f(v, dpp_from<0x143, 0xC>(v, none));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), kWave - 1));
}
// The wave's sum and largest value (NaN left out), in scalar registers.
__device__ __forceinline__ float wave_total(float v) {
    return wave_fold(v, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_most_of(float v) {
    return wave_fold(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

template <typename V>
__device__ __forceinline__ V wave_add(V v) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d, kWave)));
    return v;
}

#endif  // __HIPCC__

}  // namespace tropnn
