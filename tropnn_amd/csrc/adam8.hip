// Adam / AdamW step whose states are held in 8 bits (tropnn_hip_adam8_step in
// include/tropnn_hip_train.h): the first moment m and the root u of the second
// as e4m3 numbers, 32 of them to a power of two.
//
// The root, and not the second moment itself: it has half the exponent range,
// so e4m3 keeps elements 2^18 below their block's largest, and m / u comes
// straight from it. Both are rounded at random with the expected value kept:
// an average that moves by 1 - beta of itself a step stands still under rounding
// to nearest once that is less than half an e4m3 step (1/32 to 1/16 of the
// value), which beta2 = 0.999 always is. On normal gradients, 3000 steps at
// beta2 = 0.999, u ends 2.6 times too small by rounding to nearest, and at
// random right in the mean with 14 % of noise. A root above 0 stays above 0
// (the smallest number), so that a first moment never meets a denominator of
// eps alone. The parameter takes the step before m and u are rounded.
#include "train.hpp"

namespace tropnn {
namespace {

constexpr int kThreads = 256;
constexpr int kEach = 4;                           // elements of a thread: 16 bytes of the parameter, and
constexpr int kChunk = kEach * kThreads;           // those of a workgroup
constexpr int kLanes = TROPNN_STATE_BLOCK / kEach;  // lanes whose elements share an exponent
constexpr int kGroup = 50;                         // tensors of one launch: their arguments fill most of 4 KB
static_assert(kLanes == 8, "half a row of lanes shares an exponent");
static_assert(kGroup <= 64, "a bit per tensor");

struct StepArgs {
    float *steps[256];
    int n, first;
    double lr, beta1, beta2;
    float2 *scalars;
};

// Counts the step and forms the scalars that depend on it, in f64:
// lr / (1 - beta1^t) and 1 / sqrt(1 - beta2^t).
__global__ __launch_bounds__(256) void adam8_count_kernel(StepArgs a) {
    const int k = threadIdx.x;
    if (k >= a.n) return;
    const float step = *a.steps[k] + 1.f;
    *a.steps[k] = step;
    const double t = static_cast<double>(step);
    a.scalars[a.first + k] = make_float2(static_cast<float>(a.lr / (1.0 - pow(a.beta1, t))),
                                         static_cast<float>(1.0 / sqrt(1.0 - pow(a.beta2, t))));
}

struct Tensor8 {
    float *p;
    const float *g;
    uint8_t *m, *m_exp, *u, *u_exp;
    const float *step;
    int64_t numel;
};

struct KernelArgs {
    Tensor8 t[kGroup];
    uint32_t first_chunk[kGroup];  // of the grid
    uint32_t skip[kGroup];         // chunks of the tensor that come before
    int tensor[kGroup];            // its number among all of the call's
    uint64_t aligned;  // bit k: p and g are 16-byte aligned, m and u 4-byte aligned
    const float2 *scalars;
    float beta1, beta2, w1, w2, eps;
    float decay, coupled;  // 1 - lr wd, or 1; wd, or 0
    int n;
};

// What an exponent byte stands for: 2^(b - 127).
__device__ __forceinline__ float unit_of(uint32_t b) { return __builtin_bit_cast(float, b ? b << 23 : 0x400000u); }

// The largest over the lanes of a block.
__device__ __forceinline__ float block_most(float v) {
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    return fmaxf(v, dpp_mov<0x141>(v));
}

// The largest finite size of a block's values, of which this lane has four.
__device__ __forceinline__ float block_most(const float (&v)[kEach]) {
    float most = block_most(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))));  // passes over NaN
    if (__any(most == INFINITY)) {
        most = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) most = fabsf(v[i]) < INFINITY ? fmaxf(most, fabsf(v[i])) : most;
        most = block_most(most);
    }
    return most;
}

// The least exponent byte at which `most` is no more than 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t exponent_of(float most) {
    const uint32_t k = (__builtin_bit_cast(uint32_t, most) + 0x1fffffu) >> 23;
    return k > 8 ? k - 8 : 0;
}

// |v| in e4m3 with exponent byte b, rounded up where the 20 bits behind the
// code pass 2^20 with the random ones; 0x7f (NaN) for what is not finite.
// Scaled by 2^-120 more, an f32's exponent field is e4m3's, subnormals included.
__device__ __forceinline__ uint32_t code_of(float v, uint32_t b, uint32_t random16) {
    const float x = __builtin_amdgcn_ldexpf(fabsf(v), 7 - static_cast<int>(b));
    return min((__builtin_bit_cast(uint32_t, x) + (random16 << 4 | 8u)) >> 20, 0x7fu);
}

__device__ __forceinline__ uint32_t random_of(uint32_t x) {
    x = (x ^ x >> 16) * 0x6A09E667u;
    x = (x ^ x >> 15) * 0x3C6EF373u;
    return x ^ x >> 16;
}

// Square roots of numbers that are not negative: an approximate reciprocal root and
// one Newton step whose residual an fma has exactly (Markstein's sequence). With
// a reciprocal root that is off by a unit in the last place, 4 of the 16.8 million
// f32 in [1, 4) get the one beside the nearest. Numbers below 2^-100, whose residual
// would leave f32, are rare and taken by the library's form. So is infinity, of
// which the sequence makes a NaN, and so is NaN, which counts as infinity: a root
// past f32 is held as NaN, and a gradient of NaN makes the first moment NaN too.
__device__ __forceinline__ void roots_of(float (&x)[kEach]) {
    float root[kEach];
    uint32_t least = ~0u;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const float y = fminf(__builtin_amdgcn_rsqf(x[i]), 0x1p51f);  // of 0: the root is 0
        const float s = x[i] * y;
        root[i] = fmaf(fmaf(-s, s, x[i]), 0.5f * y, s);
        least = min(least, __builtin_bit_cast(uint32_t, x[i]) - 1u);  // 0 comes last
    }
    const float all = (root[0] + root[1]) + (root[2] + root[3]);  // finite, or one of them is NaN
    if (__any(least < __builtin_bit_cast(uint32_t, 0x1p-100f) || all != all)) {
#pragma unroll 1
        for (int i = 0; i < kEach; ++i) root[i] = !(x[i] < INFINITY) ? INFINITY : x[i] < 0x1p-100f ? sqrtf(x[i]) : root[i];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = root[i];
}

// A thread's elements: m and u as codes, in and out, with their exponent bytes.
struct Elements {
    float p[kEach], g[kEach];
    uint32_t m, u, m_exp, u_exp;
};

__device__ __forceinline__ void decode(uint32_t w, uint32_t exponent, float (&v)[kEach]) {
    const float unit = unit_of(exponent);
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    v[0] = low[0] * unit;
    v[1] = low[1] * unit;
    v[2] = high[0] * unit;
    v[3] = high[1] * unit;
}

// The signs of four values, each the top bit of its byte.
__device__ __forceinline__ uint32_t signs_of(const float (&v)[kEach]) {
    auto bits = [&](int i) { return __builtin_bit_cast(uint32_t, v[i]); };
    const uint32_t low = __builtin_amdgcn_perm(bits(1), bits(0), 0x0c0c0703u), high = __builtin_amdgcn_perm(bits(3), bits(2), 0x07030c0cu);
    return (low | high) & 0x80808080u;
}

// element: of the tensor, the first one; mixed: the step's share of the random
// numbers. m and the square of u are formed by the operations that the header names,
// each rounded by itself, so that their exponents do not hang on the compiler; u's
// root is as above, and the parameter's quotient is to two units in the last place.
__device__ __forceinline__ void step_elements(Elements &e, const KernelArgs &a, float2 scalars, uint32_t element, uint32_t mixed) {
#pragma clang fp contract(off)
    float m[kEach], u[kEach];
    decode(e.m, e.m_exp, m);
    decode(e.u, e.u_exp, u);
    if (a.coupled != 0.f) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) e.g[i] = e.g[i] + a.coupled * e.p[i];
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        m[i] = m[i] * a.beta1 + e.g[i] * a.w1;
        u[i] = (u[i] * u[i]) * a.beta2 + (e.g[i] * e.g[i]) * a.w2;
    }
    roots_of(u);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        // a denominator below the least normal number, which has no reciprocal here, counts as that
        const float denominator = fmaxf(fmaf(u[i], scalars.y, a.eps), 0x1p-126f);  // a root is no NaN
        e.p[i] = fmaf(-scalars.x, m[i] * __builtin_amdgcn_rcpf(denominator), e.p[i] * a.decay);
    }
    e.m_exp = exponent_of(block_most(m));
    e.u_exp = exponent_of(block_most(u));
    e.m = signs_of(m);
    e.u = 0;
    const uint32_t seed = element * 0x9E3779B9u + mixed;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const uint32_t random = random_of(seed + static_cast<uint32_t>(i) * 0x9E3779B9u);
        const uint32_t root = code_of(u[i], e.u_exp, random >> 16);
        e.m |= code_of(m[i], e.m_exp, random & 0xffffu) << 8 * i;
        e.u |= max(root, u[i] > 0.f ? 1u : 0u) << 8 * i;
    }
}

typedef float f4 __attribute__((ext_vector_type(4)));

// A chunk of a tensor per workgroup. 67 M elements (1.08 GB) take 175 us, 6.2
// TB/s, 268 M 729. At 16 bytes an element, memory leaves time for about 95 vector
// instructions each. IEEE square roots and divisions, and a test of every value
// for what is not finite, made that 110, and the time 193; eight elements a thread
// from 32 consecutive bytes, two requests a cache line, 203. NT: parameters and
// gradients go past the caches, which are worth nothing to a step that exceeds them
// (200 us without).
template <bool NT>
__global__ __launch_bounds__(kThreads) void adam8_kernel(KernelArgs a) {
    int k = 0;
    while (k < a.n - 1 && blockIdx.x >= a.first_chunk[k + 1]) ++k;
    const Tensor8 t = a.t[k];
    const int64_t at = static_cast<int64_t>(blockIdx.x - a.first_chunk[k] + a.skip[k]) * kChunk + threadIdx.x * kEach;
    const float2 scalars = a.scalars[a.tensor[k]];
    const uint32_t mixed = static_cast<uint32_t>(static_cast<int64_t>(*t.step)) * 0xBB67AE85u;
    const int64_t block = at / TROPNN_STATE_BLOCK;
    const bool there = at < t.numel, whole = (a.aligned >> k & 1) && at + kEach <= t.numel;
    Elements e{};
    if (there) {
        e.m_exp = t.m_exp[block];
        e.u_exp = t.u_exp[block];
    }
    if (whole) {
        const f4 *const from_p = reinterpret_cast<const f4 *>(t.p + at), *const from_g = reinterpret_cast<const f4 *>(t.g + at);
        const f4 p = NT ? __builtin_nontemporal_load(from_p) : *from_p, g = NT ? __builtin_nontemporal_load(from_g) : *from_g;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            e.p[i] = p[i];
            e.g[i] = g[i];
        }
        e.m = *reinterpret_cast<const uint32_t *>(t.m + at);
        e.u = *reinterpret_cast<const uint32_t *>(t.u + at);
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (at + i >= t.numel) continue;
            e.p[i] = t.p[at + i];
            e.g[i] = t.g[at + i];
            e.m |= static_cast<uint32_t>(t.m[at + i]) << 8 * i;
            e.u |= static_cast<uint32_t>(t.u[at + i]) << 8 * i;
        }
    }
    step_elements(e, a, scalars, static_cast<uint32_t>(at), mixed);
    if (whole) {
        const f4 p = {e.p[0], e.p[1], e.p[2], e.p[3]};
        if constexpr (NT)
            __builtin_nontemporal_store(p, reinterpret_cast<f4 *>(t.p + at));
        else
            *reinterpret_cast<f4 *>(t.p + at) = p;
        *reinterpret_cast<uint32_t *>(t.m + at) = e.m;
        *reinterpret_cast<uint32_t *>(t.u + at) = e.u;
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (at + i >= t.numel) continue;
            t.p[at + i] = e.p[i];
            t.m[at + i] = static_cast<uint8_t>(e.m >> 8 * i);
            t.u[at + i] = static_cast<uint8_t>(e.u >> 8 * i);
        }
    }
    if (there && threadIdx.x % kLanes == 0) {
        t.m_exp[block] = static_cast<uint8_t>(e.m_exp);
        t.u_exp[block] = static_cast<uint8_t>(e.u_exp);
    }
}

bool aligned_to(const void *p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

// The scalars of every tensor.
size_t adam8_workspace(int n) { return sizeof(float2) * static_cast<size_t>(n); }

hipError_t launch_adam8(const Adam8Args &a, void *workspace, hipStream_t stream) {
    float2 *scalars = static_cast<float2 *>(workspace);
    for (int first = 0; first < a.n; first += 256) {
        StepArgs s{};
        s.n = a.n - first < 256 ? a.n - first : 256;
        for (int k = 0; k < s.n; ++k) s.steps[k] = a.steps[first + k];
        s.first = first;
        s.lr = a.lr;
        s.beta1 = a.beta1;
        s.beta2 = a.beta2;
        s.scalars = scalars;
        hipLaunchKernelGGL(adam8_count_kernel, dim3(1), dim3(256), 0, stream, s);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    constexpr int64_t kMostChunks = 1 << 23;  // of one grid: the runtime's limit is 2^32 threads
    int next = 0;      // the tensor that comes next,
    int64_t done = 0;  // and how many of its chunks earlier launches have
    while (next < a.n) {
        KernelArgs k{};
        k.scalars = scalars;
        k.beta1 = static_cast<float>(a.beta1);
        k.beta2 = static_cast<float>(a.beta2);
        k.w1 = static_cast<float>(1.0 - a.beta1);
        k.w2 = static_cast<float>(1.0 - a.beta2);
        k.eps = static_cast<float>(a.eps);
        k.decay = a.decoupled ? static_cast<float>(1.0 - a.lr * a.weight_decay) : 1.f;
        k.coupled = a.decoupled ? 0.f : static_cast<float>(a.weight_decay);
        int64_t chunks = 0;
        while (next < a.n && k.n < kGroup && chunks < kMostChunks) {
            const int64_t all = (a.numels[next] + kChunk - 1) / kChunk;
            const int64_t take = all - done < kMostChunks - chunks ? all - done : kMostChunks - chunks;
            if (take > 0) {
                k.t[k.n] = Tensor8{a.params[next], a.grads[next], a.exp_avgs[next], a.exp_avg_exponents[next], a.roots[next],
                                   a.root_exponents[next], a.steps[next], a.numels[next]};
                if (aligned_to(a.params[next], 16) && aligned_to(a.grads[next], 16) && aligned_to(a.exp_avgs[next], 4) &&
                    aligned_to(a.roots[next], 4))
                    k.aligned |= uint64_t{1} << k.n;
                k.tensor[k.n] = next;
                k.skip[k.n] = static_cast<uint32_t>(done);
                k.first_chunk[k.n++] = static_cast<uint32_t>(chunks);
                chunks += take;
                done += take;
            }
            if (done == all) {
                ++next;
                done = 0;
            }
        }
        if (k.n == 0) break;  // what was left is empty
        // 16 M elements move more than the caches hold
        const auto kernel = chunks >= (1 << 24) / kChunk ? adam8_kernel<true> : adam8_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(chunks)), dim3(kThreads), 0, stream, k);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace tropnn
