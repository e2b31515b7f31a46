// Selection in rows of logits: a teacher's record (tropnn_hip_top_logits) and
// a token drawn from a truncated distribution (tropnn_hip_sample).
//
// A logit's place in the row's order is one 64-bit number, its key above the
// complement of its index: all of a row's are different, and "the first k",
// "the shortest prefix of that mass" are the logits at or above one of them,
// the cut. A cut is found digit by digit: the mass (a count, or the sampling
// weights as integers) of every value of the key's next eight bits among the
// logits that share the digits before, summed in LDS, tells which value the
// cut has. Integer sums do not depend on their order, so neither does the cut.
#include "logits.hpp"

namespace tropnn {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 256;
constexpr float kFixed = 1099511627776.f;  // 2^40: sampling weights are multiples of 2^-40

using u64 = unsigned long long;

// Larger is earlier in the row's order. No logit's place is 0.
__device__ __forceinline__ u64 place(uint32_t key, int i) { return (static_cast<u64>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(i)); }
// Kept below n, so that no logits, however they change under the kernel, make
// it read outside their row.
__device__ __forceinline__ int place_index(u64 p, int n) {
    return static_cast<int>(min(0xffffffffu - static_cast<uint32_t>(p), static_cast<uint32_t>(n - 1)));
}

struct Shared {
    u64 bins[kBins];
    u64 wave[kWaves];
    u64 pick[2];
    uint32_t wave_key[kWaves];
    float2 wave_rest[kWaves];
    int count;
};

// A row, read by the whole workgroup in pieces of kPerLoad elements.
template <typename T>
struct Row {
    static constexpr int N = kPerLoad<T>;
    const T *x;
    int n;

    // f(value, index) for every logit
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        for (int at = threadIdx.x * N; at < n; at += kThreads * N) {
            const words4 w = load_piece_to(x, at, n);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < n) f(piece_value<T>(w, i), at + i);
        }
    }
};

// The sum of the threads' values before this one's, and of all.
__device__ __forceinline__ u64 block_scan(u64 v, u64 &total, Shared &sh) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    u64 up = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const u64 o = __shfl_up(up, d, kWave);
        if (lane >= d) up += o;
    }
    __syncthreads();
    if (lane == kWave - 1) sh.wave[wave] = up;
    __syncthreads();
    u64 before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sh.wave[w];
        total += sh.wave[w];
    }
    return before + up - v;
}

__device__ __forceinline__ u64 block_sum(u64 v, Shared &sh) {
    u64 total;
    block_scan(v, total, sh);
    return total;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, Shared &sh) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh.wave_key[threadIdx.x / kWave] = v;
    __syncthreads();
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = max(m, sh.wave_key[w]);
    return m;
}

// The first index, in order, at which the running sum of mass(value, index)
// passes `target` (which is below the row's sum).
template <typename T, typename M>
__device__ int find_by_index(const Row<T> &row, u64 target, M &&mass, Shared &sh) {
    constexpr int N = Row<T>::N;
    u64 running = 0;
    __syncthreads();
    if (threadIdx.x == 0) sh.pick[0] = 0;
    for (int base = 0; base < row.n; base += kThreads * N) {
        const int at = base + threadIdx.x * N;
        u64 v[N], own = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = at + i < row.n ? mass(static_cast<float>(row.x[at + i]), at + i) : 0;
            own += v[i];
        }
        u64 total;
        u64 before = running + block_scan(own, total, sh);
        if (before <= target && target < before + own) {
            int found = -1;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (found < 0 && target < before + v[i]) found = at + i;
                before += v[i];
            }
            sh.pick[0] = static_cast<u64>(found);
        }
        running += total;
        if (running > target) break;
    }
    __syncthreads();
    const int found = min(static_cast<int>(sh.pick[0]), row.n - 1);
    __syncthreads();
    return found;
}

// The place of the last logit of the shortest prefix of the order whose mass
// reaches `limit` (1 <= limit <= the row's mass). mass(value, index) of equal
// values is equal, or 0.
template <typename T, typename M>
__device__ u64 find_cut(const Row<T> &row, u64 limit, M &&mass, Shared &sh) {
    const int tid = threadIdx.x;
    uint32_t key = 0;
    u64 above = 0, ties = 0;  // mass before the digits found so far; of those that share them all
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < kBins) sh.bins[tid] = 0;
        __syncthreads();
        row.each([&](float x, int i) {
            const uint32_t k = logit_key(x);
            if (shift == 24 || (k >> (shift + 8)) == (key >> (shift + 8))) {
                const u64 m = mass(x, i);
                if (m) atomicAdd(&sh.bins[(k >> shift) & (kBins - 1)], m);
            }
        });
        __syncthreads();
        if (tid < kWave) {
            // lane l has bins 255 - 4 l and the three below
            u64 own = 0;
            for (int j = 0; j < 4; ++j) own += sh.bins[kBins - 1 - 4 * tid - j];
            u64 up = own;
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) {
                const u64 o = __shfl_up(up, d, kWave);
                if (tid >= d) up += o;
            }
            u64 before = above + up - own;
            if (before < limit && limit <= before + own) {
                int digit = kBins - 1 - 4 * tid;
                while (before + sh.bins[digit] < limit) before += sh.bins[digit--];
                sh.pick[0] = static_cast<u64>(digit);  // in [0, kBins)
                sh.pick[1] = before;
            }
        }
        __syncthreads();
        key |= static_cast<uint32_t>(sh.pick[0]) << shift;
        above = sh.pick[1];
        ties = sh.bins[sh.pick[0]];
    }
    __syncthreads();
    if (above + ties == limit) return place(key, 0x7fffffff);
    // some of the equal logits only: the first ones, by index
    return place(key, find_by_index(row, limit - above - 1, [&](float x, int i) { return logit_key(x) == key ? mass(x, i) : 0; }, sh));
}

// Sorts `n` (a power of two) numbers in LDS, largest first.
__device__ void sort_down(u64 *v, int n) {
    for (int size = 2; size <= n; size <<= 1) {
        for (int d = size >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += kThreads) {
                const int a = 2 * i - (i & (d - 1)), b = a + d;
                const bool down = (a & size) == 0;
                const u64 p = v[a], q = v[b];
                if ((p < q) == down) {
                    v[a] = q;
                    v[b] = p;
                }
            }
        }
    }
    __syncthreads();
}

struct TopKernelArgs {
    const void *x;
    int64_t stride;
    int vocab, k;
    float temperature;
    void *values;
    int64_t *indices;
    float *log_rest;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void top_logits_kernel(TopKernelArgs a) {
    __shared__ Shared sh;
    __shared__ u64 list[TROPNN_MAX_TOP];
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const Row<T> row{static_cast<const T *>(a.x) + r * a.stride, a.vocab};
    int slots = 1;
    while (slots < a.k) slots <<= 1;
    for (int i = tid; i < slots; i += kThreads) list[i] = 0;
    if (tid == 0) sh.count = 0;
    const u64 cut = find_cut(row, static_cast<u64>(a.k), [](float, int) -> u64 { return 1; }, sh);
    const float c = kLog2e / a.temperature;
    ExpSum rest;
    row.each([&](float x, int i) {
        const u64 p = place(logit_key(x), i);
        if (p >= cut) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < slots) list[at] = p;
        } else {
            rest.join(ExpSum::of(x), c);
        }
    });
    rest = wave_join(rest, c);
    if ((tid & (kWave - 1)) == 0) sh.wave_rest[tid / kWave] = make_float2(rest.m, rest.s);
    sort_down(list, slots);
    for (int j = tid; j < a.k; j += kThreads) {
        const int i = place_index(list[j], row.n);
        a.indices[r * a.k + j] = i;
        static_cast<T *>(a.values)[r * a.k + j] = row.x[i];
    }
    if (tid == 0) {
        for (int w = 1; w < kWaves; ++w) {
            ExpSum o;
            o.m = sh.wave_rest[w].x;
            o.s = sh.wave_rest[w].y;
            rest.join(o, c);
        }
        a.log_rest[r] = rest.m == INFINITY ? INFINITY : rest.m / a.temperature + logf(rest.s);
    }
}

struct SampleKernelArgs {
    const void *x;
    int64_t stride;
    int vocab;
    const float *uniforms, *temperatures, *top_ps, *min_ps;
    const int32_t *top_ks;
    float temperature, top_p, min_p;
    int top_k;
    int64_t *tokens;
    float *log_probs;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleKernelArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const Row<T> row{static_cast<const T *>(a.x) + r * a.stride, a.vocab};
    const float temperature = a.temperatures ? a.temperatures[r] : a.temperature;
    const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = fminf(a.min_ps ? a.min_ps[r] : a.min_p, 1.f);
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    const float u = a.uniforms[r];

    uint32_t top = 0;
    row.each([&](float x, int) { top = max(top, logit_key(x)); });
    top = block_max(top, sh);
    int token = -1;
    float log_prob = NAN;
    if (top == kKeyNan || top == kKeyNegInf) {
    } else if (!(temperature > 0.f)) {
        token = find_by_index(row, 0, [&](float x, int) -> u64 { return logit_key(x) == top; }, sh);
        log_prob = 0.f;
    } else {
        const float m = key_logit(top);
        const float inverse = fminf(fmaxf(kLog2e / temperature, 1.17549435e-38f), 3.402823466e38f);  // neither 0 nor inf
        auto weight = [&](float x) { return x == m ? 1.f : fast_exp2((x - m) * inverse); };
        auto fixed = [&](float x) { return static_cast<u64>(weight(x) * kFixed); };
        u64 cut = 0;
        if (top_k > 0 && top_k < a.vocab)
            cut = find_cut(row, static_cast<u64>(top_k), [](float, int) -> u64 { return 1; }, sh);
        auto mass = [&](float x, int i) -> u64 { return place(logit_key(x), i) >= cut ? fixed(x) : 0; };
        if (top_p < 1.f) {
            u64 sum = 0;
            row.each([&](float x, int i) { sum += mass(x, i); });
            sum = block_sum(sum, sh);
            const double part = static_cast<double>(top_p) * static_cast<double>(sum);
            const u64 limit = part >= 1.0 ? static_cast<u64>(part) : 1;
            cut = find_cut(row, limit, mass, sh);
        }
        auto kept = [&](float x, int i) -> u64 { return place(logit_key(x), i) >= cut && weight(x) >= min_p ? fixed(x) : 0; };
        u64 sum = 0;
        row.each([&](float x, int i) { sum += kept(x, i); });
        sum = block_sum(sum, sh);
        const double part = static_cast<double>(u) * static_cast<double>(sum);
        u64 target = part > 0.0 ? static_cast<u64>(part) : 0;
        if (target > sum - 1) target = sum - 1;
        token = find_by_index(row, target, kept, sh);
        log_prob = logf(static_cast<float>(static_cast<double>(fixed(static_cast<float>(row.x[token]))) / static_cast<double>(sum)));
    }
    if (tid == 0) {
        a.tokens[r] = token;
        a.log_probs[r] = log_prob;
    }
}

}  // namespace

size_t top_logits_workspace(const LogitRows &, int) { return 0; }

hipError_t launch_top_logits(const TopArgs &a, void *, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    const TopKernelArgs k{a.x.p, a.x.stride, a.x.vocab, a.k, a.temperature, a.values, a.indices, a.log_rest};
    return with_logit_type(a.x.dtype, [&](auto t) {
        hipLaunchKernelGGL(top_logits_kernel<decltype(t)>, dim3(static_cast<uint32_t>(a.x.rows)), dim3(kThreads), 0, stream, k);
        return hipGetLastError();
    });
}

size_t sample_workspace(const LogitRows &) { return 0; }

hipError_t launch_sample(const SampleArgs &a, void *, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    const SampleKernelArgs k{a.x.p, a.x.stride, a.x.vocab, a.uniforms, a.temperatures, a.top_ps, a.min_ps, a.top_ks,
                             a.temperature, a.top_p, a.min_p, a.top_k, a.tokens, a.log_probs};
    return with_logit_type(a.x.dtype, [&](auto t) {
        hipLaunchKernelGGL(sample_kernel<decltype(t)>, dim3(static_cast<uint32_t>(a.x.rows)), dim3(kThreads), 0, stream, k);
        return hipGetLastError();
    });
}

}  // namespace tropnn
