// Selection in rows of logits: a teacher's record (tropnn_hip_top_logits) and
// a token drawn from a truncated distribution (tropnn_hip_sample). One
// workgroup has a row.
//
// A logit's place in the row's order is one 64-bit number, its key above the
// complement of its index: all of a row's are different, and "the first k",
// "the shortest prefix of that mass" are the logits at or above one of them.
//
// Most of a row is far from its k-th logit, so it is read once, as a stream,
// against a bound: the k-th largest of the maxima of the first slab's pieces
// (16 bytes each) cannot be above the k-th largest logit. A piece below the
// bound costs one comparison; the few others are put aside in LDS (collect)
// and end as a short list that is sorted there. A share of the mass needs the
// whole row's: the weights are summed by exponent in LDS, which gives the mass
// and the narrow range of logits in which the prefix ends. Rows that defeat
// these (thousands of equal logits at the bound, rising rows) take the exact
// search instead: a cut is found digit by digit, from the mass (a count, or the sampling weights as integers) of every
// value of the key's next eight bits among the logits that share the digits
// before (find_cut). Integer sums do not depend on their order, so neither
// does a cut or a drawn token.
#include "logits.hpp"

namespace tropnn {
namespace {

constexpr int kBins = 256;
constexpr int kSlab = 8;        // pieces of a thread that are in flight together
constexpr int kMassBins = 2048; // of a row's weights, by exponent
constexpr int kMaxSlabs = 64;
constexpr float kFixed = 1099511627776.f;  // 2^40: sampling weights are multiples of 2^-40

using u64 = unsigned long long;

// Larger is earlier in the row's order. No logit's place is 0.
__device__ __forceinline__ u64 place(uint32_t key, int i) { return (static_cast<u64>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(i)); }
__device__ __forceinline__ uint32_t place_key(u64 p) { return static_cast<uint32_t>(p >> 32); }
// Kept below n, so that no logits, however they change under the kernel, make
// it read outside their row.
__device__ __forceinline__ int place_index(u64 p, int n) {
    return static_cast<int>(min(0xffffffffu - static_cast<uint32_t>(p), static_cast<uint32_t>(n - 1)));
}

// NaN if either is.
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Logits that a workgroup can collect: eight a thread.
template <int THREADS>
constexpr int kList = THREADS < 512 ? 8 * THREADS : 4096;

// The largest logit of a piece, NaN if one is.
template <typename T>
__device__ __forceinline__ float piece_most(const words4 &w) {
    float most = piece_value<T>(w, 0);
#pragma unroll
    for (int i = 1; i < kPerLoad<T>; ++i) most = nan_max(most, piece_value<T>(w, i));
    return most;
}

template <int THREADS>
struct Shared {
    static constexpr int kWaves = THREADS / kWave;
    u64 list[kList<THREADS>];
    union {
        u64 bins[kBins];
        uint32_t counts[kBins];
    };
    u64 wave[kWaves < 2 ? 2 : kWaves];
    u64 pick[2];
    float2 wave_rest[kWaves];
    uint32_t wave_key[kWaves];
    int count;
    uint32_t bound;
};

// A row, read by the whole workgroup in pieces of kPerLoad elements.
template <typename T, int THREADS>
struct Row {
    static constexpr int N = kPerLoad<T>;
    static constexpr int kSlabLogits = THREADS * kSlab * N;
    const T *x;
    int n;

    __device__ __forceinline__ int slabs() const { return (n + kSlabLogits - 1) / kSlabLogits; }

    // The first logit of piece u of this thread in a slab.
    static __device__ __forceinline__ int at(int slab, int u) {
        return slab * kSlabLogits + (u * THREADS + static_cast<int>(threadIdx.x)) * N;
    }
    // Logits past the row's end are -inf.
    __device__ __forceinline__ void load(int slab, words4 (&w)[kSlab]) const {
        if ((slab + 1) * kSlabLogits <= n) {
#pragma unroll
            for (int u = 0; u < kSlab; ++u) w[u] = load_piece(x + at(slab, u));
        } else {
            float none[N];
#pragma unroll
            for (int i = 0; i < N; ++i) none[i] = -INFINITY;
#pragma unroll
            for (int u = 0; u < kSlab; ++u) {
                w[u] = make_piece<T>(none);
                if (at(slab, u) < n) w[u] = load_piece_to(x, at(slab, u), n);
            }
        }
    }
    // f(values, index of the first) for every piece; values past the end are
    // -inf.
    template <typename F>
    __device__ __forceinline__ void pieces(int slab, F &&f) const {
        words4 w[kSlab];
        load(slab, w);
#pragma unroll
        for (int u = 0; u < kSlab; ++u) {
            float y[N];
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = piece_value<T>(w[u], i);
            f(y, at(slab, u));
        }
    }
    // f(value, index) for every logit
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        for (int from = threadIdx.x * N; from < n; from += THREADS * N) {
            const words4 w = load_piece_to(x, from, n);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (from + i < n) f(piece_value<T>(w, i), from + i);
        }
    }
};

__device__ __forceinline__ u64 wave_scan(u64 v) {  // the lanes' sum up to and with this one
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const u64 o = __shfl_up(v, d, kWave);
        if (lane >= d) v += o;
    }
    return v;
}

// The sum of the threads' values before this one's, and of all.
template <int THREADS>
__device__ __forceinline__ u64 block_scan(u64 v, u64 &total, Shared<THREADS> &sh) {
    constexpr int kWaves = THREADS / kWave;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const u64 up = wave_scan(v);
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

template <int THREADS>
__device__ __forceinline__ u64 block_sum(u64 v, Shared<THREADS> &sh) {
    u64 total;
    block_scan(v, total, sh);
    return total;
}

// ---- the exact search, for any row ----

// The first index, in order, at which the running sum of mass(value, index)
// passes `target` (which is below the row's sum).
template <typename T, int THREADS, typename M>
__device__ int find_by_index(const Row<T, THREADS> &row, u64 target, M &&mass, Shared<THREADS> &sh) {
    constexpr int N = Row<T, THREADS>::N;
    u64 running = 0;
    __syncthreads();
    if (threadIdx.x == 0) sh.pick[0] = 0;
    for (int base = 0; base < row.n; base += THREADS * N) {
        const int at = base + static_cast<int>(threadIdx.x) * N;
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
template <typename T, int THREADS, typename M>
__device__ u64 find_cut(const Row<T, THREADS> &row, u64 limit, M &&mass, Shared<THREADS> &sh) {
    const int tid = threadIdx.x;
    uint32_t key = 0;
    u64 above = 0, ties = 0;  // mass before the digits found so far; of those that share them all
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int b = tid; b < kBins; b += THREADS) sh.bins[b] = 0;
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
            u64 before = above + wave_scan(own) - own;
            if (before < limit && limit <= before + own) {
                int digit = kBins - 1 - 4 * tid;
                while (before + sh.bins[digit] < limit) before += sh.bins[digit--];
                sh.pick[0] = static_cast<u64>(digit);  // in [0, kBins)
                sh.pick[1] = before;
            }
        }
        __syncthreads();
        const int digit = static_cast<int>(sh.pick[0]) & (kBins - 1);
        key |= static_cast<uint32_t>(digit) << shift;
        above = sh.pick[1];
        ties = sh.bins[digit];
    }
    __syncthreads();
    if (above + ties == limit) return place(key, 0x7fffffff);
    // some of the equal logits only: the first ones, by index
    return place(key, find_by_index(row, limit - above - 1, [&](float x, int i) { return logit_key(x) == key ? mass(x, i) : 0; }, sh));
}

// ---- the list ----

// Sorts `n` (a power of two) numbers in LDS, largest first. A wave's 64 pairs
// at a distance of up to 64 lie in 128 numbers that no other wave touches, so
// only the longer distances need the workgroup's barrier.
template <int THREADS>
__device__ void sort_down(u64 *v, int n) {
    bool far = true;
    for (int size = 2; size <= n; size <<= 1) {
        for (int d = size >> 1; d > 0; d >>= 1) {
            if (far || d > kWave)
                __syncthreads();
            else
                wave_lds_fence();
            far = d > kWave;
            for (int i = threadIdx.x; i < n / 2; i += THREADS) {
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

__device__ __forceinline__ int slots_for(int n) { return n <= 1 ? 1 : 1 << (32 - __builtin_clz(n - 1)); }

// Sorts the n collected logits.
template <int THREADS>
__device__ void sort_list(int n, Shared<THREADS> &sh) {
    const int slots = slots_for(n);
    __syncthreads();
    for (int i = n + static_cast<int>(threadIdx.x); i < slots; i += THREADS) sh.list[i] = 0;
    sort_down<THREADS>(sh.list, slots);
}

// The largest multiple of 2^16 that at least k of the keys reach; keys(f)
// calls f for this thread's keys, and there are at least k in all.
template <int THREADS, typename K>
__device__ uint32_t bound_of(int k, K &&keys, Shared<THREADS> &sh) {
    const int tid = threadIdx.x;
    uint32_t bound = 0, need = static_cast<uint32_t>(k);
#pragma unroll 1
    for (int shift = 24; shift >= 16; shift -= 8) {
        __syncthreads();
        for (int b = tid; b < kBins; b += THREADS) sh.counts[b] = 0;
        __syncthreads();
        keys([&](uint32_t key) {
            if (shift == 24 || (key >> 24) == (bound >> 24)) atomicAdd(&sh.counts[(key >> shift) & (kBins - 1)], 1u);
        });
        __syncthreads();
        if (tid < kWave) {
            const int top = kBins - 1 - 4 * tid;
            const u64 own = sh.counts[top] + sh.counts[top - 1] + sh.counts[top - 2] + sh.counts[top - 3];
            u64 before = wave_scan(own) - own;
            if (before < need && need <= before + own) {
                int digit = top;
                while (before + sh.counts[digit] < need) before += sh.counts[digit--];
                sh.bound = bound | static_cast<uint32_t>(digit) << shift;
                sh.pick[1] = need - before;
            }
        }
        __syncthreads();
        bound = sh.bound;
        need = static_cast<uint32_t>(sh.pick[1]);
    }
    return bound;
}

// The sum of all threads' parts (not negative), the same bits however they are
// dealt to the threads: as integers in units of 2^-40 of the largest. NaN where
// one is NaN or infinite.
template <int COUNT, int THREADS>
__device__ float sum_in_any_order(const float (&parts)[COUNT], Shared<THREADS> &sh) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) most = max(most, __builtin_bit_cast(uint32_t, parts[j]) & 0x7fffffffu);
    most = wave_max(most);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh.wave_key[threadIdx.x / kWave] = most;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < THREADS / kWave; ++v) most = max(most, sh.wave_key[v]);
    if (most >= 0x7f800000u) return NAN;
    const int up = 40 - (static_cast<int>(most >> 23) - 127);
    u64 q = 0;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) q += static_cast<u64>(ldexp(static_cast<double>(parts[j]), up));
    return static_cast<float>(ldexp(static_cast<double>(block_sum(q, sh)), -up));
}

// Reads the row once and leaves in the list every logit at or above `bound`, a
// bound that at least k logits reach (k <= kList / 4, or the whole row). A
// piece of which some logit reaches the bound of the moment is put aside as
// its largest key and its number; when the row has been read, the k-th largest
// of those keys is the last bound (no piece below it holds one of the first
// k), and the pieces put aside are read again. Where they become many before
// the end, the bound is raised early. begin(bound, most), given the first
// bound (NaN or infinite: no finite one) and, with MOST, the first slab's
// largest logit, returns the bound to take: the same, or a higher one where
// fewer than k will do. With SUM, sum(values) is added up over all that is not
// in the list, which has -inf in its place: total is this thread's share of the
// stream, extra that of the pieces put aside, whose order among the threads
// changes from run to run. Returns the number collected, in no
// particular order, or -1 if they were too many.
template <bool MOST, bool SUM, typename T, int THREADS, typename Begin, typename Sum>
__device__ int collect(const Row<T, THREADS> &row, int k, Shared<THREADS> &sh, float &bound, float &total, float &extra,
                       Begin &&begin, Sum &&sum) {
    using R = Row<T, THREADS>;
    constexpr int N = R::N, kOwn = kList<THREADS> / THREADS;
    const int slabs = row.slabs(), n = row.n, tid = threadIdx.x;
    words4 w[kSlab], next[kSlab];
    row.load(0, w);
    if (tid == 0) sh.count = 0;
    uint32_t most_key = 0;
    if constexpr (MOST) {
#pragma unroll
        for (int u = 0; u < kSlab; ++u)
            if (R::at(0, u) < n) most_key = max(most_key, logit_key(piece_most<T>(w[u])));
        most_key = wave_max(most_key);
        if ((tid & (kWave - 1)) == 0) sh.wave_key[tid / kWave] = most_key;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < THREADS / kWave; ++v) most_key = max(most_key, sh.wave_key[v]);
    }
    const bool few = (min(n, R::kSlabLogits) + N - 1) / N < k;  // pieces: then the row is one slab, bounded logit by logit
    bound = key_logit(bound_of<THREADS>(
        min(k, n),
        [&](auto &&f) {
            if (few) {
                row.each([&](float x, int) { f(logit_key(x)); });
            } else {
#pragma unroll
                for (int u = 0; u < kSlab; ++u)
                    if (R::at(0, u) < n) f(logit_key(piece_most<T>(w[u])));
            }
        },
        sh));
    bound = begin(bound, key_logit(most_key));
    total = extra = 0.f;

    // the pieces put aside, this thread's share of them, are summed or read
    // again: those that reach the bound into the list
    u64 own[kOwn];
    int aside = 0;
    auto take_own = [&] {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) own[j] = j * THREADS + tid < aside ? sh.list[j * THREADS + tid] : 0;
    };
    auto own_bound = [&] {
        return bound_of<THREADS>(
            k,
            [&](auto &&f) {
#pragma unroll
                for (int j = 0; j < kOwn; ++j)
                    if (own[j]) f(place_key(own[j]));
            },
            sh);
    };
    auto read_again = [&](u64 entry, float (&y)[N]) {
        const int at = static_cast<int>(static_cast<uint32_t>(entry)) * N;
        const words4 p = load_piece_to(row.x, at, n);
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<T>(p, i);
        return at;
    };

    __syncthreads();
    for (int slab = 0; slab < slabs; ++slab) {
        if (slab + 1 < slabs) row.load(slab + 1, next);
#pragma unroll
        for (int u = 0; u < kSlab; ++u) {
            const float most = piece_most<T>(w[u]);
            const int at = R::at(slab, u);
            const bool reaches = !(most < bound) && at < n;
            if (reaches) {
                const int slot = atomicAdd(&sh.count, 1);
                if (slot < kList<THREADS>) sh.list[slot] = static_cast<u64>(logit_key(most)) << 32 | static_cast<uint32_t>(at / N);
            }
            if constexpr (SUM) {
                float y[N];
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = piece_value<T>(w[u], i);
                const float part = sum(y);
                total += reaches ? 0.f : part;
            }
        }
        if (slab + 1 < slabs) {
            __syncthreads();
            aside = sh.count;
            if (aside > kList<THREADS>) return -1;
            __syncthreads();
            if (aside > kList<THREADS> / 2) {
                take_own();
                const uint32_t key = own_bound();
                bound = key_logit(key);
                if (tid == 0) sh.count = 0;
                __syncthreads();
                float parts[kOwn];
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    parts[j] = 0.f;
                    if (!own[j]) continue;
                    if (place_key(own[j]) >= key) {
                        sh.list[atomicAdd(&sh.count, 1)] = own[j];
                    } else if constexpr (SUM) {
                        float y[N];
                        read_again(own[j], y);
                        parts[j] = sum(y);
                    }
                }
                if constexpr (SUM) extra += sum_in_any_order(parts, sh);
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < kSlab; ++u) w[u] = next[u];
        }
    }
    __syncthreads();
    aside = sh.count;
    if (aside > kList<THREADS>) return -1;
    take_own();
    if (!few && aside > k) bound = key_logit(own_bound());
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    float parts[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        parts[j] = 0.f;
        if (!own[j]) continue;
        float y[N];
        const int at = read_again(own[j], y);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!(y[i] < bound) && at + i < n) {
                const int slot = atomicAdd(&sh.count, 1);
                if (slot < kList<THREADS>) sh.list[slot] = place(logit_key(y[i]), at + i);
                y[i] = -INFINITY;
            }
        }
        if constexpr (SUM) parts[j] = sum(y);
    }
    if constexpr (SUM) extra += sum_in_any_order(parts, sh);
    __syncthreads();
    return sh.count <= kList<THREADS> ? sh.count : -1;
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

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void top_logits_kernel(TopKernelArgs a) {
    constexpr int N = Row<T, THREADS>::N;
    __shared__ Shared<THREADS> sh;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const Row<T, THREADS> row{static_cast<const T *>(a.x) + r * a.stride, a.vocab};
    const float c = kLog2e / a.temperature;

    // The others' sum, in units of 2^(c bound): all of them are below the bound,
    // so nothing overflows, and only a rest far below it could be lost to
    // underflow.
    float bound, first_bound = 0.f, offset = 0.f, sum, extra;
    const int n = collect<false, true>(
        row, a.k, sh, bound, sum, extra,
        [&](float b, float) {
            first_bound = fabsf(b) < 1e30f ? b : 0.f;
            offset = first_bound * c;
            return b;
        },
        [&](const float (&y)[N]) {
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) part += fast_exp2(fmaf(y[i], c, -offset));
            return part;
        });
    u64 cut = 0;
    ExpSum rest;
    if (n < 0) {
        cut = find_cut(row, static_cast<u64>(a.k), [](float, int) -> u64 { return 1; }, sh);
        if (tid == 0) sh.count = 0;
        __syncthreads();
        row.each([&](float x, int i) {
            const u64 p = place(logit_key(x), i);
            if (p >= cut) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kList<THREADS>) sh.list[at] = p;
            }
        });
        sort_list(a.k, sh);
    } else {
        sort_list(n, sh);
        for (int j = a.k + tid; j < n; j += THREADS) rest.join(ExpSum::of(key_logit(place_key(sh.list[j]))), c);
    }
    for (int j = tid; j < a.k; j += THREADS) {
        const int i = place_index(sh.list[j], row.n);
        a.indices[r * a.k + j] = i;
        static_cast<T *>(a.values)[r * a.k + j] = row.x[i];
    }
    sum = wave_sum(sum);
    if ((tid & (kWave - 1)) == 0) sh.wave_key[tid / kWave] = __builtin_bit_cast(uint32_t, sum);
    __syncthreads();
    sum = extra;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) {
        const uint32_t u = sh.wave_key[w];
        sum += __builtin_bit_cast(float, u);
    }
    // where everything was collected, the list's end is the whole rest
    const bool listed = n == row.n;
    if (n < 0 || (!listed && !(sum > 0x1p-90f && sum < 0x1p90f))) {
        // out of the range of that unit: once more, each sum in its own
        cut = sh.list[a.k - 1];
        rest = ExpSum{};
        row.each([&](float x, int i) {
            if (place(logit_key(x), i) < cut) rest.join(ExpSum::of(x), c);
        });
    } else if (!listed && tid == 0) {
        ExpSum o;
        o.m = first_bound;
        o.s = sum * fast_exp2(-fmaf(first_bound, c, -offset));  // the unit's rounding
        rest.join(o, c);
    }
    rest = wave_join(rest, c);
    if ((tid & (kWave - 1)) == 0) sh.wave_rest[tid / kWave] = make_float2(rest.m, rest.s);
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < THREADS / kWave; ++w) {
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

// What a row's sampling weights need.
struct Weights {
    float m, inverse;
    __device__ __forceinline__ float of(float x) const { return x == m ? 1.f : fast_exp2((x - m) * inverse); }
    __device__ __forceinline__ u64 fixed(float x) const { return static_cast<u64>(of(x) * kFixed); }
    // the same where the largest logit is finite: 2^0 is 1
    __device__ __forceinline__ float of_finite(float x) const { return fast_exp2((x - m) * inverse); }
    __device__ __forceinline__ u64 fixed_finite(float x) const { return static_cast<u64>(of_finite(x) * kFixed); }
};

__device__ __forceinline__ u64 limit_of(float top_p, u64 sum) {
    const double part = static_cast<double>(top_p) * static_cast<double>(sum);
    return part >= 1.0 ? static_cast<u64>(part) : 1;
}

__device__ __forceinline__ u64 target_of(float u, u64 sum) {
    const double part = static_cast<double>(u) * static_cast<double>(sum);
    const u64 target = part > 0.0 ? static_cast<u64>(part) : 0;
    return target < sum ? target : sum - 1;
}

struct Drawn {
    int token;
    u64 weight, sum;
};

// The exact search for any row and parameters.
template <typename T, int THREADS>
__device__ Drawn draw_by_search(const Row<T, THREADS> &row, const Weights &w, int top_k, float top_p, float min_p, float u,
                                Shared<THREADS> &sh) {
    u64 cut = 0;
    if (top_k > 0 && top_k < row.n)
        cut = find_cut(row, static_cast<u64>(top_k), [](float, int) -> u64 { return 1; }, sh);
    auto mass = [&](float x, int i) -> u64 { return place(logit_key(x), i) >= cut ? w.fixed(x) : 0; };
    u64 sum = 0;
    if (top_p < 1.f) {
        row.each([&](float x, int i) { sum += mass(x, i); });
        cut = find_cut(row, limit_of(top_p, block_sum(sum, sh)), mass, sh);
    }
    auto kept = [&](float x, int i) -> u64 { return w.of(x) >= min_p ? mass(x, i) : 0; };
    sum = 0;
    row.each([&](float x, int i) { sum += kept(x, i); });
    Drawn d;
    d.sum = block_sum(sum, sh);
    d.token = find_by_index(row, target_of(u, d.sum), kept, sh);
    d.weight = w.fixed(static_cast<float>(row.x[d.token]));
    return d;
}

// Draws among the first `n` of the sorted list, which hold everything that
// top_k leaves or that can be kept; `limit` of the mass is top_p's.
template <int THREADS>
__device__ Drawn draw_from_list(int n, u64 limit, const Weights &w, float min_p, float u, int vocab, Shared<THREADS> &sh) {
    constexpr int kOwn = kList<THREADS> / THREADS;
    // the kept logits are the first ones of the list: how many, and their sum
    const int per = (n + THREADS - 1) / THREADS, from = static_cast<int>(threadIdx.x) * per;
    u64 own = 0;
    for (int j = 0; j < per; ++j)
        if (from + j < n) own += w.fixed(key_logit(place_key(sh.list[from + j])));
    u64 total;
    u64 before = block_scan(own, total, sh);
    u64 sum = 0;
    int kept = 0;
    for (int j = 0; j < per; ++j) {
        if (from + j < n) {
            const float x = key_logit(place_key(sh.list[from + j]));
            const u64 f = w.fixed(x);
            if (before < limit && w.of(x) >= min_p) {
                ++kept;
                sum += f;
            }
            before += f;
        }
    }
    Drawn d;
    d.sum = block_sum(sum, sh);
    kept = static_cast<int>(block_sum(static_cast<u64>(kept), sh));
    // by index: halves swapped, the larger complement of the index is first
    u64 turned[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int i = j * THREADS + static_cast<int>(threadIdx.x);
        turned[j] = i < kept ? sh.list[i] << 32 | sh.list[i] >> 32 : 0;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int i = j * THREADS + static_cast<int>(threadIdx.x);
        if (i < kept) sh.list[i] = turned[j];
    }
    sort_list(kept, sh);
    const u64 target = target_of(u, d.sum);
    const int each = (kept + THREADS - 1) / THREADS, first = static_cast<int>(threadIdx.x) * each;
    own = 0;
    for (int j = 0; j < each; ++j)
        if (first + j < kept) own += w.fixed(key_logit(static_cast<uint32_t>(sh.list[first + j])));
    before = block_scan(own, total, sh);
    if (before <= target && target < before + own) {
        int j = first;
        u64 f = w.fixed(key_logit(static_cast<uint32_t>(sh.list[j])));
        while (target >= before + f) {
            before += f;
            f = w.fixed(key_logit(static_cast<uint32_t>(sh.list[++j])));
        }
        sh.pick[0] = sh.list[j] >> 32;
        sh.pick[1] = f;
    }
    __syncthreads();
    d.token = place_index(sh.pick[0], vocab);
    d.weight = sh.pick[1];
    return d;
}

// The weights of a row's logits by exponent, largest first.
struct MassBins {
    u64 bins[kMassBins];
    u64 slab[kMaxSlabs];
};

// The bin of a weight 2^-a: a / 40 of them all, monotone in the logit.
__device__ __forceinline__ int mass_bin(float x, const Weights &w) {
    const float a = (w.m - x) * w.inverse;
    return static_cast<int>(fminf(a * (kMassBins / 40.f), static_cast<float>(kMassBins - 1)));
}

// Draws from all logits of which mass(value, index) is not 0, given the mass
// of every slab.
template <typename T, int THREADS, typename M>
__device__ Drawn draw_from_slabs(const Row<T, THREADS> &row, const u64 *slab_mass, float u, M &&mass,
                                 Shared<THREADS> &sh) {
    constexpr int N = Row<T, THREADS>::N, kWaves = THREADS / kWave;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int slabs = row.slabs();
    Drawn d;
    d.sum = 0;
    for (int s = 0; s < slabs; ++s) d.sum += slab_mass[s];
    u64 target = target_of(u, d.sum);
    int slab = 0;
    while (slab + 1 < slabs && target >= slab_mass[slab]) target -= slab_mass[slab++];
    // in that slab: which piece of which wave, by the pieces' order
    words4 p[kSlab];
    row.load(slab, p);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSlab; ++k) {
        u64 own = 0;
        const int at = Row<T, THREADS>::at(slab, k);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < row.n) own += mass(piece_value<T>(p[k], i), at + i);
        own = wave_add(own);
        if (lane == 0) sh.list[k * kWaves + wave] = own;
    }
    __syncthreads();
    constexpr int kSums = kSlab * kWaves, kEach = (kSums + kWave - 1) / kWave;
    u64 mine[kEach], all = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        mine[j] = lane * kEach + j < kSums ? sh.list[lane * kEach + j] : 0;
        all += mine[j];
    }
    u64 upto = wave_scan(all) - all;
    int which = -1;
    u64 less = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        if (upto <= target && target < upto + mine[j]) {
            which = lane * kEach + j;
            less = upto;
        }
        upto += mine[j];
    }
    const u64 holders = __ballot(which >= 0);
    const int holder = holders ? __builtin_ctzll(holders) : 0;
    which = max(__shfl(which, holder, kWave), 0);
    target -= __shfl(less, holder, kWave);
    const int from = slab * Row<T, THREADS>::kSlabLogits + which * kWave * N;
    if (wave == 0) {
        const int at = from + lane * N;
        u64 v[N], own = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = at + i < row.n ? mass(static_cast<float>(row.x[at + i]), at + i) : 0;
            own += v[i];
        }
        u64 before = wave_scan(own) - own;
        if (before <= target && target < before + own) {
            int found = -1;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (found < 0 && target < before + v[i]) {
                    found = at + i;
                    sh.pick[1] = v[i];
                }
                before += v[i];
            }
            sh.pick[0] = static_cast<u64>(found);
        }
    }
    __syncthreads();
    d.token = min(static_cast<int>(sh.pick[0]), row.n - 1);
    d.weight = sh.pick[1];
    return d;
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void sample_kernel(SampleKernelArgs a) {
    using R = Row<T, THREADS>;
    constexpr int N = R::N;
    __shared__ Shared<THREADS> sh;
    __shared__ MassBins mass;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const R row{static_cast<const T *>(a.x) + r * a.stride, a.vocab};
    const float temperature = a.temperatures ? a.temperatures[r] : a.temperature;
    const float top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    const float min_p = fminf(a.min_ps ? a.min_ps[r] : a.min_p, 1.f);
    const float u = a.uniforms[r];
    int top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    if (top_k >= row.n || top_k < 0) top_k = 0;
    const bool greedy = !(temperature > 0.f);
    // neither 0 nor inf, so that no difference of 0 and none of inf makes a NaN
    const float inverse = fminf(fmaxf(kLog2e / temperature, 1.17549435e-38f), 3.402823466e38f);
    const int slabs = row.slabs();

    auto answer = [&](int token, float log_prob) {
        if (tid == 0) {
            a.tokens[r] = token;
            a.log_probs[r] = log_prob;
        }
    };
    auto finish = [&](const Drawn &d) {
        answer(d.token, logf(static_cast<float>(static_cast<double>(d.weight) / static_cast<double>(d.sum))));
    };

    if (greedy || (top_k > 0 && top_k <= kList<THREADS> / 4)) {
        float bound, unused, none_aside;
        int n = collect<true, false>(
            row, greedy ? 1 : top_k, sh, bound, unused, none_aside,
            [&](float b, float most) {
                // what has no weight beside the largest so far is left out: rows of
                // which a mask leaves little are collected whole
                const float none = fmaxf(greedy ? most : most - 41.f / inverse, -3.402823466e38f);
                return b == b ? fmaxf(b, none) : none;
            },
            [](const float (&)[N]) { return 0.f; });
        if (n == 0) return answer(-1, NAN);  // no logit above -inf
        if (n > 0) {
            sort_list(n, sh);
            const u64 top = sh.list[0];
            const Weights w{key_logit(place_key(top)), inverse};
            if (place_key(top) == kKeyNan || place_key(top) == kKeyNegInf) return answer(-1, NAN);
            if (greedy) return answer(place_index(top, row.n), 0.f);
            if (w.m < INFINITY) {
                n = min(top_k, n);
                u64 limit = ~0ull;
                if (top_p < 1.f) {
                    u64 sum = 0;
                    for (int j = tid; j < n; j += THREADS) sum += w.fixed(key_logit(place_key(sh.list[j])));
                    limit = limit_of(top_p, block_sum(sum, sh));
                }
                return finish(draw_from_list(n, limit, w, min_p, u, row.n, sh));
            }
        }
    }

    // the largest logit
    uint32_t top = 0;
    {
        float most = -INFINITY;
        for (int s = 0; s < slabs; ++s) {
            words4 w[kSlab];
            row.load(s, w);
#pragma unroll
            for (int p = 0; p < kSlab; ++p) most = nan_max(most, piece_most<T>(w[p]));
        }
        top = wave_max(logit_key(most));
        __syncthreads();
        if ((tid & (kWave - 1)) == 0) sh.wave_key[tid / kWave] = top;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < THREADS / kWave; ++v) top = max(top, sh.wave_key[v]);
    }
    if (top == kKeyNan || top == kKeyNegInf) return answer(-1, NAN);
    if (greedy) return answer(find_by_index(row, 0, [&](float x, int) -> u64 { return logit_key(x) == top; }, sh), 0.f);
    const Weights w{key_logit(top), inverse};
    if (top_k > 0 || w.m == INFINITY) return finish(draw_by_search(row, w, top_k, top_p, min_p, u, sh));

    for (int s = tid; s < kMaxSlabs; s += THREADS) mass.slab[s] = 0;
    if (!(top_p < 1.f)) {
        auto kept = [&](float x, int) -> u64 { return w.of_finite(x) >= min_p ? w.fixed_finite(x) : 0; };
        __syncthreads();
        for (int s = 0; s < slabs; ++s) {
            u64 sum = 0;
            row.pieces(s, [&](const float (&y)[N], int) {
#pragma unroll
                for (int i = 0; i < N; ++i) sum += kept(y[i], 0);
            });
            sum = wave_add(sum);
            if ((tid & (kWave - 1)) == 0) atomicAdd(&mass.slab[s], sum);
        }
        __syncthreads();
        return finish(draw_from_slabs(row, mass.slab, u, kept, sh));
    }

    // the row's mass by exponent
    for (int b = tid; b < kMassBins; b += THREADS) mass.bins[b] = 0;
    __syncthreads();
    for (int s = 0; s < slabs; ++s) {
        row.pieces(s, [&](const float (&y)[N], int) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const u64 f = w.fixed_finite(y[i]);
                if (f) atomicAdd(&mass.bins[mass_bin(y[i], w)], f);
            }
        });
    }
    __syncthreads();
    constexpr int kOwnBins = kMassBins / THREADS;
    u64 own = 0, total;
#pragma unroll
    for (int j = 0; j < kOwnBins; ++j) own += mass.bins[tid * kOwnBins + j];
    u64 before = block_scan(own, total, sh);
    const u64 limit = limit_of(top_p, total);

    // the prefix ends in one of the bins: what is in the bins before is kept,
    // the bin's own logits are sorted
    for (int j = 0; j < kOwnBins; ++j) {
        const u64 in_bin = mass.bins[tid * kOwnBins + j];
        if (before < limit && limit <= before + in_bin) {
            sh.pick[0] = static_cast<u64>(tid * kOwnBins + j);
            sh.pick[1] = before;
        }
        before += in_bin;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const int cut_bin = static_cast<int>(sh.pick[0]);
    const u64 above = sh.pick[1];
    // below this no logit is in the bins kept (a margin of two bins)
    const float least = w.m - (static_cast<float>(cut_bin) + 3.f) * (40.f / kMassBins) / w.inverse;
    for (int s = 0; s < slabs; ++s) {
        u64 sum = 0;
        words4 p[kSlab];
        row.load(s, p);
#pragma unroll
        for (int k = 0; k < kSlab; ++k) {
            if (piece_most<T>(p[k]) < least) continue;
            const int at = R::at(s, k);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = piece_value<T>(p[k], i);
                const u64 f = w.fixed_finite(x);
                if (!f) continue;
                const int b = mass_bin(x, w);
                if (b < cut_bin) {
                    if (w.of_finite(x) >= min_p) sum += f;
                } else if (b == cut_bin) {
                    const int slot = atomicAdd(&sh.count, 1);
                    if (slot < kList<THREADS>) sh.list[slot] = place(logit_key(x), at + i);
                }
            }
        }
        sum = wave_add(sum);
        if ((tid & (kWave - 1)) == 0) atomicAdd(&mass.slab[s], sum);
    }
    __syncthreads();
    const int n = sh.count;
    if (n > kList<THREADS>) return finish(draw_by_search(row, w, top_k, top_p, min_p, u, sh));
    sort_list(n, sh);
    const int per = (n + THREADS - 1) / THREADS, from = tid * per;
    own = 0;
    for (int j = 0; j < per; ++j)
        if (from + j < n) own += w.fixed_finite(key_logit(place_key(sh.list[from + j])));
    before = above + block_scan(own, total, sh);
    __syncthreads();
    for (int j = 0; j < per; ++j) {
        if (from + j < n && before < limit) {
            const u64 p = sh.list[from + j];
            const float x = key_logit(place_key(p));
            const u64 f = w.fixed_finite(x);
            if (w.of_finite(x) >= min_p) atomicAdd(&mass.slab[place_index(p, row.n) / R::kSlabLogits], f);
            before += f;
            if (before >= limit) sh.pick[0] = p;  // the last one kept
        }
    }
    __syncthreads();
    const u64 cut = sh.pick[0];
    __syncthreads();
    finish(draw_from_slabs(
        row, mass.slab, u,
        [&](float x, int i) -> u64 {
            return place(logit_key(x), i) >= cut && w.of_finite(x) >= min_p ? w.fixed_finite(x) : 0;
        },
        sh));
}

// Threads for a row: its pieces fill a slab or a few, and no row has more
// than kMaxSlabs slabs; the list holds four times k.
int threads_for(int vocab, int per_load, int k) {
    const int pieces = (vocab + per_load - 1) / per_load;
    const int by_row = pieces <= 64 ? 64 : pieces <= 2048 ? 256 : pieces <= 8192 ? 512 : 1024;
    return max(by_row, k <= 128 ? 64 : k <= 512 ? 256 : 512);
}
static_assert(TROPNN_MAX_VOCAB / (1024 * kSlab * kPerLoad<float>) <= kMaxSlabs, "slabs of the widest row");

template <typename F>
hipError_t with_threads(int threads, F &&f) {
    switch (threads) {
        case 64: return f(std::integral_constant<int, 64>{});
        case 256: return f(std::integral_constant<int, 256>{});
        case 512: return f(std::integral_constant<int, 512>{});
        default: return f(std::integral_constant<int, 1024>{});
    }
}

}  // namespace

size_t top_logits_workspace(const LogitRows &, int) { return 0; }

hipError_t launch_top_logits(const TopArgs &a, void *, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    const TopKernelArgs k{a.x.p, a.x.stride, a.x.vocab, a.k, a.temperature, a.values, a.indices, a.log_rest};
    return with_logit_type(a.x.dtype, [&](auto t) {
        using T = decltype(t);
        return with_threads(min(512, threads_for(a.x.vocab, kPerLoad<T>, a.k)), [&](auto threads) {
            constexpr int kThreads = decltype(threads)::value;
            hipLaunchKernelGGL((top_logits_kernel<T, kThreads>), dim3(static_cast<uint32_t>(a.x.rows)), dim3(kThreads), 0, stream, k);
            return hipGetLastError();
        });
    });
}

size_t sample_workspace(const LogitRows &) { return 0; }

hipError_t launch_sample(const SampleArgs &a, void *, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    const SampleKernelArgs k{a.x.p, a.x.stride, a.x.vocab, a.uniforms, a.temperatures, a.top_ps, a.min_ps, a.top_ks,
                             a.temperature, a.top_p, a.min_p, a.top_k, a.tokens, a.log_probs};
    return with_logit_type(a.x.dtype, [&](auto t) {
        using T = decltype(t);
        return with_threads(threads_for(a.x.vocab, kPerLoad<T>, 1), [&](auto threads) {
            constexpr int kThreads = decltype(threads)::value;
            hipLaunchKernelGGL((sample_kernel<T, kThreads>), dim3(static_cast<uint32_t>(a.x.rows)), dim3(kThreads), 0, stream, k);
            return hipGetLastError();
        });
    });
}

}  // namespace tropnn
