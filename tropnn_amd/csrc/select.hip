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
// search instead: a cut is found digit by digit, from the mass (a count, or the
// sampling weights as integers) of every value of the key's next eight bits
// among the logits that share the digits before (find_cut). It reads the row
// five times and more: 256 rows of 131072 bf16, 32 first of equal logits 531 us,
// of random ones 23. Integer sums do not depend on their order, so neither does
// a cut or a drawn token.
#include "logits.hpp"

namespace tropnn {
namespace {

constexpr int kBins = 256;
constexpr int kSlab = 8;        // pieces of a thread that are in flight together
constexpr int kKeyBinBits = 11;
constexpr int kKeyBins = 1 << kKeyBinBits;  // of keys, by their distance from the largest
constexpr int kKeyShift = 15;   // 2^15 keys a bin, 256 bins an octave
constexpr int kMassBins = 2048; // of a row's weights, by exponent
constexpr int kRanked = 256;    // logits sorted by counting all of them
constexpr uint32_t kCrowd = 64; // of a bin, where they are sorted by bins
constexpr uint32_t kSteps = 256; // different keys of a list sorted by key and index
constexpr int kMaxChunks = 512; // a wave's share of a slab, in the widest row
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

// Logits that a workgroup can collect: four a thread, so that of the workgroups
// of 256 as many fit a CU's LDS as its registers hold.
template <int THREADS>
constexpr int kList = 4 * THREADS;
// Of these, logits that can be among the first.
template <int THREADS>
constexpr int kSpare = kList<THREADS> < 2048 ? kList<THREADS> : 2048;

// The largest logit of a piece, NaN if one is.
template <typename T>
__device__ __forceinline__ float piece_most(const words4 &w) {
    float most = piece_value<T>(w, 0);
#pragma unroll
    for (int i = 1; i < kPerLoad<T>; ++i) most = nan_max(most, piece_value<T>(w, i));
    return most;
}

template <int THREADS, bool MASS>
struct Shared {
    static constexpr int kThreads = THREADS;
    static constexpr int kWaves = THREADS / kWave;
    u64 list[kList<THREADS>];
    union {
        u64 bins[kBins];
        uint32_t counts[kBins];
        uint32_t key_counts[kKeyBins];
        uint32_t ranks[kRanked];
        u64 mass[MASS ? kMassBins : 1];
        u64 spare[kSpare<THREADS>];
    };
    u64 wave[kWaves < 2 ? 2 : kWaves];
    u64 pick[3];
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

    // Different keys of the type differ by 2^kKeyStep at least.
    static constexpr int kKeyStep = sizeof(T) == 4 ? 0 : __is_same(T, __bf16) ? 16 : 13;
    __device__ __forceinline__ int index_bits() const { return n > 1 ? 32 - __builtin_clz(n - 1) : 0; }

    __device__ __forceinline__ int slabs() const { return (n + kSlabLogits - 1) / kSlabLogits; }

    // The first logit of piece u of this thread in a slab. A wave's pieces of
    // a slab are one chunk of the row.
    static constexpr int kChunk = kWave * kSlab * N;
    static __device__ __forceinline__ int chunk(int slab) { return slab * (THREADS / kWave) + static_cast<int>(threadIdx.x) / kWave; }
    static __device__ __forceinline__ int at(int slab, int u) {
        return chunk(slab) * kChunk + (u * kWave + (static_cast<int>(threadIdx.x) & (kWave - 1))) * N;
    }
    __device__ __forceinline__ bool full(int slab) const { return (slab + 1) * kSlabLogits <= n; }
    // Piece u of a slab; all -inf where it is not whole.
    __device__ __forceinline__ words4 load_one(int slab, int u, bool full) const {
        const int from = at(slab, u);
        if (full || from + N <= n) return load_piece(x + from);
        float none[N];
#pragma unroll
        for (int i = 0; i < N; ++i) none[i] = -INFINITY;
        return make_piece<T>(none);
    }
    // The row's last logits, where they do not fill a piece, in the slab that
    // has them; the rest of that piece is -inf.
    __device__ __forceinline__ void load_end(int slab, words4 (&w)[kSlab]) const {
        const int from = n - n % N;
        if (from == n || full(slab)) return;
        bool mine = false;
#pragma unroll
        for (int u = 0; u < kSlab; ++u) mine |= at(slab, u) == from;
        if (!mine) return;
        const words4 end = load_piece_to(x, from, n);
#pragma unroll
        for (int u = 0; u < kSlab; ++u)
            if (at(slab, u) == from) w[u] = end;
    }
    // Logits past the row's end are -inf.
    __device__ __forceinline__ void load(int slab, words4 (&w)[kSlab]) const {
        const bool whole = full(slab);
#pragma unroll
        for (int u = 0; u < kSlab; ++u) w[u] = load_one(slab, u, whole);
        load_end(slab, w);
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

// The lanes' sum up to and with this one.
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
    v += dpp_from<0x111, 0xF>(v);
    v += dpp_from<0x112, 0xF>(v);
    v += dpp_from<0x114, 0xF>(v);
    v += dpp_from<0x118, 0xF>(v);
    v += dpp_from<0x142, 0xA>(v);
    v += dpp_from<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), kWave - 1)); }
__device__ __forceinline__ u64 last_lane(u64 v) {
    return static_cast<u64>(last_lane(static_cast<uint32_t>(v >> 32))) << 32 | last_lane(static_cast<uint32_t>(v));
}

// The sum of the threads' values before this one's, and of all.
template <typename SH>
__device__ __forceinline__ u64 block_scan(u64 v, u64 &total, SH &sh) {
    constexpr int THREADS = SH::kThreads;
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

template <typename SH>
__device__ __forceinline__ u64 block_sum(u64 v, SH &sh) {
    u64 total;
    block_scan(v, total, sh);
    return total;
}

template <typename SH>
__device__ __forceinline__ uint32_t block_max(uint32_t v, SH &sh) {
    constexpr int THREADS = SH::kThreads;
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh.wave_key[threadIdx.x / kWave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) v = max(v, sh.wave_key[w]);
    return v;
}

// ---- the exact search, for any row ----

// The first index, in order, at which the running sum of mass(value, index)
// passes `target` (which is below the row's sum).
template <typename T, int THREADS, typename M, typename SH>
__device__ __forceinline__ int find_by_index(const Row<T, THREADS> &row, u64 target, M &&mass, SH &sh) {
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
template <typename T, int THREADS, typename M, typename SH>
__device__ __forceinline__ u64 find_cut(const Row<T, THREADS> &row, u64 limit, M &&mass, SH &sh) {
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
__device__ __forceinline__ void sort_down(u64 *v, int n) {
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

// Sorts the first n numbers of the list (all different), largest first.
//
// Few: a number's place is the count of larger ones; the threads share the
// counting, n^2 / THREADS comparisons against broadcast reads (80 numbers, 512
// threads: 1 us, 5 with the sorting network's chain of LDS round trips).
// More: their upper words are counted in bins that share out their range; a
// number's place is the count of the bins before and of the larger ones of its
// own bin. 16-bit logits take few different keys, 2^step apart at least; where
// the list has at most kSteps of them, each has bins of its own that share out
// the places' indices (below 2^bits). Only where a bin is crowded all the same,
// the network sorts. 500 of a row, 256 threads: 2.6 us, 9.4 with the network;
// 1024, 1024 threads: 7.6, 20 by counting.
template <typename SH>
__device__ __forceinline__ void sort_list(int n, SH &sh, int step, int bits) {
    constexpr int THREADS = SH::kThreads, kEach = kList<THREADS> / THREADS, kOwn = kKeyBins / THREADS;
    const int tid = threadIdx.x, slots = slots_for(max(n, kWave));
    __syncthreads();
    if (slots <= min(kRanked, THREADS)) {
        const int i = tid & (slots - 1), part = tid / slots, parts = THREADS / slots;
        const int per = (n + parts - 1) / parts, to = min(n, (part + 1) * per);
        const u64 v = i < n ? sh.list[i] : 0;
        if (part == 0) sh.ranks[i] = 0;
        uint32_t rank = 0;
#pragma unroll 4
        for (int j = part * per; j < to; ++j) rank += sh.list[j] > v;
        __syncthreads();
        if (i < n && rank) atomicAdd(&sh.ranks[i], rank);
        __syncthreads();
        if (part == 0 && i < n) sh.list[min(static_cast<int>(sh.ranks[i]), n - 1)] = v;
        __syncthreads();
        return;
    }
    const int lane = tid & (kWave - 1), wave = tid / kWave;
    u64 v[kEach];
    uint32_t most = 0, least = 0;  // the least one's complement
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int j = tid + e * THREADS;
        v[e] = j < n ? sh.list[j] : 0;
        if (j < n) {
            most = max(most, place_key(v[e]));
            least = max(least, ~place_key(v[e]));
        }
    }
    most = wave_max(most);
    least = wave_max(least);
    if (lane == 0) sh.wave[wave] = static_cast<u64>(most) << 32 | least;
    for (int b = tid; b < kKeyBins; b += THREADS) sh.key_counts[b] = 0;
    if (tid == 0) sh.bound = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) {
        most = max(most, place_key(sh.wave[w]));
        least = max(least, static_cast<uint32_t>(sh.wave[w]));
    }
    const uint32_t span = most - ~least;
    const int shift = span < kKeyBins ? 0 : 21 - __builtin_clz(span);  // span >> shift < kKeyBins
    const bool stepped = (span >> step) < kSteps;
    const int each = kKeyBinBits - (span >> step ? 32 - __builtin_clz(span >> step) : 0);  // log2 of a key's own bins
    const int index_shift = max(bits - each, 0);
    auto bin_of = [&](u64 p) {
        const uint32_t below = most - place_key(p);
        return min(stepped ? (below >> step) << each | (~static_cast<uint32_t>(p) >> index_shift) : below >> shift,
                   static_cast<uint32_t>(kKeyBins - 1));
    };
    uint32_t before[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (tid + e * THREADS < n) before[e] = atomicAdd(&sh.key_counts[bin_of(v[e])], 1u);
    __syncthreads();
    uint32_t count[kOwn], own = 0, crowd = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        count[j] = sh.key_counts[tid * kOwn + j];
        own += count[j];
        crowd = max(crowd, count[j]);
    }
    const uint32_t upto = wave_scan(own);
    if (lane == kWave - 1) sh.wave_key[wave] = upto;
    if (crowd > kCrowd) sh.bound = 1;
    __syncthreads();
    if (sh.bound) {
        const int padded = slots_for(n);
        for (int i = n + tid; i < padded; i += THREADS) sh.list[i] = 0;
        sort_down<THREADS>(sh.list, padded);
        return;
    }
    uint32_t from = upto - own;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) from += w < wave ? sh.wave_key[w] : 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        sh.key_counts[tid * kOwn + j] = from;
        from += count[j];
    }
    __syncthreads();
    // bin by bin
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (tid + e * THREADS < n) sh.list[min(sh.key_counts[bin_of(v[e])] + before[e], static_cast<uint32_t>(n - 1))] = v[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if (tid + e * THREADS < n) {
            const uint32_t bin = bin_of(v[e]), first = sh.key_counts[bin];
            const uint32_t end = bin + 1 < kKeyBins ? sh.key_counts[bin + 1] : static_cast<uint32_t>(n);
            before[e] = first;
            for (uint32_t j = first; j < end; ++j) before[e] += sh.list[j] > v[e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (tid + e * THREADS < n) sh.list[min(before[e], static_cast<uint32_t>(n - 1))] = v[e];
    __syncthreads();
}

// A key that at least k of the given ones reach, and few more; keys(f) calls f
// for this thread's, and there are at least k in all. The keys are counted by
// their distance from the largest, in bins of 2^15: of a positive largest they
// resolve 2^-8 of it over eight octaves, as finely as bf16, and spread even keys
// of one exponent over many bins (the threads' additions to one bin go one by
// one). Where the k-th is farther, digit by digit: 16 bits of it.
template <typename K, typename SH>
__device__ __forceinline__ uint32_t bound_of(int k, K &&keys, SH &sh) {
    constexpr int THREADS = SH::kThreads;
    constexpr int kOwn = kKeyBins / THREADS;
    const int tid = threadIdx.x;
    const uint32_t wanted = static_cast<uint32_t>(k);
    uint32_t most = 0;
    keys([&](uint32_t key) { most = max(most, key); });
    most = wave_max(most);
    __syncthreads();
    if ((tid & (kWave - 1)) == 0) sh.wave_key[tid / kWave] = most;
    for (int b = tid; b < kKeyBins; b += THREADS) sh.key_counts[b] = 0;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < THREADS / kWave; ++v) most = max(most, sh.wave_key[v]);
    keys([&](uint32_t key) { atomicAdd(&sh.key_counts[min((most - key) >> kKeyShift, static_cast<uint32_t>(kKeyBins - 1))], 1u); });
    __syncthreads();
    uint32_t own = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) own += sh.key_counts[tid * kOwn + j];
    const uint32_t upto = wave_scan(own);
    if ((tid & (kWave - 1)) == kWave - 1) sh.wave_key[tid / kWave] = upto;
    __syncthreads();
    uint32_t before = upto - own;
#pragma unroll
    for (int v = 0; v < THREADS / kWave; ++v) before += v < tid / kWave ? sh.wave_key[v] : 0;
    if (before < wanted && wanted <= before + own) {
        int bin = tid * kOwn;
        while (before + sh.key_counts[bin] < wanted) before += sh.key_counts[bin++];
        sh.bound = static_cast<uint32_t>(bin);
    }
    __syncthreads();
    const uint32_t bin = sh.bound;
    // a bin holds the keys down to most - (bin + 1) * 2^15 + 1
    if (bin < kKeyBins - 1) {
        const uint32_t span = ((bin + 1) << kKeyShift) - 1;
        return most > span ? most - span : 0;
    }

    uint32_t bound = 0, need = wanted;
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
            const uint32_t four = sh.counts[top] + sh.counts[top - 1] + sh.counts[top - 2] + sh.counts[top - 3];
            uint32_t above = wave_scan(four) - four;
            if (above < need && need <= above + four) {
                int digit = top;
                while (above + sh.counts[digit] < need) above += sh.counts[digit--];
                sh.bound = bound | static_cast<uint32_t>(digit) << shift;
                sh.pick[1] = need - above;
            }
        }
        __syncthreads();
        bound = sh.bound;
        need = static_cast<uint32_t>(sh.pick[1]);
    }
    return bound;
}

// The sum of n parts (not negative; part(j), the same whenever it is asked
// for), the same bits in whatever order they lie: as integers in units of
// 2^-40 of the largest. NaN where one is NaN or infinite.
template <typename P, typename SH>
__device__ __forceinline__ float sum_in_any_order(int n, P &&part, SH &sh) {
    constexpr int THREADS = SH::kThreads;
    uint32_t most = 0;
    for (int j = threadIdx.x; j < n; j += THREADS) most = max(most, __builtin_bit_cast(uint32_t, part(j)) & 0x7fffffffu);
    most = block_max(most, sh);
    if (most >= 0x7f800000u) return NAN;
    const int up = 40 - (static_cast<int>(most >> 23) - 127);
    u64 q = 0;
    for (int j = threadIdx.x; j < n; j += THREADS) q += static_cast<u64>(ldexp(static_cast<double>(part(j)), up));
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
template <bool MOST, bool SUM, typename T, int THREADS, typename Begin, typename Sum, typename SH>
__device__ __forceinline__ int collect(const Row<T, THREADS> &row, int k, SH &sh, float &bound, float &total, float &extra,
                       Begin &&begin, Sum &&sum) {
    using R = Row<T, THREADS>;
    constexpr int N = R::N;
    const int slabs = row.slabs(), n = row.n, tid = threadIdx.x;
    words4 w[kSlab];
    row.load(0, w);
    if (tid == 0) sh.count = 0;
    uint32_t most_key = 0;
    if constexpr (MOST) {
#pragma unroll
        for (int u = 0; u < kSlab; ++u)
            if (R::at(0, u) < n) most_key = max(most_key, logit_key(piece_most<T>(w[u])));
        most_key = block_max(most_key, sh);
    }
    const bool few = (min(n, R::kSlabLogits) + N - 1) / N < k;  // pieces: then the row is one slab, bounded logit by logit
    bound = key_logit(bound_of(
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

    auto raise = [&](int aside) {
        const float next = key_logit(bound_of(
            k,
            [&](auto &&f) {
                for (int j = tid; j < aside; j += THREADS) f(place_key(sh.list[j]));
            },
            sh));
        if (!(next < bound)) bound = next;
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
    };
    // the values of a piece put aside
    auto read_again = [&](u64 entry, float (&y)[N]) {
        const int at = static_cast<int>(static_cast<uint32_t>(entry)) * N;
        const words4 p = load_piece_to(row.x, at, n);
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<T>(p, i);
        return at;
    };
    // what is left in the list after the pieces put aside: their parts of the sum
    auto add_parts = [&](int aside) {
        __syncthreads();
        if constexpr (SUM)
            extra += sum_in_any_order(
                aside,
                [&](int j) {
                    const uint32_t bits = static_cast<uint32_t>(sh.list[j]);
                    return __builtin_bit_cast(float, bits);
                },
                sh);
    };
    // the spare list becomes the list
    auto take_spare = [&](int count) {
        __syncthreads();
        for (int j = tid; j < count; j += THREADS) sh.list[j] = sh.spare[j];
        __syncthreads();
    };

    __syncthreads();
    for (int slab = 0; slab < slabs; ++slab) {
        // each piece's registers take the next slab's as soon as it is done
        const bool more = slab + 1 < slabs, whole = row.full(slab + 1);
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
                // here and now: left to itself, the compiler moves the sums after
                // the last piece, with all the slab's values in registers
                asm volatile("" : "+v"(total));
            }
            if (more) w[u] = row.load_one(slab + 1, u, whole);
        }
        if (more) {
            row.load_end(slab + 1, w);
            __syncthreads();
            const int aside = sh.count;
            if (aside > kList<THREADS>) return -1;
            __syncthreads();
            if (aside > kList<THREADS> / 2) {
                raise(aside);
                for (int j = tid; j < aside; j += THREADS) {
                    const u64 entry = sh.list[j];
                    float part = 0.f;
                    if (!(key_logit(place_key(entry)) < bound)) {
                        const int slot = atomicAdd(&sh.count, 1);
                        if (slot < kSpare<THREADS>) sh.spare[slot] = entry;
                    } else if constexpr (SUM) {
                        float y[N];
                        read_again(entry, y);
                        part = sum(y);
                    }
                    sh.list[j] = __builtin_bit_cast(uint32_t, part);
                }
                __syncthreads();
                const int kept = sh.count;
                if (kept > kSpare<THREADS>) return -1;
                // the sum's scratch is not the spare list's
                add_parts(aside);
                take_spare(kept);
            }
        }
    }
    __syncthreads();
    const int aside = sh.count;
    if (aside > kList<THREADS>) return -1;
    if (!few && aside > k) {
        raise(aside);
    } else {
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
    }
    for (int j = tid; j < aside; j += THREADS) {
        float y[N];
        const int at = read_again(sh.list[j], y);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (!(y[i] < bound) && at + i < n) {
                const int slot = atomicAdd(&sh.count, 1);
                if (slot < kSpare<THREADS>) sh.spare[slot] = place(logit_key(y[i]), at + i);
                y[i] = -INFINITY;
            }
        }
        if constexpr (SUM) sh.list[j] = __builtin_bit_cast(uint32_t, sum(y));
    }
    add_parts(aside);
    const int count = sh.count;
    if (count > kSpare<THREADS>) return -1;
    take_spare(count);
    return count;
}

struct TopKernelArgs {
    const void *x;
    int64_t stride, first_row;
    int vocab, k;
    float temperature;
    void *values;
    int64_t *indices;
    float *log_rest;
};

// The row is read once, and the k entries once more (they are in the caches):
// a row of 4096 x 131072 bf16, k = 64, costs its exponentials and comparisons
// as much as its bytes: 215 us for 1.07 GB (5 TB/s) with the vector units 76 %
// busy, where a reading rate of 6.7 TB/s would take 160. Of few rows, the chain
// of the bound, the list and its sorting is left: 8 rows take 10 us of 1024
// logits, 12 of 16384 and 15 of 65536. Exponentials are taken around the bound, known before
// the stream begins, so no running maximum is carried: one product and
// addition, one power of two and one addition a logit.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void top_logits_kernel(TopKernelArgs a) {
    constexpr int N = Row<T, THREADS>::N;
    __shared__ Shared<THREADS, false> sh;
    const int tid = threadIdx.x;
    const int64_t r = a.first_row + blockIdx.x;
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
        sort_list(a.k, sh, row.kKeyStep, row.index_bits());
    } else {
        sort_list(n, sh, row.kKeyStep, row.index_bits());
        for (int j = a.k + tid; j < n; j += THREADS) rest.join(ExpSum::of(key_logit(place_key(sh.list[j]))), c);
    }
    for (int j = tid; j < a.k; j += THREADS) {
        const int i = place_index(sh.list[j], row.n);
        a.indices[r * a.k + j] = i;
        static_cast<T *>(a.values)[r * a.k + j] = row.x[i];
    }
    sum = wave_total(sum);
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
        // infinite logits, but not beside a NaN
        a.log_rest[r] = rest.m == INFINITY && rest.s == rest.s ? INFINITY : rest.m / a.temperature + logf(rest.s);
    }
}

struct SampleKernelArgs {
    const void *x;
    int64_t stride, first_row;
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
    // 1 for the largest, an infinite one too
    __device__ __forceinline__ float of(float x) const { return x == m ? 1.f : fast_exp2((x - m) * inverse); }
    __device__ __forceinline__ u64 fixed(float x) const { return whole(of(x)); }
    // the exponent, where the largest logit is finite
    __device__ __forceinline__ float exponent(float x) const { return (x - m) * inverse; }
    // floor(2^40 e): exact products with powers of two, so the two halves are
    static __device__ __forceinline__ u64 whole(float e) {
        const float high = truncf(e * 256.f);
        const uint32_t low = static_cast<uint32_t>(fmaf(e, kFixed, high * -4294967296.f));
        return static_cast<u64>(static_cast<uint32_t>(high)) << 32 | low;
    }
    // the same as an f64: a thread's sum over a slab stays below 2^53, so it is exact
    static __device__ __forceinline__ double whole_f64(float e) { return static_cast<double>(truncf(e * kFixed)); }
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
template <typename T, int THREADS, typename SH>
__device__ __forceinline__ Drawn draw_by_search(const Row<T, THREADS> &row, const Weights &w, int top_k, float top_p, float min_p, float u,
                                SH &sh) {
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

// Draws among the first n of the sorted list, which are all that top_k leaves
// (but for logits without weight). The first wave has the list's sums.
template <typename SH>
__device__ __forceinline__ Drawn draw_from_list(int n, const Weights &w, float top_p, float min_p, float u, int vocab, SH &sh) {
    constexpr int THREADS = SH::kThreads;
    const int tid = threadIdx.x;
    if (tid < kWave) {
        const int per = (n + kWave - 1) / kWave, from = tid * per, to = min(n, from + per);
        u64 own = 0;
        for (int j = from; j < to; ++j) own += w.fixed(key_logit(place_key(sh.list[j])));
        const u64 upto = wave_scan(own), total = last_lane(upto);
        const u64 limit = top_p < 1.f ? limit_of(top_p, total) : ~0ull;
        u64 before = upto - own, sum = 0;
        uint32_t kept = 0;
        for (int j = from; j < to; ++j) {
            const float e = w.of(key_logit(place_key(sh.list[j])));
            const u64 f = Weights::whole(e);
            if (before < limit && e >= min_p) {
                ++kept;
                sum += f;
            }
            before += f;
        }
        // the kept logits are the first ones of the list
        sum = last_lane(wave_scan(sum));
        kept = last_lane(wave_scan(kept));
        if (tid == 0) {
            sh.pick[0] = sum;
            sh.pick[1] = kept;
        }
    }
    __syncthreads();
    Drawn d;
    d.sum = sh.pick[0];
    const int kept = static_cast<int>(sh.pick[1]);
    if (kept == 1) {
        d.token = place_index(sh.list[0], vocab);
        d.weight = d.sum;
        return d;
    }
    // by index: halves swapped, the larger complement of the index is first
    for (int i = tid; i < kept; i += THREADS) sh.list[i] = sh.list[i] << 32 | sh.list[i] >> 32;
    sort_list(kept, sh, 0, 32);
    if (tid < kWave) {
        const u64 target = target_of(u, d.sum);
        const int per = (kept + kWave - 1) / kWave, from = tid * per, to = min(kept, from + per);
        u64 own = 0;
        for (int j = from; j < to; ++j) own += w.fixed(key_logit(static_cast<uint32_t>(sh.list[j])));
        u64 before = wave_scan(own) - own;
        if (before <= target && target < before + own) {
            int j = from;
            u64 f = w.fixed(key_logit(static_cast<uint32_t>(sh.list[j])));
            while (j + 1 < to && target >= before + f) {
                before += f;
                f = w.fixed(key_logit(static_cast<uint32_t>(sh.list[++j])));
            }
            sh.pick[1] = f;
            sh.pick[2] = sh.list[j] >> 32;
        }
    }
    __syncthreads();
    d.weight = sh.pick[1];
    d.token = place_index(sh.pick[2], vocab);
    return d;
}

// The bin of an exponent y <= 0, as a number to compare whole ones with:
// monotone in the logit, 0 for the largest, below kMassBins for a weight that
// is not 0.
__device__ __forceinline__ float mass_bin(float y) { return y * (-kMassBins / 41.f); }

// Draws from all logits of which mass(value, index) is not 0, given its sum
// over every chunk.
template <typename T, int THREADS, typename M, typename SH>
__device__ __forceinline__ Drawn draw_from_chunks(const Row<T, THREADS> &row, const u64 *chunks, float u, M &&mass, SH &sh) {
    using R = Row<T, THREADS>;
    constexpr int kEach = R::kChunk / THREADS;
    const int tid = threadIdx.x;
    if (tid < kWave) {
        const int n = (row.n + R::kChunk - 1) / R::kChunk, per = (n + kWave - 1) / kWave;
        const int from = tid * per, to = min(n, from + per);
        u64 own = 0;
        for (int c = from; c < to; ++c) own += chunks[c];
        const u64 upto = wave_scan(own), sum = last_lane(upto), target = target_of(u, sum);
        u64 before = upto - own;
        if (before <= target && target < upto) {
            int c = from;
            while (c + 1 < to && target >= before + chunks[c]) before += chunks[c++];
            sh.pick[0] = static_cast<u64>(c);
            sh.pick[1] = target - before;
        }
        if (tid == 0) sh.pick[2] = sum;
    }
    __syncthreads();
    Drawn d;
    d.sum = sh.pick[2];
    const u64 target = sh.pick[1];
    const int from = static_cast<int>(sh.pick[0]) * R::kChunk + tid * kEach;
    u64 own = 0, total;
    for (int i = 0; i < kEach; ++i)
        if (from + i < row.n) own += mass(static_cast<float>(row.x[from + i]), from + i);
    u64 before = block_scan(own, total, sh);
    if (before <= target && target < before + own) {
        int i = 0;
        u64 f = mass(static_cast<float>(row.x[from]), from);
        while (i + 1 < kEach && from + i + 1 < row.n && target >= before + f) {
            before += f;
            ++i;
            f = mass(static_cast<float>(row.x[from + i]), from + i);
        }
        sh.pick[0] = static_cast<u64>(from + i);
        sh.pick[1] = f;
    }
    __syncthreads();
    d.token = min(static_cast<int>(sh.pick[0]), row.n - 1);
    d.weight = sh.pick[1];
    return d;
}

// A row whose top_k fits the list is read once (collect) and drawn from the
// sorted list: 24 us for 256 rows of 131072 bf16 (2.8 TB/s; the chain after the
// stream is half of it). Any other row is read for its largest logit, and then
// from the caches: once without top_p (29 us), where each wave's share of a slab
// has its exact sum and the draw reads one such share again; with top_p (60 us)
// once for the mass by exponent and once for the sums up to the cut. There
// memory is done after 10 us and what bounds it are the additions to the
// histogram in LDS (19 us: neighbours in a wave often hit one bin and go one by
// one) and the second pass's exponentials and f64 sums (18 us). Holding the row
// in registers between the passes spills or leaves one workgroup a CU (78 us).
// The larger of the two ways a top_k can go: by the list up to a logit a thread,
// 41 us for 1024 of a row at its widest, 33 for 512, 24 for 50; by search 205.
// Five workgroups of 256 threads fit a CU (LDS, and registers if no more than
// 96): 8192 x 1024, top_p 0.9, 106 us, with four 125.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS == 256 ? 5 : 4) void sample_kernel(SampleKernelArgs a) {
    using R = Row<T, THREADS>;
    constexpr int N = R::N;
    __shared__ Shared<THREADS, true> sh;
    __shared__ u64 chunks[kMaxChunks];
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int64_t r = a.first_row + blockIdx.x;
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
        const int n = collect<true, false>(
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
            sort_list(n, sh, row.kKeyStep, row.index_bits());
            const u64 top = sh.list[0];
            const Weights w{key_logit(place_key(top)), inverse};
            if (place_key(top) == kKeyNan || place_key(top) == kKeyNegInf) return answer(-1, NAN);
            if (greedy) return answer(place_index(top, row.n), 0.f);
            if (w.m < INFINITY) return finish(draw_from_list(min(top_k, n), w, top_p, min_p, u, row.n, sh));
        }
    }

    // the largest logit
    float most = -INFINITY;
    for (int s = 0; s < slabs; ++s) {
        words4 p[kSlab];
        row.load(s, p);
#pragma unroll
        for (int k = 0; k < kSlab; ++k) most = nan_max(most, piece_most<T>(p[k]));
    }
    const uint32_t top = block_max(logit_key(most), sh);
    if (top == kKeyNan || top == kKeyNegInf) return answer(-1, NAN);
    if (greedy) return answer(find_by_index(row, 0, [&](float x, int) -> u64 { return logit_key(x) == top; }, sh), 0.f);
    const Weights w{key_logit(top), inverse};
    if (top_k > 0 || w.m == INFINITY) return finish(draw_by_search(row, w, top_k, top_p, min_p, u, sh));

    // The sum over a slab of what is kept, chunk by chunk; kept(exponent, weight)
    // says of what. Pieces below `least` hold nothing of it.
    auto sum_chunks = [&](float least, auto &&kept) {
        for (int s = 0; s < slabs; ++s) {
            double sum = 0.0;
            words4 p[kSlab];
            row.load(s, p);
#pragma unroll
            for (int k = 0; k < kSlab; ++k) {
                if (piece_most<T>(p[k]) < least) continue;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float y = w.exponent(piece_value<T>(p[k], i)), e = fast_exp2(y);
                    sum += Weights::whole_f64(kept(y, e, s, k, i, p[k]) ? e : 0.f);
                }
            }
            const u64 upto = wave_scan(static_cast<u64>(sum));
            if (lane == kWave - 1 && R::chunk(s) < kMaxChunks) chunks[R::chunk(s)] = upto;
        }
        __syncthreads();
    };
    if (!(top_p < 1.f)) {
        if (min_p > 0.f)
            sum_chunks(w.m - 41.f / inverse, [&](float, float e, int, int, int, const words4 &) { return e >= min_p; });
        else
            sum_chunks(w.m - 41.f / inverse, [](float, float, int, int, int, const words4 &) { return true; });
        return finish(draw_from_chunks(
            row, chunks, u,
            [&](float x, int) -> u64 {
                const float e = fast_exp2(w.exponent(x));
                return e >= min_p ? Weights::whole(e) : 0;
            },
            sh));
    }

    // the row's mass by exponent
    for (int b = tid; b < kMassBins; b += THREADS) sh.mass[b] = 0;
    __syncthreads();
    const float weightless = w.m - 41.f / inverse;
    for (int s = 0; s < slabs; ++s) {
        words4 p[kSlab];
        row.load(s, p);
#pragma unroll
        for (int k = 0; k < kSlab; ++k) {
            if (piece_most<T>(p[k]) < weightless) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float y = w.exponent(piece_value<T>(p[k], i));
                const u64 f = Weights::whole(fast_exp2(y));
                if (f) atomicAdd(&sh.mass[static_cast<int>(mass_bin(y))], f);
            }
        }
    }
    __syncthreads();
    constexpr int kOwnBins = kMassBins / THREADS;
    u64 own = 0, total;
#pragma unroll
    for (int j = 0; j < kOwnBins; ++j) own += sh.mass[tid * kOwnBins + j];
    u64 before = block_scan(own, total, sh);
    const u64 limit = limit_of(top_p, total);

    // the prefix ends in one of the bins: what is in the bins before is kept,
    // the bin's own logits are sorted
    for (int j = 0; j < kOwnBins; ++j) {
        const u64 in_bin = sh.mass[tid * kOwnBins + j];
        if (before < limit && limit <= before + in_bin) {
            sh.pick[0] = static_cast<u64>(tid * kOwnBins + j);
            sh.pick[1] = before;
        }
        before += in_bin;
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const float cut_bin = static_cast<float>(static_cast<int>(sh.pick[0]));
    const u64 above = sh.pick[1];
    // below this no logit is in the bins kept (a margin of two bins)
    sum_chunks(w.m - (cut_bin + 3.f) * (41.f / kMassBins) / inverse,
               [&](float y, float e, int s, int k, int i, const words4 &p) {
                   const float b = mass_bin(y);
                   if (b >= cut_bin && b < cut_bin + 1.f) {
                       const int slot = atomicAdd(&sh.count, 1);
                       if (slot < kList<THREADS>) sh.list[slot] = place(logit_key(piece_value<T>(p, i)), R::at(s, k) + i);
                   }
                   return b < cut_bin && e >= min_p;
               });
    const int n = sh.count;
    if (n > kList<THREADS>) return finish(draw_by_search(row, w, top_k, top_p, min_p, u, sh));
    sort_list(n, sh, row.kKeyStep, row.index_bits());
    const int per = (n + THREADS - 1) / THREADS, from = tid * per, to = min(n, from + per);
    own = 0;
    for (int j = from; j < to; ++j) own += w.fixed(key_logit(place_key(sh.list[j])));
    before = above + block_scan(own, total, sh);
    for (int j = from; j < to; ++j) {
        if (before < limit) {
            const u64 p = sh.list[j];
            const float e = w.of(key_logit(place_key(p)));
            const u64 f = Weights::whole(e);
            if (e >= min_p) atomicAdd(&chunks[min(place_index(p, row.n) / R::kChunk, kMaxChunks - 1)], f);
            before += f;
            if (before >= limit) sh.pick[0] = p;  // the last one kept
        }
    }
    __syncthreads();
    const u64 cut = sh.pick[0];
    __syncthreads();
    finish(draw_from_chunks(
        row, chunks, u,
        [&](float x, int i) -> u64 {
            const float e = fast_exp2(w.exponent(x));
            return place(logit_key(x), i) >= cut && e >= min_p ? Weights::whole(e) : 0;
        },
        sh));
}

// Threads for a row, at least a quarter of what the list holds for each of the
// k. Many rows take few threads, so that several workgroups fit a CU and one's
// reductions, chains of LDS round trips that no more threads shorten, hide
// behind another's stream; few rows take as many as shorten the stream.
constexpr int kManyRows = 512;
int threads_for_list(int k) { return k <= 64 ? 64 : k <= 256 ? 256 : k <= 512 ? 512 : 1024; }

// bf16, k = 32, us: 8192 x 1024 64 threads 50, 256 61, 512 161; 4096 x 4096 36,
// 40, 93; 1024 x 16384 30, 17, 28; 1024 x 131072 92, 56, 61; of 8 rows, 1024
// classes 14.1, 10.5, 11.2; 16384 23, 11.6, 12.0; 131072 77, 26.9, 20.1 and 20.8
// with 1024.
int top_threads(const LogitRows &x, int pieces, int k) {
    const int by_row = x.rows >= kManyRows ? (pieces <= 512 ? 64 : 256) : pieces <= 2048 ? 256 : 512;
    return max(by_row, threads_for_list(k));
}

// bf16, us, untruncated / top_p 0.9 / top_k 50: 4096 x 512 64 threads 61 / 98 /
// 54, 256 32 / 55 / 39, 512 54 / 90 / 76; 1024 x 32768 256 31 / 59 / 22, 512 28 /
// 56 / 32, 1024 39 / 84 / 53; of 8 rows, 1024 classes 256 9.0 / 15.6 / 10.3, 512
// 7.4 / 12.2 / 10.3, 1024 8.3 / 13.0 / 12.0; 32768 512 9.2 / 19.7 / 11.8, 1024
// 9.4 / 20.8 / 12.9; 65536 512 12.8 / 31.1 / 14.0, 1024 11.7 / 27.3 / 14.7.
// A top_k of each row's own is on the device and plans nothing: rows whose own
// is above the threads taken (256 at least) go by search.
int sample_threads(const LogitRows &x, int pieces, int top_k) {
    const int by_row = x.rows >= kManyRows ? (pieces <= 2048 || top_k > 0 ? 256 : 512) : pieces <= 4096 ? 512 : 1024;
    return max(by_row, threads_for_list(top_k));
}
static_assert(TROPNN_MAX_VOCAB / (kWave * kSlab * kPerLoad<float>) <= kMaxChunks, "chunks of the widest row");

template <typename F>
hipError_t with_threads(int threads, F &&f) {
    switch (threads) {
        case 256: return f(std::integral_constant<int, 256>{});
        case 512: return f(std::integral_constant<int, 512>{});
        default: return f(std::integral_constant<int, 1024>{});
    }
}

}  // namespace

size_t top_logits_workspace(const LogitRows &, int) { return 0; }

hipError_t launch_top_logits(const TopArgs &a, void *, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    TopKernelArgs k{a.x.p, a.x.stride, 0, a.x.vocab, a.k, a.temperature, a.values, a.indices, a.log_rest};
    return with_logit_type(a.x.dtype, [&](auto t) {
        using T = decltype(t);
        auto with = [&](auto threads) {
            constexpr int kThreads = decltype(threads)::value;
            return by_grids(a.x.rows, [&](int64_t first, uint32_t rows) {
                k.first_row = first;
                hipLaunchKernelGGL((top_logits_kernel<T, kThreads>), dim3(rows), dim3(kThreads), 0, stream, k);
            });
        };
        const int threads = top_threads(a.x, (a.x.vocab + kPerLoad<T> - 1) / kPerLoad<T>, a.k);
        return threads == 64 ? with(std::integral_constant<int, 64>{}) : with_threads(threads, with);
    });
}

size_t sample_workspace(const LogitRows &) { return 0; }

hipError_t launch_sample(const SampleArgs &a, void *, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    SampleKernelArgs k{a.x.p, a.x.stride, 0, a.x.vocab, a.uniforms, a.temperatures, a.top_ps, a.min_ps, a.top_ks,
                             a.temperature, a.top_p, a.min_p, a.top_k, a.tokens, a.log_probs};
    return with_logit_type(a.x.dtype, [&](auto t) {
        using T = decltype(t);
        const int pieces = (a.x.vocab + kPerLoad<T> - 1) / kPerLoad<T>, top_k = a.top_ks ? 0 : a.top_k;
        return with_threads(sample_threads(a.x, pieces, top_k), [&](auto threads) {
            constexpr int kThreads = decltype(threads)::value;
            return by_grids(a.x.rows, [&](int64_t first, uint32_t rows) {
                k.first_row = first;
                hipLaunchKernelGGL((sample_kernel<T, kThreads>), dim3(rows), dim3(kThreads), 0, stream, k);
            });
        });
    });
}

}  // namespace tropnn
