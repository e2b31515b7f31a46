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

struct DistillKernelArgs {
    const void *x;
    int64_t rows, stride, first_row;  // first_row: of the streaming kernel's grid
    int vocab, k, values_dtype;
    const void *values;
    const int64_t *indices;
    const float *log_rest, *weights;
    const float *norm;  // sum of the weights, or NULL: norm_value
    float norm_value;
    float temperature, scale;
    float *row_loss;
    void *grad;
    const float *factor;  // of the gradient, or NULL: 1
    bool holds;           // grad has the gradient for a factor of one
    int bitmap_words;

    // Nothing is left to do where a gradient that is there is multiplied by one.
    __device__ __forceinline__ bool done(float f) const { return holds && f == 1.f; }
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

// The smallest and largest sum, in units of 2^(c reference), that is taken as
// it is; others are taken again around their own largest term.
constexpr float kLeast = 0x1p-90f, kMost = 0x1p90f;

// A row's list, as one wave has it: the log-sums of the teacher's and of the
// student's logits in it, and how many entries.
struct ListSums {
    float teacher_m, teacher_s, listed_m, listed_s, entries;
};

// The wave's sums; every lane has one entry (at < 0: none).
__device__ __forceinline__ ListSums wave_list(const Entry &e, float c) {
    const bool there = e.at >= 0;
    ListSums t;
    t.teacher_m = wave_most_of(there ? e.v : -INFINITY);
    t.listed_m = wave_most_of(there ? e.y : -INFINITY);
    const float tm = t.teacher_m == -INFINITY ? 0.f : t.teacher_m, ym = t.listed_m == -INFINITY ? 0.f : t.listed_m;
    t.teacher_s = wave_total(there ? fast_exp2((e.v - tm) * c) : 0.f);
    t.listed_s = wave_total(there ? fast_exp2((e.y - ym) * c) : 0.f);
    t.entries = static_cast<float>(__builtin_popcountll(__ballot(there)));
    return t;
}

__device__ __forceinline__ ExpSum exp_sum(float m, float s) {
    ExpSum t;
    t.m = m;
    t.s = s;
    return t;
}

// What a row's loss and gradient need, the same in every thread.
struct RowTotals {
    float all_m, l;            // the student's log-sum
    float ref, l_ref;          // of the classes outside the list
    float teacher_m, l_teacher;
    float log_p0, log_q0;
    float scale;               // of a probability's difference in the gradient
    bool none;                 // the classes outside the list are all -inf, or there are none
    __device__ __forceinline__ float log_q(float y, float c) const { return fmaf(y - all_m, c, -l); }
    __device__ __forceinline__ float log_p(float v, float c) const { return fmaf(v - teacher_m, c, -l_teacher); }
};

template <typename T, int THREADS, bool REST, bool GRAD>
struct RowWork {
    static constexpr int N = kPerLoad<T>, kWaves = THREADS / kWave;
    const DistillKernelArgs &a;
    float c;
    int body, body_end;  // whole pieces, and where the logits after them begin

    __device__ __forceinline__ RowWork(const DistillKernelArgs &args)
        : a(args), c(kLog2e / args.temperature), body(args.vocab / N), body_end(args.vocab / N * N) {}

    __device__ __forceinline__ const T *x(int64_t row) const { return static_cast<const T *>(a.x) + row * a.stride; }
    __device__ __forceinline__ T *grad(int64_t row) const { return static_cast<T *>(a.grad) + row * a.vocab; }
    __device__ __forceinline__ float weight(int64_t row) const { return a.weights ? a.weights[row] : 1.f; }
    // the teacher's rest, as a logit
    __device__ __forceinline__ float rest(int64_t row) const { return REST ? a.log_rest[row] * a.temperature : -INFINITY; }

    // Piece first + tid; past the body's end its last one again.
    __device__ __forceinline__ words4 load(const T *row, int first, int tid) const {
        const uint32_t at = static_cast<uint32_t>(min(first + tid, body - 1)) * 16u;
        return load_piece(reinterpret_cast<const T *>(reinterpret_cast<const char *>(row) + at));
    }

    __device__ __forceinline__ Entry entry(int64_t row, int64_t at, float v) const {
        Entry e{-1, -INFINITY, -INFINITY};
        if (at >= 0) {
            e.v = v;
            if (at < a.vocab) {
                e.at = static_cast<int>(at);
                e.y = static_cast<float>(x(row)[at]);
            } else {
                e.at = a.vocab;
                e.v = e.y = NAN;  // no such class: the row's loss and gradient are NaN
            }
        }
        return e;
    }
    __device__ __forceinline__ int64_t entry_class(int64_t row, int j) const { return a.indices[row * a.k + j]; }
    __device__ __forceinline__ float entry_value(int64_t row, int j) const { return any_value(a.values, a.values_dtype, row * a.k + j); }
    __device__ __forceinline__ Entry entry(int64_t row, int j) const { return entry(row, entry_class(row, j), entry_value(row, j)); }

    // The list's classes in the bitmap, and the waves' sums of it.
    __device__ __forceinline__ void take_list(int64_t row, const Entry &first, uint32_t *bits, ListSums *lists, int tid) const {
        const int wave = tid / kWave;
        if (wave * kWave >= a.k) return;
        auto mark = [&](const Entry &e) {
            if (REST && e.at >= 0 && e.at < a.vocab) atomicOr(&bits[e.at >> 5], 1u << (e.at & 31));
        };
        mark(first);
        ListSums t = wave_list(first, c);
#pragma unroll 1
        for (int j = tid + THREADS; j - (tid & (kWave - 1)) < a.k; j += THREADS) {
            Entry e{-1, -INFINITY, -INFINITY};
            if (j < a.k) e = entry(row, j);
            mark(e);
            const ListSums o = wave_list(e, c);
            ExpSum teacher = exp_sum(t.teacher_m, t.teacher_s), listed = exp_sum(t.listed_m, t.listed_s);
            teacher.join(exp_sum(o.teacher_m, o.teacher_s), c);
            listed.join(exp_sum(o.listed_m, o.listed_s), c);
            t = ListSums{teacher.m, teacher.s, listed.m, listed.s, t.entries + o.entries};
        }
        if ((tid & (kWave - 1)) == 0) lists[wave] = t;
    }
    __device__ __forceinline__ int list_waves() const { return min(kWaves, (a.k + kWave - 1) / kWave); }
    __device__ __forceinline__ ListSums join_lists(const ListSums *lists) const {
        ListSums t = lists[0];
#pragma unroll 1
        for (int v = 1; v < list_waves(); ++v) {
            const ListSums o = lists[v];
            ExpSum teacher = exp_sum(t.teacher_m, t.teacher_s), listed = exp_sum(t.listed_m, t.listed_s);
            teacher.join(exp_sum(o.teacher_m, o.teacher_s), c);
            listed.join(exp_sum(o.listed_m, o.listed_s), c);
            t = ListSums{teacher.m, teacher.s, listed.m, listed.s, t.entries + o.entries};
        }
        return t;
    }

    // The values of piece first + tid, -inf in place of the listed ones.
    __device__ __forceinline__ void unlisted(const words4 &v, int first, const uint32_t *bits, int tid, float (&y)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<T>(v, i);
        if (REST) {
            // a byte has the bits of 8 / N pieces
            const uint8_t *bytes = reinterpret_cast<const uint8_t *>(bits) + first * N / 8;
            const uint32_t b = N == 8 ? bytes[tid] : bytes[tid >> 1] >> (tid & 1) * 4 & 15;
            if (b) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (b & (1u << i)) y[i] = -INFINITY;
            }
        }
    }
    __device__ __forceinline__ float unlisted_tail(float x_tail, const uint32_t *bits, int tid) const {
        const int at = body_end + tid;
        return REST && at < a.vocab && (bits[at >> 5] >> (at & 31) & 1) ? -INFINITY : x_tail;
    }
    // The terms of piece first + tid, in units of 2^offset.
    __device__ __forceinline__ void add(float &s, const words4 &v, int first, const uint32_t *bits, float offset, int tid) const {
        float y[N];
        unlisted(v, first, bits, tid, y);
        float part = fast_exp2(fmaf(y[0], c, -offset));
#pragma unroll
        for (int i = 1; i < N; ++i) part += fast_exp2(fmaf(y[i], c, -offset));
        s += first + tid < body ? part : 0.f;
        // piece by piece: no values of later ones in registers yet
        asm volatile("" : "+v"(s));
        __builtin_amdgcn_sched_barrier(0);
    }

    // From the workgroup's sum s around `reference` and the list's sums.
    __device__ __forceinline__ RowTotals totals(int64_t row, float s, float reference, const ListSums &list, float x_tail,
                                                const uint32_t *bits, float *scratch, float weight, float norm, float factor,
                                                int tid) const {
        ExpSum teacher = exp_sum(list.teacher_m, list.teacher_s);
        const float r = rest(row);
        if (REST) teacher.join(ExpSum::of(r), c);
        const float offset = reference * c;
        ExpSum u = exp_sum(reference, s * fast_exp2(-fmaf(reference, c, -offset)));  // the unit's rounding
        if (!(s > kLeast && s < kMost)) {
            // once more, around the largest term
            u = ExpSum::of(unlisted_tail(x_tail, bits, tid));
#pragma unroll 1
            for (int p = 0; p + tid < body; p += THREADS) {
                float y[N];
                unlisted(load(x(row), p, tid), p, bits, tid, y);
#pragma unroll 1
                for (int i = 0; i < N; ++i) u.join(ExpSum::of(y[i]), c);
            }
            u = wave_join(u, c);
            __syncthreads();
            if ((tid & (kWave - 1)) == 0) {
                scratch[2 * (tid / kWave)] = u.m;
                scratch[2 * (tid / kWave) + 1] = u.s;
            }
            __syncthreads();
            u = ExpSum{};
#pragma unroll 1
            for (int v = 0; v < kWaves; ++v) u.join(exp_sum(scratch[2 * v], scratch[2 * v + 1]), c);
        }
        ExpSum all = u;
        if (REST) all.join(exp_sum(list.listed_m, list.listed_s), c);
        RowTotals t;
        t.all_m = all.m;
        t.l = log2f(all.s);
        t.none = REST && u.m == -INFINITY && u.s == 0.f;
        t.ref = t.none ? 0.f : u.m;
        t.l_ref = t.none ? 0.f : REST ? log2f(u.s) : t.l;
        t.teacher_m = teacher.m;
        t.l_teacher = log2f(teacher.s);
        t.log_p0 = t.log_p(r, c);
        t.log_q0 = t.none ? -INFINITY : fmaf(t.ref - all.m, c, t.l_ref - t.l);
        t.scale = a.temperature * a.scale * weight / norm * factor;
        return t;
    }

    // This wave's part of the row's divergence, in units of ln 2.
    __device__ __forceinline__ float loss_part(int64_t row, const Entry &first, const RowTotals &t, int tid) const {
        float part = first.at >= 0 ? kl_term(t.log_p(first.v, c), t.log_q(first.y, c)) : 0.f;
#pragma unroll 1
        for (int j = tid + THREADS; j < a.k; j += THREADS) {
            const Entry e = entry(row, j);
            if (e.at >= 0) part += kl_term(t.log_p(e.v, c), t.log_q(e.y, c));
        }
        if (REST && tid == 0) part += kl_term(t.log_p0, t.log_q0);
        return wave_total(part);
    }
    __device__ __forceinline__ void store_loss(int64_t row, const float *parts, float weight) const {
        float sum = 0.f;
#pragma unroll 1
        for (int v = 0; v < list_waves(); ++v) sum += parts[v];
        a.row_loss[row] = weight * a.temperature * a.temperature * kLn2 * sum;
    }

    // Gradients of classes outside the list. `near`: the difference and the
    // product with c as one multiply-add from `from`. Below 2^8 it is a multiple
    // of 2^-16, so its rounding moves a gradient by 2^-17 of itself at most, far
    // below the rounding to 16 bits.
    struct Outer {
        float by, from, ref, l_ref, c;
        bool near;
        __device__ __forceinline__ float operator()(float y) const {
            return by * fast_exp2(near ? fmaf(y, c, from) : fmaf(y - ref, c, -l_ref));
        }
    };
    __device__ __forceinline__ Outer outer(const RowTotals &t) const {
        Outer o;
        o.by = t.none ? 0.f : REST ? t.scale * (fast_exp2(t.log_q0) - fast_exp2(t.log_p0)) : t.scale;
        o.ref = t.ref;
        o.l_ref = t.l_ref;
        o.c = c;
        o.from = fmaf(-t.ref, c, -t.l_ref);
        o.near = sizeof(T) == 2 && __builtin_amdgcn_readfirstlane(fabsf(o.from) < 256.f);
        return o;
    }
    __device__ __forceinline__ void store(T *to, int first, int tid, const words4 &v) const {
        const uint32_t at = static_cast<uint32_t>(first + tid) * 16u;
        if (first + tid < body) store_piece(reinterpret_cast<T *>(reinterpret_cast<char *>(to) + at), v);
    }
    __device__ __forceinline__ words4 gradient(const words4 &v, const Outer &o) const {
        float g[N];
        if (o.near) {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = o.by * fast_exp2(fmaf(piece_value<T>(v, i), c, o.from));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = o.by * fast_exp2(fmaf(piece_value<T>(v, i) - o.ref, c, -o.l_ref));
        }
        return make_piece<T>(g);
    }
    __device__ __forceinline__ void store_zeros(int64_t row, int tid) const {
        const words4 zero = {0, 0, 0, 0};
#pragma unroll 1
        for (int p = 0; p < body; p += THREADS) store(grad(row), p, tid, zero);
        if (body_end + tid < a.vocab) grad(row)[body_end + tid] = static_cast<T>(0.f);
    }
    __device__ __forceinline__ void store_listed(int64_t row, const Entry &first, const RowTotals &t, int tid) const {
        auto put = [&](const Entry &e) {
            if (e.at >= 0 && e.at < a.vocab)
                grad(row)[e.at] = static_cast<T>(t.scale * (fast_exp2(t.log_q(e.y, c)) - fast_exp2(t.log_p(e.v, c))));
        };
        put(first);
#pragma unroll 1
        for (int j = tid + THREADS; j < a.k; j += THREADS) put(entry(row, j));
    }
    __device__ __forceinline__ void clear(uint32_t *bits, int tid) const {
#pragma unroll 1
        for (int i = tid; i < (a.vocab + 31) / 32; i += THREADS) bits[i] = 0;
    }
    // The largest listed logit of the student, around which the row is summed:
    // a logit then costs one multiply-add, one power of two and one addition.
    __device__ __forceinline__ float reference(const ListSums &list) const { return fabsf(list.listed_m * c) < 1e30f ? list.listed_m : 0.f; }
};

template <int THREADS>
__device__ __forceinline__ float block_total(float s, float *sums, int tid) {
    s = wave_total(s);
    if ((tid & (kWave - 1)) == 0) sums[tid / kWave] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int v = 0; v < THREADS / kWave; ++v) s += sums[v];
    return s;
}

// Rows that fit a workgroup's registers, HOLD pieces a thread, with gradient:
// each is read once. A workgroup has the rows from its number on, a grid apart,
// and works on two at a time: as a piece's gradient is stored, the next row's
// piece takes its registers, and the next row's list has been looked up before,
// so that memory is idle only while a row's sums meet. The row has a whole
// piece. 4096 x 131072 bf16 (32 entries), one row a CU, 443 us for 2.1 GB moved
// (4.85 TB/s; a copy of that size 326 us): 7 of a row's 26 us pass between its
// last load and its first store, while waves reduce, the totals' logarithms
// follow and the list is marked. 2048 x 8192 f32 (134 MB) 28 us with the
// launches around it, 2048 x 32768 bf16 (268 MB) 65.
template <typename T, int THREADS, int HOLD, bool REST>
__global__ __launch_bounds__(THREADS) void distill_held_kernel(DistillKernelArgs args) {
    using W = RowWork<T, THREADS, REST, true>;
    constexpr int kWaves = W::kWaves;
    extern __shared__ uint32_t listed_bits[];  // REST: two bitmaps, bit i: class i is in the list
    __shared__ float sums[2][2 * kWaves], parts[kWaves];
    __shared__ ListSums lists[kWaves];
    const W k(args);
    const float factor = args.factor ? *args.factor : 1.f;
    if (args.done(factor)) return;
    const int words = REST ? args.bitmap_words : 0;
    const float norm = args.norm ? *args.norm : args.norm_value;
    const int64_t rows = args.rows, grid = gridDim.x;
    // the first of this workgroup's rows from `row` on that counts; those left
    // out get their zeros here
    auto counted = [&](int64_t row) {
        while (row < rows && k.weight(row) == 0.f) {
            k.store_zeros(row, threadIdx.x);
            if (threadIdx.x == 0) args.row_loss[row] = 0.f;
            row += grid;
        }
        return row;
    };
    int64_t row = counted(blockIdx.x);
    if (row >= rows) return;
    int64_t next = counted(row + grid);
    uint32_t *bits = listed_bits, *next_bits = listed_bits + words;

    words4 w[HOLD];
    Entry first{-1, 0.f, 0.f};
    int64_t next_class = -1;
    float next_value = 0.f;
    {
        const int tid = threadIdx.x;
#pragma unroll
        for (int u = 0; u < HOLD; ++u) w[u] = k.load(k.x(row), u * THREADS, tid);
        if (tid < args.k) {
            first = k.entry(row, tid);
            if (next < rows) {
                next_class = k.entry_class(next, tid);
                next_value = k.entry_value(next, tid);
            }
        }
        if (REST) k.clear(bits, tid);
        __syncthreads();
        k.take_list(row, first, bits, lists, tid);
        __syncthreads();
    }
    for (;;) {
        // nothing of the thread's places is kept from row to row: that would
        // take more registers than the pieces
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const bool has_tail = k.body_end + tid < args.vocab;
        const float x_tail = has_tail ? static_cast<float>(k.x(row)[k.body_end + tid]) : -INFINITY;
        const float weight = k.weight(row);
        const ListSums list = k.join_lists(lists);
        const float reference = k.reference(list), offset = reference * k.c;
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < HOLD; ++u)
            if (u * THREADS < k.body) k.add(s, w[u], u * THREADS, bits, offset, tid);
        s += fast_exp2(fmaf(k.unlisted_tail(x_tail, bits, tid), k.c, -offset));
        s = block_total<THREADS>(s, sums[0], tid);
        const bool dead = __builtin_amdgcn_readfirstlane(list.entries == 0.f);  // nothing to learn from this row
        const RowTotals t = k.totals(row, dead ? 1.f : s, reference, list, x_tail, bits, sums[1], weight, norm, factor, tid);
        if (tid / kWave < k.list_waves()) {
            const float part = k.loss_part(row, first, t, tid);
            if ((tid & (kWave - 1)) == 0) parts[tid / kWave] = dead ? 0.f : part;
        }
        const bool more = next < rows;
        const int64_t after = more ? counted(next + grid) : next;
        if (!more) next = row;
        // the next row's list, and the classes of the one after it
        Entry next_first{-1, 0.f, 0.f};
        if (tid < args.k) {
            next_first = k.entry(next, next_class, next_value);
            if (after < rows) {
                next_class = k.entry_class(after, tid);
                next_value = k.entry_value(after, tid);
            }
        }
        if (REST) k.clear(next_bits, tid);
        const typename W::Outer outer = k.outer(t);
        T *grad = k.grad(row);
        const uint32_t lanes = more ? ~0u : 0u;  // after the last row, all lanes read one piece
#pragma unroll
        for (int u = 0; u < HOLD; ++u) {
            if (u * THREADS < k.body) k.store(grad, u * THREADS, tid, dead ? words4{0, 0, 0, 0} : k.gradient(w[u], outer));
            w[u] = k.load(k.x(next), (u * THREADS) & lanes, tid & lanes);
            __builtin_amdgcn_sched_barrier(0);  // not all of the next loads at once, into registers of their own
        }
        if (has_tail) grad[k.body_end + tid] = static_cast<T>(dead ? 0.f : outer(x_tail));
        __syncthreads();  // the row's stores come before the listed classes'
        if (!dead) k.store_listed(row, first, t, tid);
        if (tid == 0) k.store_loss(row, parts, dead ? 0.f : weight);
        if (!more) return;
        k.take_list(next, next_first, next_bits, lists, tid);
        __syncthreads();
        row = next;
        next = after;
        first = next_first;
        uint32_t *const swap = bits;
        bits = next_bits;
        next_bits = swap;
    }
}

// Other rows, and rows whose loss alone is wanted: streamed, and once more for
// the gradient (from the caches: the rows in flight fit them). The loss alone
// is bound by memory where rows are many: 4 pieces a thread in flight, 2048 x
// 32768 f16 (134 MB) 23 us, 5.8 TB/s of the 6.7 that a read reaches.
template <typename T, int THREADS, bool REST, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_stream_kernel(DistillKernelArgs args) {
    using W = RowWork<T, THREADS, REST, GRAD>;
    constexpr int kWaves = W::kWaves, U = 4;
    extern __shared__ uint32_t listed_bits[];  // REST: bit i: class i is in the list
    __shared__ float sums[2][2 * kWaves], parts[kWaves];
    __shared__ ListSums lists[kWaves];
    const W k(args);
    const float factor = GRAD && args.factor ? *args.factor : 1.f;
    if (args.done(factor)) return;
    const int tid = threadIdx.x;
    const int64_t row = args.first_row + blockIdx.x;
    const float norm = args.norm ? *args.norm : args.norm_value, weight = k.weight(row);
    if (weight == 0.f) {
        if (GRAD) k.store_zeros(row, tid);
        if (tid == 0) args.row_loss[row] = 0.f;
        return;
    }
    words4 w[U];
    if (k.body > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = k.load(k.x(row), u * THREADS, tid);
    }
    const bool has_tail = k.body_end + tid < args.vocab;
    const float x_tail = has_tail ? static_cast<float>(k.x(row)[k.body_end + tid]) : -INFINITY;
    Entry first{-1, 0.f, 0.f};
    if (tid < args.k) first = k.entry(row, tid);
    if (REST) k.clear(listed_bits, tid);
    __syncthreads();
    k.take_list(row, first, listed_bits, lists, tid);
    __syncthreads();
    const ListSums list = k.join_lists(lists);
    const float reference = k.reference(list), offset = reference * k.c;
    float s = 0.f;
    for (int p = 0; p < k.body; p += U * THREADS) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u * THREADS < k.body) k.add(s, w[u], p + u * THREADS, listed_bits, offset, tid);
            w[u] = k.load(k.x(row), p + (U + u) * THREADS, tid);
        }
    }
    s += fast_exp2(fmaf(k.unlisted_tail(x_tail, listed_bits, tid), k.c, -offset));
    s = block_total<THREADS>(s, sums[0], tid);
    if (list.entries == 0.f) {  // no list: nothing to learn from this row
        if (GRAD) k.store_zeros(row, tid);
        if (tid == 0) args.row_loss[row] = 0.f;
        return;
    }
    const RowTotals t = k.totals(row, s, reference, list, x_tail, listed_bits, sums[1], weight, norm, factor, tid);
    if (tid / kWave < k.list_waves()) {
        const float part = k.loss_part(row, first, t, tid);
        if ((tid & (kWave - 1)) == 0) parts[tid / kWave] = part;
    }
    if (GRAD) {
        const typename W::Outer outer = k.outer(t);
        T *grad = k.grad(row);
        for (int p = 0; p < k.body; p += U * THREADS) {
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = k.load(k.x(row), p + u * THREADS, tid);
#pragma unroll
            for (int u = 0; u < U; ++u) k.store(grad, p + u * THREADS, tid, k.gradient(w[u], outer));
        }
        if (has_tail) grad[k.body_end + tid] = static_cast<T>(outer(x_tail));
    }
    __syncthreads();  // the row's stores come before the listed classes'
    if (GRAD) k.store_listed(row, first, t, tid);
    if (tid == 0) k.store_loss(row, parts, weight);
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

template <typename T, int THREADS, bool REST, bool GRAD>
hipError_t launch_stream(DistillKernelArgs k, hipStream_t stream) {
    const auto kernel = distill_stream_kernel<T, THREADS, REST, GRAD>;
    const int lds = REST ? k.bitmap_words * 4 : 0;
    if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void *>(kernel), lds); e != hipSuccess) return e;
    return by_grids(k.rows, [&](int64_t first, uint32_t rows) {
        k.first_row = first;
        hipLaunchKernelGGL(kernel, dim3(rows), dim3(THREADS), lds, stream, k);
    });
}

template <typename T, int THREADS, bool GRAD>
hipError_t launch_streamed(const DistillKernelArgs &k, hipStream_t stream) {
    return k.log_rest ? launch_stream<T, THREADS, true, GRAD>(k, stream) : launch_stream<T, THREADS, false, GRAD>(k, stream);
}

constexpr int kCus = 256;

template <typename T, int THREADS, int HOLD, bool REST>
hipError_t launch_hold(const DistillKernelArgs &k, int64_t grid, hipStream_t stream) {
    const auto kernel = distill_held_kernel<T, THREADS, HOLD, REST>;
    const int lds = REST ? 2 * k.bitmap_words * 4 : 0;
    if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void *>(kernel), lds); e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grid)), dim3(THREADS), lds, stream, k);
    return hipGetLastError();
}

// WGS workgroups of a CU share the rows.
template <typename T, int THREADS, int HOLD, int WGS>
hipError_t launch_held(const DistillKernelArgs &k, hipStream_t stream) {
    const int64_t grid = k.rows < kCus * WGS ? k.rows : kCus * WGS;
    return k.log_rest ? launch_hold<T, THREADS, HOLD, true>(k, grid, stream) : launch_hold<T, THREADS, HOLD, false>(k, grid, stream);
}

// The kernel for rows of `pieces` pieces. With gradient, the row is held
// wherever it fits (bf16, 32 entries: 8192 x 8192 58 us held, 71 streamed;
// 2048 x 32768 56 and 71; 1024 x 131072 126 and 142), by as few threads as
// keep it to eight pieces a thread while several workgroups share a CU:
// 8192 x 1024 f32 21 us with 64 threads, 29 with 256, 54 with 512; 8192 x 8192
// bf16 58 with 256, 61 with 64, 80 with 512; 2048 x 65536 bf16 115 with 512,
// 118 with 1024, 158 streamed by 256. For the loss alone, nothing is read
// twice, and small workgroups hide each other's reductions: 2048 x 32768 f16
// 23 us with 256 threads, 29 with 1024; few wide rows take more threads.
template <typename T>
hipError_t launch_by_width(const DistillKernelArgs &k, hipStream_t stream) {
    const int pieces = (k.vocab + kPerLoad<T> - 1) / kPerLoad<T>;
    if (k.grad) {
        if (k.vocab < kPerLoad<T>) return launch_streamed<T, 64, true>(k, stream);  // no whole piece to hold
        if (pieces <= 128) return launch_held<T, 64, 2, 16>(k, stream);
        if (pieces <= 256) return launch_held<T, 64, 4, 16>(k, stream);
        if (pieces <= 512) return launch_held<T, 64, 8, 16>(k, stream);
        if (pieces <= 1024) return launch_held<T, 256, 4, 6>(k, stream);
        if (pieces <= 2048) return launch_held<T, 256, 8, 6>(k, stream);
        if (pieces <= 4096) return launch_held<T, 512, 8, 2>(k, stream);
        if (pieces <= 8192) return launch_held<T, 512, 16, 2>(k, stream);
        if (pieces <= 16384) return launch_held<T, 1024, 16, 1>(k, stream);
        return launch_streamed<T, 1024, true>(k, stream);
    }
    if (pieces <= 256) return launch_streamed<T, 64, false>(k, stream);
    if (pieces <= 4096 || k.rows >= 4 * kCus) return launch_streamed<T, 256, false>(k, stream);
    return launch_streamed<T, 1024, false>(k, stream);
}

}  // namespace

// 16 bytes for the sum of the weights, then a loss per row.
size_t distill_workspace(const LogitRows &x, int, bool) { return 16 + sizeof(float) * static_cast<size_t>(x.rows); }

hipError_t launch_distill(const DistillArgs &a, void *workspace, hipStream_t stream) {
    float *norm = static_cast<float *>(workspace), *row_loss = norm + 4;
    const bool sum_weights = a.mean && a.weights;
    DistillKernelArgs k{a.x.p, a.x.rows, a.x.stride, 0, a.x.vocab, a.k, a.values_dtype, a.values, a.indices, a.log_rest, a.weights,
                        sum_weights ? norm : nullptr, a.mean ? static_cast<float>(a.x.rows) : 1.f, a.temperature,
                        a.scale, row_loss, a.grad, a.factor, a.holds, 0};
    if (sum_weights && !a.holds) {
        hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kSumThreads), 0, stream, a.weights, a.x.rows, 1.f,
                           static_cast<const float *>(nullptr), 1.f, norm);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (a.x.rows > 0) {
        k.bitmap_words = (a.x.vocab + 31) / 32 + 256;  // pieces past the row's end read bits, too
        hipError_t e = with_logit_type(a.x.dtype, [&](auto t) { return launch_by_width<decltype(t)>(k, stream); });
        if (e != hipSuccess) return e;
    }
    if (!a.loss) return hipSuccess;
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
