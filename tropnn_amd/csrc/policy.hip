// Log-probabilities of given tokens, their gradient, and the losses on them
// (include/tropnn_hip_train.h).
//
// With c = log2(e) / temperature and a the row's token, the other classes are summed
// in one pass, each thread around its largest logit so far: terms 2^(c x - o) with o
// the whole number next to c times that logit, so that the exponent is rounded where
// it is small, and a new largest logit scales the sum by a power of two. c is in two
// parts: its rounding would be in every term alike. With m the largest of the others,
// s their sum around it and d = (m - x_a) / temperature, the token's log-probability
// is -(d + log(s + e^-d)), or -log(1 + s e^d) where the token is the largest: full
// relative precision where it has nearly all of the mass. These few numbers of a row
// are f64, since a loss may be the small rest of large terms of both signs: 1.5e-8 of a
// log-probability at 131072 classes (3e-7 with all of it in f32, 1% faster), 3e-8 at
// ten, where a term's own exponential is the error and the worst of 100000 rows has
// 1.6e-7.
// A row's statistics (ref, l) give every class's probability as 2^(c (x_i - ref) - l),
// and the token's gradient 1 - p_a as 1 - 2^(...) by expm1. Sixteen terms are summed
// in f32, what they come to and sums over rows and tokens in f64.
#include "train.hpp"

namespace tropnn {
namespace {

// A sum of terms 2^(c x) around the largest x: s in units of 2^offset.
struct Mass {
    double s;
    float m, offset;

    static __device__ __forceinline__ Mass none() { return Mass{0.0, -INFINITY, -1e30f}; }
    static __device__ __forceinline__ float offset_of(float m, float c) { return fmaxf(rintf(m * c), -1e30f); }
    // s in units of 2^other, which is no less than 2^offset.
    __device__ __forceinline__ double in(float other) const {
        return __builtin_amdgcn_ldexp(s, static_cast<int>(fmaxf(offset - other, -300.f)));
    }
    __device__ __forceinline__ void join(const Mass &o) {
        const float most = fmaxf(offset, o.offset);
        s = in(most) + o.in(most);
        offset = most;
        m = fmaxf(m, o.m);
    }
    static __device__ __forceinline__ Mass of(float x, const Temper &by) {
        Mass t;
        t.m = x;
        t.offset = offset_of(x, by.c);
        t.s = static_cast<double>(fast_exp2(fmaf(x, by.rest, fmaf(x, by.c, -t.offset))));
        return t;
    }
};

// The sums between which a row's is taken as it is; others (no mass, or logits of 1e30
// and more) are taken again.
constexpr double kLeastMass = 0x1p-100, kMostMass = 0x1p100;

// Functions of f64 numbers to about 2^-24, by the f32 ones and what their argument
// lost. All threads of a row compute them, between its loads and its stores: with the
// f64 ones 32768 x 4096 f32 take 104 us, with these 87.
__device__ __forceinline__ float lost(double x, float h) { return static_cast<float>(x - static_cast<double>(h)); }
__device__ __forceinline__ double exp_of(double x) {
    x = x > 2000.0 ? 2000.0 : x < -2000.0 ? -2000.0 : x;  // inf and 0; a NaN stays
    x *= 1.44269504088896340736;
    const double k = rint(x);
    return __builtin_amdgcn_ldexp(static_cast<double>(fast_exp2(static_cast<float>(x - k))), static_cast<int>(k));
}
__device__ __forceinline__ double expm1_of(double x) {
    if (x > 1.0) return exp_of(x) - 1.0;
    if (x < -100.0) return -1.0;
    const float h = static_cast<float>(x);
    const double e = static_cast<double>(expm1f(h));
    return e + (1.0 + e) * static_cast<double>(lost(x, h));
}
// Of a normal f32's size: the exponent apart, and a logarithm of at most log(2) / 2.
__device__ __forceinline__ double log_of(double x) {
    const float h = static_cast<float>(x);
    const int k = (static_cast<int>(__builtin_bit_cast(uint32_t, h)) - 0x3f3504f3) >> 23;
    return static_cast<double>(k) * 0.693147180559945309417 +
           static_cast<double>(logf(__builtin_amdgcn_ldexpf(h, -k)) + lost(x, h) * __builtin_amdgcn_rcpf(h));
}
// log(1 + x), x from 0 to 1/2.
__device__ __forceinline__ double log1p_of(double x) {
    const float h = static_cast<float>(1.0 + x);
    return static_cast<double>(logf(h) + static_cast<float>(x - static_cast<double>(h - 1.f)) * __builtin_amdgcn_rcpf(h));
}

// A piece's load and store; NT: non-temporal, for what exceeds the caches anyway.
template <bool NT, typename T>
__device__ __forceinline__ words4 load_piece(const T *p) {
    if constexpr (!NT)
        return tropnn::load_piece(p);
    else if constexpr (sizeof(T) == 2)
        return __builtin_nontemporal_load(reinterpret_cast<const words4_at2 *>(p));
    else
        return __builtin_nontemporal_load(reinterpret_cast<const words4_at4 *>(p));
}
template <bool NT, typename T>
__device__ __forceinline__ void store_piece(T *p, words4 w) {
    if constexpr (!NT)
        tropnn::store_piece(p, w);
    else if constexpr (sizeof(T) == 2)
        __builtin_nontemporal_store(w, reinterpret_cast<words4_at2 *>(p));
    else
        __builtin_nontemporal_store(w, reinterpret_cast<words4_at4 *>(p));
}

// A row, as pieces of 16 bytes and a few loose logits around them. Where a row of
// 16-bit logits starts off a 4-byte boundary (every other row of an odd
// vocabulary), its first logit is loose: loads across such boundaries take a
// fourth longer (4096 x 100001 f16 185 us, 141 with the pieces at a boundary).
template <typename T, int THREADS>
struct TokenRow {
    static constexpr int N = kPerLoad<T>, kWaves = THREADS / kWave;
    const T *x;
    int vocab, head, body, body_end;  // loose logits before the pieces, pieces, and where the logits after them begin
    int token, token_piece;           // vocab or more: no such class; the piece that the token is in, or none's number
    Temper temper;
    float c;

    __device__ __forceinline__ TokenRow(const LogitRows &rows, int64_t row, int64_t t, const Temper &by)
        : x(static_cast<const T *>(rows.p) + row * rows.stride), vocab(rows.vocab),
          head(sizeof(T) == 2 ? static_cast<int>(reinterpret_cast<uintptr_t>(x) >> 1 & 1) : 0), body((vocab - head) / N),
          body_end(head + body * N), token(t < rows.vocab ? static_cast<int>(t) : rows.vocab),
          token_piece(token < head ? -1 : (token - head) / N), temper(by), c(by.c) {}

    // Piece p's first logit.
    __device__ __forceinline__ int at(int p) const { return head + p * N; }
    // Piece p; past the body's end its last one again.
    template <bool NT = false>
    __device__ __forceinline__ words4 load(int p) const {
        return load_piece<NT>(x + static_cast<uint32_t>(at(min(p, body - 1))));
    }
    // The loose logit that the thread has, -1: none.
    __device__ __forceinline__ int loose(int tid) const {
        const int after = vocab - body_end;
        return tid < after ? body_end + tid : tid < after + head ? 0 : -1;
    }
    // f(i) in the place of logit i of piece p where that is the token.
    template <typename F>
    __device__ __forceinline__ void at_token(float (&y)[N], int p, F &&f) const {
        if (p != token_piece) return;
        const float v = f();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i == (token - head) % N) y[i] = v;
    }
    // The values of piece p, -inf in place of the token's.
    __device__ __forceinline__ void others(const words4 &v, int p, float (&y)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<T>(v, i);
        at_token(y, p, [] { return -INFINITY; });
    }
    // The thread's loose logit, -inf: none or the token's.
    __device__ __forceinline__ float loose_other(int tid) const {
        const int i = loose(tid);
        return i >= 0 && i != token ? static_cast<float>(x[i]) : -INFINITY;
    }
    __device__ __forceinline__ float logit() const { return token < vocab ? static_cast<float>(x[token]) : NAN; }
    // Adds K pieces.
    template <int K>
    __device__ __forceinline__ void add(Mass &t, const words4 (&v)[K], const int (&p)[K]) const {
        float y[K][N], most = t.m;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            others(v[k], p[k], y[k]);
            float piece = y[k][0];
#pragma unroll
            for (int i = 1; i < N; ++i) piece = fmaxf(piece, y[k][i]);
            most = p[k] < body ? fmaxf(most, piece) : most;
        }
        const float offset = Mass::offset_of(most, c);
        float part[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < N; ++i) y[k][i] = fast_exp2(fmaf(y[k][i], temper.rest, fmaf(y[k][i], c, -offset)));
#pragma unroll
            for (int n = N / 2; n > 0; n >>= 1)  // in pairs: as few roundings as can be
                for (int i = 0; i < n; ++i) y[k][i] += y[k][i + n];
            part[k] = p[k] < body ? y[k][0] : 0.f;
        }
#pragma unroll
        for (int n = K / 2; n > 0; n >>= 1)
            for (int i = 0; i < n; ++i) part[i] += part[i + n];
        t.s = t.in(offset) + static_cast<double>(part[0]);
        t.m = most;
        t.offset = offset;
    }
};

// The pieces that are added at a time: sixteen values.
template <typename T, int PIECES>
constexpr int kAtATime = PIECES * kPerLoad<T> <= 16 ? PIECES : 16 / kPerLoad<T>;

__device__ __forceinline__ double wave_total(double v) {
    auto step = [&](unsigned long long o) { v += __builtin_bit_cast(double, o); };
    auto bits = [&] { return __builtin_bit_cast(unsigned long long, v); };
    step(dpp_from<0x111, 0xF>(bits()));
    step(dpp_from<0x112, 0xF>(bits()));
    step(dpp_from<0x114, 0xF>(bits()));
    step(dpp_from<0x118, 0xF>(bits()));
    step(dpp_from<0x142, 0xA>(bits()));
    step(dpp_from<0x143, 0xC>(bits()));
    const unsigned long long u = bits();
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(u), kWave - 1);
    const uint32_t high = __builtin_amdgcn_readlane(static_cast<uint32_t>(u >> 32), kWave - 1);
    return __builtin_bit_cast(double, static_cast<unsigned long long>(high) << 32 | low);
}

__device__ __forceinline__ Mass wave_mass(const Mass &mine, float c) {
    Mass t;
    t.m = wave_most_of(mine.m);
    t.offset = Mass::offset_of(t.m, c);
    t.s = wave_total(mine.in(t.offset));
    return t;
}

// A workgroup's mass, in every thread.
template <int THREADS>
__device__ __forceinline__ Mass workgroup_mass(const Mass &mine, float c, Mass *scratch, int tid) {
    Mass t = wave_mass(mine, c);
    if constexpr (THREADS == kWave) return t;
    if ((tid & (kWave - 1)) == 0) scratch[tid / kWave] = t;
    __syncthreads();
    if constexpr (THREADS > 4 * kWave) {  // by lanes: the waves' masses in every thread are registers that a row is held in
        t = Mass::none();
        if ((tid & (kWave - 1)) < THREADS / kWave) t = scratch[tid & (kWave - 1)];
        return wave_mass(t, c);
    }
    t = scratch[0];
#pragma unroll
    for (int v = 1; v < THREADS / kWave; ++v) t.join(scratch[v]);
    return t;
}

// A row's statistics and its token's log-probability.
struct Score {
    float ref, l;
    double log_prob;
};

// From the mass of the other classes and the token's logit. The mass is the same in
// all threads of the workgroup, and all of them call.
template <typename T, int THREADS>
__device__ __forceinline__ Score score_of(const TokenRow<T, THREADS> &r, const Mass &others, float x_a, float2 *scratch, int tid) {
    constexpr double kLn2d = 0.693147180559945309417, kLog2ed = 1.44269504088896340736;
    float m = others.m;
    double s = others.s;
    double unit = static_cast<double>(others.offset) * kLn2d - static_cast<double>(m) * r.temper.inverse;  // s's, over e^(m / temperature)
    if (!(s > kLeastMass && s < kMostMass)) {
        // once more, with differences from the largest before the product with c
        ExpSum u = ExpSum::of(r.loose_other(tid));
#pragma unroll 1
        for (int p = tid; p < r.body; p += THREADS) {
            float y[TokenRow<T, THREADS>::N];
            r.others(r.load(p), p, y);
#pragma unroll 1
            for (int i = 0; i < TokenRow<T, THREADS>::N; ++i) u.join(ExpSum::of(y[i]), r.c);
        }
        u = wave_join(u, r.c);
        __syncthreads();
        if ((tid & (kWave - 1)) == 0) scratch[tid / kWave] = make_float2(u.m, u.s);
        __syncthreads();
        u = ExpSum{};
#pragma unroll 1
        for (int v = 0; v < THREADS / kWave; ++v) {
            ExpSum o;
            o.m = scratch[v].x;
            o.s = scratch[v].y;
            u.join(o, r.c);
        }
        m = u.m;
        s = u.m == INFINITY ? static_cast<double>(NAN) : static_cast<double>(u.s);
        unit = 0.0;
    }
    const double d = (static_cast<double>(m) - static_cast<double>(x_a)) * r.temper.inverse;
    const double over = d < 0.0 ? s * exp_of(unit + d) : s == 0.0 ? d : static_cast<double>(INFINITY);  // the others' mass over the token's
    Score t;
    if (over <= 0.5) {
        t.ref = x_a;
        t.log_prob = x_a == INFINITY ? static_cast<double>(NAN) : -log1p_of(over);
        t.l = static_cast<float>(-t.log_prob * kLog2ed);
    } else {
        const double l = unit + log_of(s + exp_of(-(unit + d)));
        t.ref = m;
        t.log_prob = -(d + l);
        t.l = static_cast<float>(l * kLog2ed);
    }
    if (t.log_prob != t.log_prob) t.l = NAN;
    return t;
}

// A row's loss and the loss's derivative by its log-probability.
struct PolicyRow {
    double loss, by;
};
__device__ __forceinline__ PolicyRow policy_row(const PolicyTerms &a, int64_t row, double log_prob) {
    const double advantage = static_cast<double>(a.advantages[row]);
    const double ratio = exp_of(log_prob - static_cast<double>(a.old_log_probs[row]));
    const double free = ratio * advantage;
    const double bounded = fmin(fmax(ratio, a.low), a.high) * advantage;
    const bool bound = free > bounded;  // a NaN stays
    PolicyRow t;
    t.loss = bound ? -bounded : -free;
    t.by = bound ? 0.0 : -free;
    if (a.ref_log_probs) {
        const double d = static_cast<double>(a.ref_log_probs[row]) - log_prob, e = expm1_of(d);
        t.loss += a.kl_weight * (e - d);
        t.by -= a.kl_weight * e;
    }
    return t;
}

// What a mean divides by, the sum of the weights, as a number from 1/2 to 1 and a
// power of two. What it divides is divided by the power in f64, before f32 holds it:
// the one coefficient of a mean over many rows may be past f32 where its share of
// the mean is not, and so may the sum be.
struct Norm {
    double sum;
    int power;  // 0 where the sum is 0 or not finite

    __device__ __forceinline__ explicit Norm(double by) : sum(by), power(__builtin_amdgcn_frexp_exp(by)) {}
    __device__ __forceinline__ float of(double v) const { return static_cast<float>(__builtin_amdgcn_ldexp(v, -power)); }
    __device__ __forceinline__ float fraction() const { return of(sum); }
};

struct ScoreKernelArgs {
    ScoreArgs s;
    int64_t first_row;
    PolicyTerms terms;  // old_log_probs NULL: the log-probabilities alone
    double *row_loss, *row_by;  // weighted, and the scale's product with the latter
};

__device__ __forceinline__ void store_log_prob(const ScoreArgs &a, int64_t row, double log_prob) {
    if (a.log_probs) a.log_probs[row] = static_cast<float>(log_prob);
    if (a.log_probs_f64) a.log_probs_f64[row] = log_prob;
}

// A row per workgroup, streamed, U pieces a thread in flight. Bound by memory:
// 4096 x 131072 bf16 (1.07 GB) 159 us past the caches, 6.8 TB/s; 8192 x 32768 bf16 82;
// a wave per row at 8192 x 512 f32 7.1 us.
template <typename T, int THREADS, int U, bool NT>
__global__ __launch_bounds__(THREADS) void token_score_kernel(ScoreKernelArgs a) {
    using R = TokenRow<T, THREADS>;
    __shared__ Mass masses[R::kWaves];
    __shared__ float2 scratch[R::kWaves];
    const int tid = threadIdx.x;
    const int64_t row = a.first_row + blockIdx.x;
    const int64_t token = a.s.tokens[row];
    const float weight = a.terms.weights ? a.terms.weights[row] : 1.f;
    if (token < 0 || weight == 0.f) {
        // no part of a loss; a weighted row's log-probability is still wanted
        if (tid == 0 && a.row_loss) {
            a.row_loss[row] = 0.0;
            a.row_by[row] = 0.0;
        }
        if (token < 0) {
            if (tid == 0) store_log_prob(a.s, row, 0.0);
            return;
        }
    }
    const R r(a.s.x, row, token, a.s.temper);
    words4 w[U];
    if (r.body > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = r.template load<NT>(u * THREADS + tid);
    }
    const float x_loose = r.loose_other(tid), x_a = r.logit();
    constexpr int K = kAtATime<T, U>;
    Mass mine = Mass::none();
    for (int p = tid; p - tid < r.body; p += U * THREADS) {
#pragma unroll
        for (int u = 0; u < U; u += K) {
            words4 v[K];
            int at[K];
#pragma unroll
            for (int i = 0; i < K; ++i) {
                v[i] = w[u + i];
                at[i] = p + (u + i) * THREADS;
            }
            r.add(mine, v, at);
#pragma unroll
            for (int i = 0; i < K; ++i) w[u + i] = r.template load<NT>(p + (U + u + i) * THREADS);
        }
    }
    mine.join(Mass::of(x_loose, r.temper));
    const Mass all = workgroup_mass<THREADS>(mine, r.c, masses, tid);
    const Score t = score_of<T, THREADS>(r, all, x_a, scratch, tid);
    if (tid != 0) return;
    store_log_prob(a.s, row, t.log_prob);
    if (a.s.stats) a.s.stats[row] = make_float2(t.ref, t.l);
    if (a.row_loss && weight != 0.f) {
        const PolicyRow p = policy_row(a.terms, row, t.log_prob);
        a.row_loss[row] = static_cast<double>(weight) * p.loss;
        a.row_by[row] = static_cast<double>(weight) * a.terms.scale * p.by;
    }
}

struct GradKernelArgs {
    TokenGradArgs g;
    int64_t runs;     // of all rows
    uint32_t chunks;  // runs of a row
};

// A run of U * THREADS pieces of a row: every class's product of the coefficient
// with its probability, and the token's with what is left of one.
template <typename T, int THREADS, int U, bool NT>
__device__ __forceinline__ void gradient_run(const GradKernelArgs &a, int64_t row, uint32_t chunk, float factor, int tid) {
    using R = TokenRow<T, THREADS>;
    constexpr int N = R::N;
    const int64_t token = a.g.tokens[row];
    const float norm = a.g.norm ? *a.g.norm : 1.f;
    const float coef = a.g.coefs[row / a.g.rows_per_coef];
    const R r(a.g.x, row, token, a.g.temper);
    T *grad = static_cast<T *>(a.g.grad) + row * r.vocab;
    const int first = static_cast<int>(chunk) * THREADS * U + tid;
    const int loose = chunk == a.chunks - 1 ? r.loose(tid) : -1;
    if (token < 0 || coef == 0.f || factor == 0.f) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = first + u * THREADS;
            if (p < r.body) store_piece<NT>(grad + r.at(p), words4{0, 0, 0, 0});
        }
        if (loose >= 0) grad[loose] = static_cast<T>(0.f);
        return;
    }
    words4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (first + u * THREADS < r.body) w[u] = r.template load<NT>(first + u * THREADS);
    const float2 stats = a.g.stats[row];
    const float by = coef / norm * factor / a.g.temper.t;
    auto gradient = [&](float y) { return -by * fast_exp2(fmaf(y - stats.x, r.c, -stats.y)); };
    auto of_token = [&] { return -by * expm1f(fmaf(r.logit() - stats.x, r.c, -stats.y) * kLn2); };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int p = first + u * THREADS;
        float g[N];
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = gradient(piece_value<T>(w[u], i));
        r.at_token(g, p, of_token);
        if (p < r.body) store_piece<NT>(grad + r.at(p), make_piece<T>(g));
    }
    if (loose >= 0) grad[loose] = static_cast<T>(loose == r.token ? of_token() : gradient(static_cast<float>(r.x[loose])));
}

// The logits' gradient, a run per workgroup at a time. It moves what a copy moves,
// as fast: 4096 x 131072 bf16 (2.1 GB) 347 us, 6.2 TB/s where a copy of this shape
// reaches 6.3. Short runs, all loads before all stores and both past the caches make
// that up: a whole row per workgroup has 5.1 TB/s, runs of 1024 pieces with ordinary
// accesses 5.8.
template <typename T, int THREADS, int U, bool NT>
__global__ __launch_bounds__(THREADS) void token_gradient_kernel(GradKernelArgs a) {
    const float factor = a.g.factor ? *a.g.factor : 1.f;
    if (a.g.holds && factor == 1.f) return;
    for (int64_t run = blockIdx.x; run < a.runs; run += gridDim.x) {
        const int64_t row = run / a.chunks;
        gradient_run<T, THREADS, U, NT>(a, row, static_cast<uint32_t>(run - row * a.chunks), factor, threadIdx.x);
    }
}

// A sum over rows: of their losses and of their weights.
struct RowSums {
    double loss, weight;
};

struct HeldArgs {
    ScoreArgs s;
    int64_t first_row;
    PolicyTerms terms;
    const RowSums *parts;  // of the weights, whose sum divides the loss; NULL: 1 does
    int n_parts;
    double *row_loss;
    float *coefs;
    void *grad;
};

// What the gradient of a row goes by, the same in every thread.
struct RowGrad {
    float ref, l, by, at_token;
};

// Rows that fit a workgroup's registers, HOLD pieces a thread: read once for the
// loss and the gradient together. A row per workgroup, dealt by the hardware as
// others end, so that rows without a token, which take a fraction of the time, hold
// nobody up; workgroups that keep going from row to row, with the next row's pieces
// on their way, were no faster (4096 x 131072 bf16 417 us against 419) and slower
// on narrow rows (32768 x 4096 f32 268 against 198). It takes 423 us, 5.1 TB/s with
// the launches around it: a copy in runs of a row's 256 KB has 5.5, and one row fills
// a CU, so that its memory idles while the row's sums meet. Two workgroups a CU, with
// a part of the row in LDS, were 3% faster; pieces in an order rotated by the row not.
template <typename T, int THREADS, int HOLD, bool NT>
__global__ __launch_bounds__(THREADS) void policy_held_kernel(HeldArgs a) {
    using R = TokenRow<T, THREADS>;
    constexpr int N = R::N;
    __shared__ Mass masses[R::kWaves];
    __shared__ float2 scratch[R::kWaves];
    __shared__ RowGrad shared_grad;
    const int tid = threadIdx.x;
    const int64_t row = a.first_row + blockIdx.x, token = a.s.tokens[row];
    const R r(a.s.x, row, token, a.s.temper);
    T *const grad = static_cast<T *>(a.grad) + row * r.vocab;
    const int loose = r.loose(tid);
    if (token < 0) {
        for (int p = tid; p < r.body; p += THREADS) store_piece<NT>(grad + r.at(p), words4{0, 0, 0, 0});
        if (loose >= 0) grad[loose] = static_cast<T>(0.f);
        if (tid == 0) {
            store_log_prob(a.s, row, 0.0);
            a.row_loss[row] = 0.0;
            a.coefs[row] = 0.f;
            a.s.stats[row] = make_float2(0.f, 0.f);
        }
        return;
    }
    words4 w[HOLD];
#pragma unroll
    for (int u = 0; u < HOLD; ++u) w[u] = r.template load<NT>(u * THREADS + tid);
    const float x_loose = loose >= 0 ? static_cast<float>(r.x[loose]) : -INFINITY;
    const float x_a = r.logit();
    const float weight = a.terms.weights ? a.terms.weights[row] : 1.f;
    double norm = 1.0;
    if (a.parts && tid < kWave) norm = wave_add(tid < a.n_parts ? a.parts[tid].weight : 0.0);
    constexpr int K = kAtATime<T, HOLD>;
    Mass mine = Mass::none();
#pragma unroll
    for (int u = 0; u < HOLD; u += K) {
        if (u * THREADS < r.body) {
            words4 v[K];
            int at[K];
#pragma unroll
            for (int i = 0; i < K; ++i) {
                v[i] = w[u + i];
                at[i] = (u + i) * THREADS + tid;
            }
            r.add(mine, v, at);
        }
        asm volatile("" : "+v"(mine.s));
        __builtin_amdgcn_sched_barrier(0);  // no values of later pieces in registers yet
    }
    mine.join(Mass::of(loose == r.token ? -INFINITY : x_loose, r.temper));
    const Mass all = workgroup_mass<THREADS>(mine, r.c, masses, tid);
    const Score t = score_of<T, THREADS>(r, all, x_a, scratch, tid);
    if (tid < kWave) {
        RowGrad g;
        g.ref = t.ref;
        g.l = t.l;
        PolicyRow p{0.0, 0.0};
        if (weight != 0.f) p = policy_row(a.terms, row, t.log_prob);
        const Norm by(norm);
        const float coef = by.of(static_cast<double>(weight) * a.terms.scale * p.by);
        g.by = coef == 0.f ? 0.f : coef / by.fraction() / a.s.temper.t;
        g.at_token = g.by == 0.f ? 0.f : -g.by * expm1f(fmaf(x_a - t.ref, r.c, -t.l) * kLn2);  // the row may hold anything
        if (tid == 0) {
            store_log_prob(a.s, row, t.log_prob);
            a.s.stats[row] = make_float2(t.ref, t.l);
            a.row_loss[row] = static_cast<double>(weight) * p.loss;
            a.coefs[row] = coef;
            shared_grad = g;
        }
    }
    __syncthreads();
    const RowGrad g = shared_grad;
    const bool zero = g.by == 0.f;
    auto gradient = [&](float y) { return zero ? 0.f : -g.by * fast_exp2(fmaf(y - g.ref, r.c, -g.l)); };
#pragma unroll
    for (int u = 0; u < HOLD; ++u) {
        const int p = u * THREADS + tid;
        if (u * THREADS >= r.body) break;
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = gradient(piece_value<T>(w[u], i));
        r.at_token(v, p, [&] { return g.at_token; });
        if (p < r.body) store_piece<NT>(grad + r.at(p), make_piece<T>(v));
    }
    if (loose >= 0) grad[loose] = static_cast<T>(loose == r.token ? g.at_token : gradient(x_loose));
}

constexpr int kSumThreads = 1024;

// A workgroup's sums, in the lanes of its first wave.
__device__ __forceinline__ RowSums workgroup_sums(RowSums s, RowSums *scratch) {
    const int tid = threadIdx.x, waves = static_cast<int>(blockDim.x) / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        s.loss += __shfl_xor(s.loss, d, kWave);
        s.weight += __shfl_xor(s.weight, d, kWave);
    }
    if ((tid & (kWave - 1)) == 0) scratch[tid / kWave] = s;
    __syncthreads();
    if (tid >= kWave) return s;
    s = tid < waves ? scratch[tid] : RowSums{0.0, 0.0};
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        s.loss += __shfl_xor(s.loss, d, kWave);
        s.weight += __shfl_xor(s.weight, d, kWave);
    }
    return s;
}

struct TotalArgs {
    const double *row_loss;  // or NULL: the weights alone
    const int64_t *tokens;  // or NULL: all rows count
    const float *weights;   // or NULL: ones
    int64_t rows;
    double scale;
    bool mean;
    RowSums *parts;
    float *loss, *norm;  // loss NULL: the parts alone
    const double *by;    // what the mean divides beside the loss, and
    float *coefs;        // where it goes; n_coefs 0: nothing
    int64_t n_coefs;
};

__device__ __forceinline__ Norm norm_of(const TotalArgs &a, const RowSums &s) { return Norm(a.mean ? s.weight : 1.0); }

__device__ __forceinline__ void store_total(const TotalArgs &a, const RowSums &s) {
    const Norm norm = norm_of(a, s);
    *a.norm = norm.fraction();
    *a.loss = static_cast<float>(a.scale * s.loss / norm.sum);
}

// Coefficients of one workgroup, eight of a thread in flight: loaded before the norm
// is known, stored after that.
struct Coefs {
    static constexpr int U = 8;
    double by[U];

    __device__ __forceinline__ void load(const TotalArgs &a, int64_t first) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = first + u * kSumThreads + threadIdx.x;
            by[u] = i < a.n_coefs ? a.by[i] : 0.0;
        }
    }
    __device__ __forceinline__ void store(const TotalArgs &a, const Norm &norm, int64_t first) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = first + u * kSumThreads + threadIdx.x;
            if (i < a.n_coefs) a.coefs[i] = norm.of(by[u]);
        }
    }
};
constexpr int64_t kSumRows = int64_t{Coefs::U} * kSumThreads;

// Sums over a run of rows per workgroup, in a fixed order; one workgroup of all
// rows finishes the loss and the coefficients. Eight loads of each array are in
// flight: one workgroup takes 8192 rows in a round trip to memory.
__global__ __launch_bounds__(kSumThreads) void total_kernel(TotalArgs a) {
    __shared__ RowSums scratch[kSumThreads / kWave];
    constexpr int U = 8;
    const int64_t each = ((a.rows + gridDim.x - 1) / gridDim.x + kSumThreads - 1) / kSumThreads * kSumThreads;
    const int64_t end = min(each * (blockIdx.x + 1), a.rows);
    const bool alone = a.loss && gridDim.x == 1;
    Coefs coefs;
    if (alone) coefs.load(a, 0);
    RowSums sum{0.0, 0.0};
    for (int64_t first = each * blockIdx.x; first < end; first += U * kSumThreads) {
        int64_t token[U];
        double loss[U];
        float weight[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = first + u * kSumThreads + threadIdx.x;
            const bool in = i < end;
            token[u] = in ? (a.tokens ? a.tokens[i] : 0) : -1;
            loss[u] = in && a.row_loss ? a.row_loss[i] : 0.0;
            weight[u] = in && a.weights ? a.weights[i] : 1.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            sum.loss += loss[u];
            sum.weight += token[u] >= 0 ? static_cast<double>(weight[u]) : 0.0;
        }
    }
    sum = workgroup_sums(sum, scratch);
    if (threadIdx.x == 0) a.parts[blockIdx.x] = sum;
    if (!alone) return;
    if (threadIdx.x == 0) store_total(a, sum);
    if (a.n_coefs == 0) return;
    __shared__ double weight;
    if (threadIdx.x == 0) weight = sum.weight;
    __syncthreads();
    const Norm norm = norm_of(a, RowSums{0.0, weight});
    coefs.store(a, norm, 0);
    for (int64_t first = kSumRows; first < a.n_coefs; first += kSumRows) {
        coefs.load(a, first);
        coefs.store(a, norm, first);
    }
}

// The loss from several workgroups' sums, which every wave adds up for itself, and
// the coefficients, a run of them per workgroup at a time.
__global__ __launch_bounds__(kSumThreads) void join_kernel(TotalArgs a, int parts) {
    Coefs coefs;
    int64_t first = blockIdx.x * kSumRows;
    coefs.load(a, first);
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    RowSums s = lane < parts ? a.parts[lane] : RowSums{0.0, 0.0};
    s.loss = wave_add(s.loss);
    s.weight = wave_add(s.weight);
    if (blockIdx.x == 0 && threadIdx.x == 0) store_total(a, s);
    const Norm norm = norm_of(a, s);
    while (first < a.n_coefs) {
        coefs.store(a, norm, first);
        first += gridDim.x * kSumRows;
        coefs.load(a, first);
    }
}

constexpr int kPairThreads = 256;

// A pair of sequences per workgroup.
__global__ __launch_bounds__(kPairThreads) void preference_kernel(PreferenceArgs a, int64_t first_pair, double *pair_loss,
                                                                  double *pair_by) {
    __shared__ RowSums scratch[2][kPairThreads / kWave];
    const int64_t pair = first_pair + blockIdx.x;
    RowSums part[2] = {{0.0, 0.0}, {0.0, 0.0}};  // of log-probabilities, and how many
    for (int64_t i = threadIdx.x; i < a.length; i += kPairThreads) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int64_t at = (side * a.pairs + pair) * a.length + i;
            const bool there = a.tokens[at] >= 0;
            const double log_prob = a.token_log_probs[at];
            part[side].loss += there ? log_prob : 0.0;
            part[side].weight += there ? 1.0 : 0.0;
        }
    }
    double sum[2], count[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        part[side] = workgroup_sums(part[side], scratch[side]);
        sum[side] = part[side].loss;
        count[side] = part[side].weight;
    }
    if (threadIdx.x != 0) return;
    double share[2];
    for (int side = 0; side < 2; ++side) {
        share[side] = a.average ? 1.0 / fmax(count[side], 1.0) : 1.0;
        sum[side] *= share[side];
        a.log_probs[side * a.pairs + pair] = static_cast<float>(sum[side]);
    }
    const double weight = a.weights ? static_cast<double>(a.weights[pair]) : 1.0;
    double loss = 0.0, by = 0.0;
    if (weight != 0.0) {
        double off = sum[0] - sum[1];
        if (a.reference) off -= static_cast<double>(a.reference[pair]) - static_cast<double>(a.reference[a.pairs + pair]);
        const double h = a.beta * off - a.margin;
        const double smoothing = a.smoothing;
        // -log sigmoid(h) = log(1 + e^-|h|) + max(0, -h)
        const double e = exp(-fabs(h)), soft = log1p(e);
        const double yes = soft + fmax(-h, 0.0), no = soft + fmax(h, 0.0);
        loss = h != h ? h : (smoothing == 1.0 ? 0.0 : (1.0 - smoothing) * yes) + (smoothing == 0.0 ? 0.0 : smoothing * no);
        const double sigmoid_minus_one = h >= 0.0 ? -e / (1.0 + e) : -1.0 / (1.0 + e);
        by = a.beta * (sigmoid_minus_one + smoothing);
    }
    pair_loss[pair] = weight * loss;
    pair_by[pair] = weight * by * share[0] * a.scale;
    pair_by[a.pairs + pair] = -weight * by * share[1] * a.scale;
}

template <typename T, int THREADS, int U, bool NT = false>
hipError_t launch_score(ScoreKernelArgs k, hipStream_t stream) {
    return by_grids(k.s.x.rows, [&](int64_t first, uint32_t rows) {
        k.first_row = first;
        hipLaunchKernelGGL((token_score_kernel<T, THREADS, U, NT>), dim3(rows), dim3(THREADS), 0, stream, k);
    });
}

// Bytes of logits from which on they and their gradient go past the caches: the
// two together are then more than the last of them holds.
constexpr int64_t kStreamBytes = int64_t{128} << 20;
int64_t bytes_of(const LogitRows &x) { return x.rows * x.vocab * (x.dtype == TROPNN_LOGITS_F32 ? 4 : 2); }
bool streams(const LogitRows &x) { return bytes_of(x) >= kStreamBytes; }

constexpr int64_t kCus = 256;

// As many pieces in flight as a row has, and no more threads than that keeps busy:
// 8192 x 4096 bf16 (512 pieces) 15 us with 64 threads, 23 with 256; with many rows a
// wave each meets no other wave (2048 x 9000 bf16 10.0 and 12.8, 32768 x 8192 bf16 93
// and 107, 65536 x 2500 f32 109 and 152), until the rows leave the caches and are
// wide enough to be bound by memory (16384 x 16384 bf16 95 and 85, 32768 x 4096 f32
// 91 and 87; in the caches 1024 x 32768 bf16 14.2 with both, 45.6 and 41.9 with its
// gradient). Few wide rows take more threads: 64 x 131072 bf16 11.7 us with 1024,
// 14.5 with 256. Past the caches where no backward will read the row again (8192 x
// 32768 bf16 83 us, 94 through them), or where it will find none of it there (with its
// gradient 4096 x 131072 bf16 500 and 527, 1280 x 65536 f32, 336 MB, 163 and 192, but
// 4096 x 32768 bf16, 268 MB, 131 and 125, and narrow 32768 x 4096 f32 260 and 253).
template <typename T>
hipError_t launch_scores_by_width(const ScoreKernelArgs &k, hipStream_t stream) {
    const LogitRows &x = k.s.x;
    const int pieces = (x.vocab + kPerLoad<T> - 1) / kPerLoad<T>;
    if (pieces <= 128) return launch_score<T, 64, 2>(k, stream);
    if (pieces <= 512) return launch_score<T, 64, 4>(k, stream);
    if (x.rows >= 4 * kCus && pieces <= (!streams(x) ? 2048 : sizeof(T) == 2 ? 1408 : 768)) return launch_score<T, 64, 4>(k, stream);
    if (streams(x) && (!k.s.stats || (pieces > 1024 && bytes_of(x) > 2 * kStreamBytes))) return launch_score<T, 256, 4, true>(k, stream);
    if (pieces <= 4096 || x.rows >= kCus) return launch_score<T, 256, 4>(k, stream);
    return launch_score<T, 1024, 4>(k, stream);
}

hipError_t launch_scores(const ScoreKernelArgs &k, hipStream_t stream) {
    return with_logit_type(k.s.x.dtype, [&](auto t) { return launch_scores_by_width<decltype(t)>(k, stream); });
}

// As many workgroups as runs; fewer where there may be nothing to do, which the
// 131072 of 4096 x 131072 bf16 take 30 us to find and 8192 of them 3.8 (and 370 for
// the gradient where there is, against 343).
template <typename T, int THREADS, int U, bool NT>
hipError_t launch_gradient(GradKernelArgs k, hipStream_t stream) {
    const int body = k.g.x.vocab / kPerLoad<T>;
    k.chunks = body > 0 ? static_cast<uint32_t>((body + THREADS * U - 1) / (THREADS * U)) : 1u;
    k.runs = k.g.x.rows * k.chunks;
    const int64_t most = k.g.holds ? 32 * kCus : int64_t{1} << 21;
    hipLaunchKernelGGL((token_gradient_kernel<T, THREADS, U, NT>), dim3(static_cast<uint32_t>(k.runs < most ? k.runs : most)),
                       dim3(THREADS), 0, stream, k);
    return hipGetLastError();
}

// One workgroup up to two round trips of rows, then one for each, at most a wave's
// lanes. 16000 rows take one workgroup 13.6 us, two and the launch that joins them
// 9.7, but a launch costs the host 3 (a call with its gradient 64 to 67 us and
// 67.5); 65536 take eight and a join 10.8, one 41.
int sum_parts(int64_t rows) {
    return static_cast<int>(rows <= 2 * kSumRows ? 1 : std::min<int64_t>((rows + kSumRows - 1) / kSumRows, kWave));
}

hipError_t launch_total(const TotalArgs &a, hipStream_t stream) {
    const int parts = sum_parts(a.rows);
    hipLaunchKernelGGL(total_kernel, dim3(static_cast<uint32_t>(parts)), dim3(kSumThreads), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (parts == 1 || !a.loss) return hipSuccess;
    const int64_t runs = std::min<int64_t>((a.n_coefs + kSumRows - 1) / kSumRows, 4 * kCus);
    hipLaunchKernelGGL(join_kernel, dim3(static_cast<uint32_t>(std::max<int64_t>(runs, 1))), dim3(runs > 0 ? kSumThreads : kWave), 0,
                       stream, a, parts);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_token_log_probs(const ScoreArgs &a, hipStream_t stream) {
    return launch_scores(ScoreKernelArgs{a, 0, PolicyTerms{}, nullptr, nullptr}, stream);
}

hipError_t launch_token_gradient(const TokenGradArgs &a, hipStream_t stream) {
    if (a.x.rows == 0) return hipSuccess;
    const GradKernelArgs k{a, 0, 1};
    return with_logit_type(a.x.dtype, [&](auto t) {
        using T = decltype(t);
        const int pieces = (a.x.vocab + kPerLoad<T> - 1) / kPerLoad<T>;
        if (pieces <= 128) return launch_gradient<T, 64, 2, false>(k, stream);
        return streams(a.x) ? launch_gradient<T, 256, 2, true>(k, stream) : launch_gradient<T, 256, 2, false>(k, stream);
    });
}

namespace {

template <typename T, int THREADS, int HOLD>
hipError_t launch_held(HeldArgs k, hipStream_t stream) {
    return by_grids(k.s.x.rows, [&](int64_t first, uint32_t rows) {
        k.first_row = first;
        if (streams(k.s.x))
            hipLaunchKernelGGL((policy_held_kernel<T, THREADS, HOLD, true>), dim3(rows), dim3(THREADS), 0, stream, k);
        else
            hipLaunchKernelGGL((policy_held_kernel<T, THREADS, HOLD, false>), dim3(rows), dim3(THREADS), 0, stream, k);
    });
}

// As few threads as keep it to eight pieces a thread while several workgroups share
// a CU: 32768 x 4096 f32 202 us with 256 threads, 207 with 128, 216 with 512; 8192 x
// 32768 bf16 195 with 512, 210 with 256, 216 with 1024. Sixteen a thread before a row
// fills a CU: 1000 x 50001 f16 60 us with 512 threads, 67 with 1024, 4096 of them 173
// and 208, 4096 x 65536 bf16 203 and 223 (4096 x 32768 f32, two thirds with a token,
// 168 and 164).
template <typename T>
hipError_t launch_held_by_width(const HeldArgs &k, hipStream_t stream) {
    const int pieces = (k.s.x.vocab + kPerLoad<T> - 1) / kPerLoad<T>;
    if (pieces <= 128) return launch_held<T, 64, 2>(k, stream);
    if (pieces <= 256) return launch_held<T, 64, 4>(k, stream);
    if (pieces <= 512) return launch_held<T, 64, 8>(k, stream);
    if (pieces <= 1024) return launch_held<T, 256, 4>(k, stream);
    if (pieces <= 2048) return launch_held<T, 256, 8>(k, stream);
    if (pieces <= 4096) return launch_held<T, 512, 8>(k, stream);
    if (pieces <= 8192) return launch_held<T, 512, 16>(k, stream);
    return launch_held<T, 1024, 16>(k, stream);
}

}  // namespace

// Where a workgroup holds a row and there are enough of them: reading it once then
// gains more than the launch that finds the norm beforehand costs (2048 x 4096 f32
// 22.6 us, 26.5 read twice; 8192 x 4096 56 and 74; 4096 x 131072 bf16 423 and 507),
// which it does not for few or little rows (64 x 131072 bf16 26.7 and 20.5; 2048 x
// 512 f32 12.7 and 12.2).
bool policy_grad_fits(const LogitRows &x) {
    const int per_load = x.dtype == TROPNN_LOGITS_F32 ? 4 : 8;
    return x.rows >= kCus && x.vocab >= 2 * per_load && (x.vocab + per_load - 1) / per_load <= 16384 && bytes_of(x) >= (int64_t{32} << 20);
}

namespace {

// A loss per row or pair, the sums' parts, and what becomes coefficients.
struct Losses {
    size_t parts, by, bytes;  // where they begin, and the end

    Losses(int64_t n, int64_t coefs)
        : parts((sizeof(double) * static_cast<size_t>(n) + 15) / 16 * 16),
          by(parts + sizeof(RowSums) * static_cast<size_t>(sum_parts(n))), bytes(by + sizeof(double) * static_cast<size_t>(coefs)) {}
};

}  // namespace

// A forward that writes the gradient knows the norm before its coefficients.
size_t policy_workspace(const LogitRows &x, bool want_grad) { return Losses(x.rows, want_grad ? 0 : x.rows).bytes; }

hipError_t launch_policy(const PolicyArgs &a, void *workspace, hipStream_t stream) {
    const LogitRows &x = a.score.x;
    const Losses at(x.rows, a.grad ? 0 : x.rows);
    char *const ws = static_cast<char *>(workspace);
    double *const row_loss = reinterpret_cast<double *>(ws), *const row_by = reinterpret_cast<double *>(ws + at.by);
    RowSums *const parts = reinterpret_cast<RowSums *>(ws + at.parts);
    TotalArgs t{nullptr, a.score.tokens, a.terms.weights, x.rows, a.terms.scale, a.mean, parts, nullptr, a.norm,
                row_by, a.coefs, a.grad ? 0 : x.rows};
    if (a.grad && x.rows > 0) {
        if (a.mean) {
            if (hipError_t e = launch_total(t, stream); e != hipSuccess) return e;
        }
        const HeldArgs k{a.score, 0, a.terms, a.mean ? parts : nullptr, sum_parts(x.rows), row_loss, a.coefs, a.grad};
        hipError_t e = with_logit_type(x.dtype, [&](auto t) { return launch_held_by_width<decltype(t)>(k, stream); });
        if (e != hipSuccess) return e;
    } else if (x.rows > 0) {
        if (hipError_t e = launch_scores(ScoreKernelArgs{a.score, 0, a.terms, row_loss, row_by}, stream); e != hipSuccess) return e;
    }
    t.row_loss = row_loss;
    t.loss = a.loss;
    return launch_total(t, stream);
}

size_t preference_workspace(int64_t pairs, int64_t) { return Losses(pairs, 2 * pairs).bytes; }

hipError_t launch_preference(const PreferenceArgs &a, void *workspace, hipStream_t stream) {
    const Losses at(a.pairs, 2 * a.pairs);
    char *const ws = static_cast<char *>(workspace);
    double *const pair_loss = reinterpret_cast<double *>(ws), *const pair_by = reinterpret_cast<double *>(ws + at.by);
    hipError_t e = by_grids(a.pairs, [&](int64_t first, uint32_t pairs) {
        hipLaunchKernelGGL(preference_kernel, dim3(pairs), dim3(kPairThreads), 0, stream, a, first, pair_loss, pair_by);
    });
    if (e != hipSuccess) return e;
    return launch_total(TotalArgs{pair_loss, nullptr, a.weights, a.pairs, a.scale, a.mean, reinterpret_cast<RowSums *>(ws + at.parts),
                                  a.loss, a.norm, pair_by, a.coefs, 2 * a.pairs},
                        stream);
}

}  // namespace tropnn
