// kd_drafts.hip - a draft model beside its target: verification of drafted tokens against the target's probabilities,
// and the distillation loss against the target's top logits with its gradient.
#include <algorithm>
#include <type_traits>

#include "kd_internal.h"

namespace kd {

namespace {

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) v += __shfl_xor(v, m);
    return v;
}

// 16 bytes of a row whose start is aligned to its elements only.
template <typename T> struct Piece {
    static constexpr int kCount = 16 / sizeof(T);
    T x[kCount];
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(4)));
// Past: the load takes no place in the caches.
template <bool Past = false, typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int64_t at, int64_t cols, T rest) {
    Piece<T> p;
    if (at + Piece<T>::kCount <= cols) {
        if constexpr (Past) {
            const u32x4 raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + at));
            __builtin_memcpy(&p, &raw, 16);
        } else {
            __builtin_memcpy(&p, row + at, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::kCount; ++i) p.x[i] = at + i < cols ? row[at + i] : rest;
    }
    return p;
}

// ---- verification ---------------------------------------------------------------------------------
//
// One workgroup a sequence: it finds the first draft that is not accepted, reads that one row (the target's and the draft's)
// and draws from it. Bound by the rows' bytes for many sequences (256 x 7 drafts of 50257 in f32: 20.9 us, 103 MB at 4.9 TB/s),
// by the chain of dependent loads and the rate of a CU for few. The draw narrows the row down in two steps, a sixteenth of it
// and a sixteenth of that by the waves' sums, and a wave's running sums find the entry: two passes over parts that are in the
// L2 by then instead of running sums over the whole row.

constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWaves = kVerifyThreads / 64;

// The weights that a token is drawn from: p - q where that is positive, p itself without a draft row; NaN stays NaN.
template <typename T> struct Weights {
    const T* p;
    const T* q;       // NULL: no draft row
    int64_t certain;  // q NULL: the entry whose q is 1, or -1
    static constexpr int kCount = Piece<T>::kCount;

    // the weight of entry `entry`, an entry of the pieces a and b; 0 outside from .. to - 1
    __device__ __forceinline__ double weight(T a, T b, int64_t entry, int64_t from, int64_t to) const {
        const double w = static_cast<double>(a) - (q != nullptr ? static_cast<double>(b) : entry == certain ? 1.0 : 0.0);
        return w < 0 || entry < from || entry >= to ? 0.0 : w;
    }
    // the weights of the entries at .. at + kCount - 1; 0 from `to` on
    __device__ __forceinline__ void at(int64_t at, int64_t to, double (&w)[kCount]) const {
        const Piece<T> a = load_piece(p, at, to, T(0));
        Piece<T> b{};
        if (q != nullptr) b = load_piece(q, at, to, T(0));
#pragma unroll
        for (int i = 0; i < kCount; ++i) w[i] = weight(a.x[i], b.x[i], at + i, at, to);
    }
    // Their sum over from .. to - 1, by a wave, a piece of either row at a time: more of them in flight take registers, and cost
    // (256 x 50257: one piece 19.9 us, two 21.0, four 23.6, eight 39). A piece that would reach past `to` is read from further
    // down, and its entries before its own first one count nothing.
    __device__ __forceinline__ double sum(int64_t from, int64_t to) const {
        double total = 0;
        if (to < kCount) {
            double w[kCount];
            at(from + threadIdx.x % 64 * kCount, to, w);
#pragma unroll
            for (int i = 0; i < kCount; ++i) total += w[i];
            return wave_sum(total);
        }
        for (int64_t j = from + threadIdx.x % 64 * kCount; j < to; j += 64 * kCount) {
            const int64_t start = min(j, to - kCount);
            Piece<T> a, b{};
            __builtin_memcpy(&a, p + start, 16);
            if (q != nullptr) __builtin_memcpy(&b, q + start, 16);
#pragma unroll
            for (int i = 0; i < kCount; ++i) total += weight(a.x[i], b.x[i], start + i, j, to);
        }
        return wave_sum(total);
    }
};

// The first part whose running sum exceeds `point`, else the last with any weight; `before` becomes the sum ahead of it.
__device__ __forceinline__ int part_of(const double* sums, double point, double& before) {
    int last = 0;
    double run = before, before_last = before;
    for (int w = 0; w < kVerifyWaves; ++w) {
        const double after = run + sums[w];
        if (sums[w] > 0) {
            last = w;
            before_last = run;
            if (after > point) break;
        }
        run = after;
    }
    before = before_last;
    return last;
}

// One sequence's operands, and how its vocabulary is divided: into 16 parts, and each part into 16 small ones, of whole rounds
// of a wave.
template <typename T> struct Verification {
    const T* target;
    const T* draft;
    const int64_t* drafted;
    const int64_t* counts;
    const double* uniforms;
    int64_t drafts, vocab;
    static constexpr int kRound = 64 * Weights<T>::kCount;

    __device__ __forceinline__ int64_t part() const {
        return (vocab + kVerifyWaves * kRound - 1) / (kVerifyWaves * kRound) * kRound;
    }
    __device__ __forceinline__ int64_t small() const { return (part() / kRound + kVerifyWaves - 1) / kVerifyWaves * kRound; }
    __device__ __forceinline__ int64_t count(int64_t s) const {
        const int64_t given = counts[s];
        return given < 0 ? 0 : given > drafts ? drafts : given;
    }
    __device__ __forceinline__ const int64_t* tokens(int64_t s) const { return drafted + s * drafts; }
    // How many of the sequence's drafts are accepted, by a wave.
    __device__ __forceinline__ int64_t accepted(int64_t s) const {
        const int lane = threadIdx.x % 64;
        const int64_t most = count(s);
        const double* u = uniforms + s * (drafts + 1);
        int64_t kept = 0;
        for (bool open = true; open && kept < drafts;) {
            const int64_t i = kept + lane;
            bool good = false;
            if (i < drafts) {  // not count, whose load is under way
                const int64_t token = tokens(s)[i];
                const double draw = u[i];
                if (token >= 0 && token < vocab) {
                    const double p = static_cast<double>(target[(s * (drafts + 1) + i) * vocab + token]);
                    const double q = draft != nullptr ? static_cast<double>(draft[(s * drafts + i) * vocab + token]) : 1.0;
                    good = draw * q < p;
                }
            }
            const uint64_t all = __ballot(good && i < most);
            const int n = all == ~uint64_t{0} ? 64 : __ffsll(static_cast<unsigned long long>(~all)) - 1;
            open = n == 64;
            kept += n;
        }
        return kept;
    }
    // The weights that the token after `kept` accepted drafts is drawn from.
    __device__ __forceinline__ Weights<T> weights(int64_t s, int64_t kept) const {
        Weights<T> w{target + (s * (drafts + 1) + kept) * vocab, nullptr, -1};
        if (kept < count(s)) {
            if (draft != nullptr) w.q = draft + (s * drafts + kept) * vocab;
            else w.certain = tokens(s)[kept];
        }
        return w;
    }
};

// The entry of from .. to - 1 whose running sum, `before` ahead of it, first exceeds `point`, else the last with any weight; by
// a wave.
template <typename T>
__device__ __forceinline__ int64_t entry_of(const Weights<T>& weights, int64_t from, int64_t to, double point, double before) {
    constexpr int kCount = Weights<T>::kCount, kRound = 64 * kCount;
    const int lane = threadIdx.x % 64;
    int64_t picked = -1;
    for (int64_t j0 = from; j0 < to; j0 += kRound) {
        const int64_t j = j0 + lane * kCount;
        double w[kCount], own = 0;
        weights.at(j, to, w);
#pragma unroll
        for (int i = 0; i < kCount; ++i) own += w[i];
        double run = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double other = __shfl_up(run, d);
            if (lane >= d) run += other;
        }
        const double next = before + __shfl(run, 63);
        // the lane's first entry over the point, and its last of any weight
        int over = -1, any = -1;
        run += before - own;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            run += w[i];
            if (w[i] > 0) {
                any = i;
                if (over < 0 && run > point) over = i;
            }
        }
        const uint64_t lanes_over = __ballot(over >= 0), lanes_any = __ballot(any >= 0);
        if (lanes_over != 0) {
            const int first = __ffsll(static_cast<unsigned long long>(lanes_over)) - 1;
            return j0 + first * kCount + __shfl(over, first);
        }
        if (lanes_any != 0) {
            const int last = 63 - __clzll(static_cast<long long>(lanes_any));
            picked = j0 + last * kCount + __shfl(any, last);
        }
        before = next;
    }
    return picked;
}

template <typename T>
__device__ __forceinline__ void write_tokens(int64_t* out, const int64_t* drafted, int64_t drafts, int64_t kept) {
    for (int64_t i = threadIdx.x; i <= drafts; i += blockDim.x)
        if (i != kept) out[i] = i < kept ? drafted[i] : -1;
}

template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_drafts_kernel(int64_t* __restrict__ tokens, int64_t* __restrict__ accepted,
                                                                       Verification<T> v) {
    __shared__ double sums[2][kVerifyWaves];
    const int64_t s = blockIdx.x;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const double last_u = v.uniforms[s * (v.drafts + 1) + v.drafts];
    const int64_t kept = v.accepted(s);
    Weights<T> weights = v.weights(s, kept);
    const int64_t part = v.part();
    double total = 0;
    while (true) {
        const double sum = weights.sum(wave * part, min((wave + 1) * part, v.vocab));
        if (lane == 0) sums[0][wave] = sum;
        __syncthreads();
        total = 0;
        for (int w = 0; w < kVerifyWaves; ++w) total += sums[0][w];
        if (total > 0 || (weights.q == nullptr && weights.certain < 0)) break;
        // nothing is left of p - q (or it is NaN): the target's own probabilities
        weights.q = nullptr;
        weights.certain = -1;
        __syncthreads();
    }
    int64_t* out = tokens + s * (v.drafts + 1);
    write_tokens<T>(out, v.tokens(s), v.drafts, kept);
    if (threadIdx.x == 0) accepted[s] = kept;
    if (!(total > 0 && total < INFINITY)) {
        if (threadIdx.x == 0) out[kept] = -1;
        return;
    }
    const double point = last_u * total;
    double before = 0;
    const int64_t outer = part_of(sums[0], point, before) * part, outer_end = min(outer + part, v.vocab);
    const int64_t small = v.small();
    const double sum = weights.sum(min(outer + wave * small, outer_end), min(outer + (wave + 1) * small, outer_end));
    if (lane == 0) sums[1][wave] = sum;
    __syncthreads();
    const int holder = part_of(sums[1], point, before);
    if (wave != holder) return;
    const int64_t from = outer + holder * small;
    const int64_t picked = entry_of(weights, from, min(from + small, outer_end), point, before);
    if (lane == 0) out[kept] = picked;
}

// The same for few sequences in two launches: sixteen workgroups a sequence sum the small parts, of the weights and of the
// target alone ([sequence][2][256]), and one finds the entry. 8 x 4 drafts of 50257 in f64: 5.1 + 5.0 us, each a launch and a
// chain of loads (counts, drafts, two probabilities, the row).
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(double* __restrict__ sums, int64_t* __restrict__ accepted,
                                                                     Verification<T> v) {
    const int64_t s = blockIdx.y;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, outer_part = blockIdx.x;
    const int64_t kept = v.accepted(s);
    Weights<T> weights = v.weights(s, kept);
    const int64_t part = v.part(), small = v.small();
    const int64_t outer = outer_part * part, outer_end = min(outer + part, v.vocab);
    const int64_t from = min(outer + wave * small, outer_end), to = min(outer + (wave + 1) * small, outer_end);
    double* own = sums + s * 2 * kVerifyWaves * kVerifyWaves + outer_part * kVerifyWaves + wave;
    const double sum = weights.sum(from, to);
    weights.q = nullptr;
    weights.certain = -1;
    const double alone = weights.sum(from, to);
    if (lane == 0) {
        own[0] = sum;
        own[kVerifyWaves * kVerifyWaves] = alone;
    }
    if (outer_part == 0 && threadIdx.x == 0) accepted[s] = kept;
}

template <typename T>
__global__ __launch_bounds__(kVerifyWaves * kVerifyWaves) void verify_entry_kernel(int64_t* __restrict__ tokens,
                                                                                   const int64_t* __restrict__ accepted,
                                                                                   const double* __restrict__ sums, Verification<T> v) {
    __shared__ double small_sums[2][kVerifyWaves * kVerifyWaves], part_sums[2][kVerifyWaves];
    const int64_t s = blockIdx.x;
    const int64_t kept = accepted[s];
    const double last_u = v.uniforms[s * (v.drafts + 1) + v.drafts];
    for (int k = 0; k < 2; ++k)
        small_sums[k][threadIdx.x] = sums[(s * 2 + k) * kVerifyWaves * kVerifyWaves + threadIdx.x];
    __syncthreads();
    if (threadIdx.x < 2 * kVerifyWaves) {
        const int k = threadIdx.x / kVerifyWaves, w = threadIdx.x % kVerifyWaves;
        double sum = 0;
        for (int i = 0; i < kVerifyWaves; ++i) sum += small_sums[k][w * kVerifyWaves + i];
        part_sums[k][w] = sum;
    }
    __syncthreads();
    int64_t* out = tokens + s * (v.drafts + 1);
    write_tokens<T>(out, v.tokens(s), v.drafts, kept);
    if (threadIdx.x >= 64) return;
    Weights<T> weights = v.weights(s, kept);
    int which = 0;
    double total = 0;
    while (true) {
        total = 0;
        for (int w = 0; w < kVerifyWaves; ++w) total += part_sums[which][w];
        if (total > 0 || which == 1) break;
        which = 1;
        weights.q = nullptr;
        weights.certain = -1;
    }
    int64_t picked = -1;
    if (total > 0 && total < INFINITY) {
        const double point = last_u * total;
        double before = 0;
        const int outer = part_of(part_sums[which], point, before);
        const int holder = part_of(small_sums[which] + outer * kVerifyWaves, point, before);
        const int64_t end = min((outer + 1) * v.part(), v.vocab), from = outer * v.part() + holder * v.small();
        picked = entry_of(weights, from, min(from + v.small(), end), point, before);
    }
    if (threadIdx.x == 0) out[kept] = picked;
}

// ---- distillation ---------------------------------------------------------------------------------
//
// Bound by the logits' bytes: the loss reads a row once, with each thread's running maximum and sum, the gradient reads it once
// more and writes it once. The teacher's side (a row's kept entries) is one wave's work in f64, beside the row's. f32, 2048 rows of
// 50257 with 64 kept: 76 + 164 us, 5.4 and 5.0 TB/s; 4096 of 96 with 8 kept: 7.8 + 7.4 us, the launch and the chain of an
// index, its logit and the f64 exponentials and logarithms.

constexpr int kMaxKept = 1024;
constexpr int kNarrow = 256;        // columns up to which a wave holds a row
constexpr int kNarrowRows = 4;      // rows of such a workgroup
constexpr int kMostThreads = 1024;

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) v = max_na(v, __shfl_xor(v, m));
    return v;
}

// exp(x / T) from x and c = kScale / T. f32: the hardware's power of two, whose argument's rounding is no worse than that of
// the quotient itself.
template <typename T> struct Exp;
template <> struct Exp<float> {
    static constexpr double kScale = 1.4426950408889634074;
    __device__ static __forceinline__ float of(float x, float c) { return __builtin_amdgcn_exp2f(x * c); }
};
template <> struct Exp<double> {
    static constexpr double kScale = 1.0;
    __device__ static __forceinline__ double of(double x, double c) { return std::exp(x * c); }
};

// A row's kept entries as one wave sees them: the largest teacher logit, the log of the sum of exponentials, and whether there
// is any entry.
template <typename T> struct Teacher {
    const T* t;
    const int64_t* index;
    int64_t cols;
    int kept;
    double temperature, largest, log_sum;
    bool any;

    __device__ __forceinline__ bool has(int j) const { return j < kept && index[j] >= 0 && index[j] < cols; }
    __device__ __forceinline__ void sum_up() {
        const int lane = threadIdx.x % 64;
        largest = -INFINITY;
        for (int j = lane; j < kept; j += 64)
            if (has(j)) largest = max_na(largest, static_cast<double>(t[j]));
        largest = wave_max(largest);
        any = largest != -INFINITY;
        double sum = 0;
        if (any)
            for (int j = lane; j < kept; j += 64)
                if (has(j)) sum += exp((static_cast<double>(t[j]) - largest) / temperature);
        log_sum = log(wave_sum(sum));
    }
    __device__ __forceinline__ double log_share(int j) const {
        return (static_cast<double>(t[j]) - largest) / temperature - log_sum;
    }
    // T^2 sum pi (log pi - log sigma) for a row z with its maximum and log sum of exponentials
    __device__ __forceinline__ double loss(const T* z, double row_largest, double row_log_sum) const {
        double sum = 0;
        if (any)
            for (int j = threadIdx.x % 64; j < kept; j += 64) {
                if (!has(j)) continue;
                const double own = log_share(j), share = exp(own);
                const double student = (static_cast<double>(z[index[j]]) - row_largest) / temperature - row_log_sum;
                sum += share == 0 ? 0 : share * (own - student);
            }
        return temperature * temperature * wave_sum(sum);
    }
};

template <typename T> __device__ __forceinline__ T or_zero(T largest) { return largest == -INFINITY ? T(0) : largest; }

// A thread's running maximum and its sum of exp((z - largest) / T).
template <typename T> struct Running {
    T largest = -INFINITY;
    double sum = 0;
    template <int N> __device__ __forceinline__ void add(const T (&x)[N], T c) {
        T most = largest;
#pragma unroll
        for (int i = 0; i < N; ++i) most = fmax(most, x[i]);
        const T base = or_zero(most);  // nothing but -inf so far: every exponential is 0
        if (most != largest) sum *= static_cast<double>(Exp<T>::of(largest - base, c));
        largest = most;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += static_cast<double>(Exp<T>::of(x[i] - base, c));
    }
    // the same over a wave
    __device__ __forceinline__ void over_wave(T c) {
        T most = largest;
#pragma unroll
        for (int m = 32; m > 0; m /= 2) most = fmax(most, __shfl_xor(most, m));
        sum = wave_sum(sum * static_cast<double>(Exp<T>::of(largest - or_zero(most), c)));
        largest = most;
    }
};

template <typename T>
__global__ __launch_bounds__(kNarrowRows * 64) void distill_narrow_rows_kernel(T* __restrict__ losses, T* __restrict__ stats,
                                                                               const T* __restrict__ logits,
                                                                               const int64_t* __restrict__ indices,
                                                                               const T* __restrict__ teacher, int64_t rows,
                                                                               int64_t cols, int kept, double temperature) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kNarrowRows + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if (row >= rows) return;
    const T* z = logits + row * cols;
    const T c = static_cast<T>(Exp<T>::kScale / temperature);
    T x[kNarrow / 64];
#pragma unroll
    for (int i = 0; i < kNarrow / 64; ++i) x[i] = lane + 64 * i < cols ? z[lane + 64 * i] : static_cast<T>(-INFINITY);
    Teacher<T> side{teacher + row * kept, indices + row * kept, cols, kept, temperature, 0, 0, false};
    side.sum_up();
    Running<T> run;
    run.add(x, c);
    run.over_wave(c);
    const double loss = side.loss(z, run.largest, log(run.sum));
    if (lane == 0) {
        losses[row] = static_cast<T>(loss);
        stats[2 * row] = run.largest;
        stats[2 * row + 1] = static_cast<T>(run.sum);
    }
}

template <typename T, bool PastLoads>
__global__ __launch_bounds__(kMostThreads) void distill_rows_kernel(T* __restrict__ losses, T* __restrict__ stats,
                                                                    const T* __restrict__ logits, const int64_t* __restrict__ indices,
                                                                    const T* __restrict__ teacher, int64_t cols, int kept,
                                                                    double temperature) {
    __shared__ T wave_largest[kMostThreads / 64];
    __shared__ double wave_sums[kMostThreads / 64];
    constexpr int kCount = Piece<T>::kCount, kPieces = 4;
    const int64_t row = blockIdx.x;
    const int waves = blockDim.x / 64, wave = threadIdx.x / 64;
    const T* z = logits + row * cols;
    const T c = static_cast<T>(Exp<T>::kScale / temperature);
    Running<T> run;
    const int64_t step = static_cast<int64_t>(blockDim.x) * kCount;
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * kCount; at < cols; at += kPieces * step) {
        T x[kPieces * kCount];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const Piece<T> p = load_piece<PastLoads>(z, at + i * step, cols, static_cast<T>(-INFINITY));
#pragma unroll
            for (int j = 0; j < kCount; ++j) x[i * kCount + j] = p.x[j];
        }
        run.add(x, c);
    }
    run.over_wave(c);
    if (threadIdx.x % 64 == 0) {
        wave_largest[wave] = run.largest;
        wave_sums[wave] = run.sum;
    }
    Teacher<T> side{teacher + row * kept, indices + row * kept, cols, kept, temperature, 0, 0, false};
    if (wave == 0) side.sum_up();
    __syncthreads();
    if (wave != 0) return;
    T largest = -INFINITY;
    for (int w = 0; w < waves; ++w) largest = fmax(largest, wave_largest[w]);
    double sum = 0;
    for (int w = 0; w < waves; ++w) sum += wave_sums[w] * static_cast<double>(Exp<T>::of(wave_largest[w] - or_zero(largest), c));
    const double loss = side.loss(z, largest, log(sum));
    if (threadIdx.x == 0) {
        losses[row] = static_cast<T>(loss);
        stats[2 * row] = largest;
        stats[2 * row + 1] = static_cast<T>(sum);
    }
}

template <typename T>
__global__ __launch_bounds__(kNarrowRows * 64) void distill_narrow_grad_kernel(T* out, const T* logits, const T* __restrict__ stats,
                                                                               const int64_t* __restrict__ indices,
                                                                               const T* __restrict__ teacher,
                                                                               const T* __restrict__ row_weights, int64_t rows,
                                                                               int64_t cols, int kept, double temperature) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kNarrowRows + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if (row >= rows) return;
    const T* z = logits + row * cols;
    T x[kNarrow / 64], taken[kNarrow / 64] = {};
#pragma unroll
    for (int i = 0; i < kNarrow / 64; ++i) x[i] = lane + 64 * i < cols ? z[lane + 64 * i] : T(0);
    Teacher<T> side{teacher + row * kept, indices + row * kept, cols, kept, temperature, 0, 0, false};
    side.sum_up();
    // each entry's share to the lane that holds its column, in the entries' order
    if (side.any)
        for (int j0 = 0; j0 < kept; j0 += 64) {
            const int j = j0 + lane;
            const bool in = side.has(j);
            const int place = in ? static_cast<int>(side.index[j]) : -1;
            const T share = in ? static_cast<T>(exp(side.log_share(j))) : T(0);
            for (int i = 0; i < min(64, kept - j0); ++i) {
                const int to = __shfl(place, i);
                const T add = __shfl(share, i);
#pragma unroll
                for (int n = 0; n < kNarrow / 64; ++n) taken[n] += to == lane + 64 * n ? add : T(0);
            }
        }
    const T c = static_cast<T>(Exp<T>::kScale / temperature);
    const T largest = stats[2 * row], weight = static_cast<T>(static_cast<double>(row_weights[row]) * temperature);
    const T factor = weight / stats[2 * row + 1];
    T* g = out + row * cols;
#pragma unroll
    for (int n = 0; n < kNarrow / 64; ++n)
        if (lane + 64 * n < cols) g[lane + 64 * n] = side.any ? Exp<T>::of(x[n] - largest, c) * factor - weight * taken[n] : T(0);
}

template <bool Past, typename T> __device__ __forceinline__ void store_piece(T* to, const Piece<T>& p) {
    u32x4 raw;
    __builtin_memcpy(&raw, &p, 16);
    if constexpr (Past) __builtin_nontemporal_store(raw, reinterpret_cast<u32x4*>(to));
    else *reinterpret_cast<u32x4*>(to) = raw;
}

// A workgroup takes `span` columns of a row. Shared memory: the kept entries' places and shares, and a table of the places
// (twice their number or more, a power of two) in which a place that comes twice is found out. Bound by the logits read and
// the gradient written.
template <typename T, bool PastLoads, bool PastStores>
__global__ __launch_bounds__(kMostThreads) void distill_grad_kernel(T* out, const T* logits, const T* __restrict__ stats,
                                                                    const int64_t* __restrict__ indices,
                                                                    const T* __restrict__ teacher, const T* __restrict__ row_weights,
                                                                    int64_t cols, int kept, double temperature, int64_t span,
                                                                    int spans, int table_size) {
    extern __shared__ char shared[];
    T* shares = reinterpret_cast<T*>(shared);
    int* places = reinterpret_cast<int*>(shares + kept);
    int* table = places + kept;
    __shared__ int twice;
    constexpr int kCount = Piece<T>::kCount, kPieces = 4;
    const int64_t row = blockIdx.x / spans, from = blockIdx.x % spans * span, to = min(from + span, cols);
    Teacher<T> side{teacher + row * kept, indices + row * kept, cols, kept, temperature, 0, 0, false};
    bool entry = false;
    for (int j = threadIdx.x; j < kept; j += blockDim.x) entry = entry || (side.has(j) && side.t[j] != -INFINITY);
    const bool any = __syncthreads_or(entry);
    const T weight = static_cast<T>(static_cast<double>(row_weights[row]) * temperature);
    if (any && threadIdx.x < 64) {
        const int lane = threadIdx.x;
        for (int i = lane; i < table_size; i += 64) table[i] = -1;
        if (lane == 0) twice = 0;
        side.sum_up();
        for (int j = lane; j < kept; j += 64) {
            const bool in = side.has(j) && side.index[j] >= from && side.index[j] < to;
            const int place = in ? static_cast<int>(side.index[j]) : -1;
            places[j] = place;
            shares[j] = in ? static_cast<T>(exp(side.log_share(j))) : T(0);
            if (!in) continue;
            // half of the table at least stays empty, so the walk ends
            for (uint32_t at = static_cast<uint32_t>(place) * 2654435761u;; ++at) {
                const int there = atomicCAS(&table[at & (table_size - 1)], -1, place);
                if (there == place) twice = 1;
                if (there == place || there == -1) break;
            }
        }
    }
    const T c = static_cast<T>(Exp<T>::kScale / temperature);
    const T largest = stats[2 * row], factor = weight / stats[2 * row + 1];
    const T* z = logits + row * cols;
    T* g = out + row * cols;
    const int64_t step = static_cast<int64_t>(blockDim.x) * kCount;
    for (int64_t at = from + static_cast<int64_t>(threadIdx.x) * kCount; at < to; at += kPieces * step) {
        Piece<T> p[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) p[i] = load_piece<PastLoads>(z, at + i * step, to, T(0));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int64_t own = at + i * step;
#pragma unroll
            for (int j = 0; j < kCount; ++j) p[i].x[j] = any ? Exp<T>::of(p[i].x[j] - largest, c) * factor : T(0);
            if (own + kCount <= to) {
                store_piece<PastStores>(g + own, p[i]);
            } else {
#pragma unroll
                for (int j = 0; j < kCount; ++j)
                    if (own + j < to) g[own + j] = p[i].x[j];
            }
        }
    }
    if (!any) return;
    __syncthreads();
    for (int j = threadIdx.x; j < kept; j += blockDim.x) {
        const int place = places[j];
        if (place < 0) continue;
        T share = shares[j];
        if (twice) {
            // the first entry of a place takes the shares of all entries there
            bool first = true;
            for (int i = 0; i < j; ++i) first = first && places[i] != place;
            if (!first) continue;
            for (int i = j + 1; i < kept; ++i) share += places[i] == place ? shares[i] : T(0);
        }
        g[place] -= weight * share;
    }
}

int check_distill(const char* what, int dtype, int64_t rows, int64_t cols, int64_t kept, double temperature) {
    const std::string name(what);
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (rows < 0 || cols < 1 || !fits_grid(rows + 3, cols <= 1024 ? 64 : 256) || cols >= (int64_t{1} << 31))
        return fail(KD_E_INVALID, name + ": bad number of rows or columns");
    if (kept < 1 || kept > kMaxKept) return fail(KD_E_INVALID, name + ": 1 to 1024 kept entries");
    if (!(temperature >= 1e-6 && temperature <= 1e6))
        return fail(KD_E_INVALID, name + ": temperature must be between 1e-6 and 1e6");
    return KD_OK;
}

// Threads of a row's workgroup: one wave for short rows, 1024 threads for long ones where there are too few to fill the card
// with 256.
int row_threads(int64_t rows, int64_t cols) {
    if (cols <= 1024) return 64;
    return rows < 2 * compute_units() && cols >= 8192 ? kMostThreads : 256;
}

// What goes past the caches, by the bytes of the logits: the 256 MiB of the last one hold small logits between the loss, its
// gradient and the gradient's reader; larger ones only drive each other out. Loss and gradient together, f32 rows of 50257,
// logits that were not in the caches, in us: nothing past them / loads past them in both / loads and stores past them in the
// gradient alone:
//   80 MB 52 / 56 / 57    110 MB 82 / 76 / 74    160 MB 125 / 102 / 107    230 MB 169 / 134 / 167
//   300 MB 216 / 183 / 171    412 MB 284 / 272 / 242    800 MB 531 / 557 / 502
struct PastCaches {
    bool loss_loads, grad_loads, grad_stores;
};
PastCaches past_caches(int64_t bytes) {
    const bool large = bytes > int64_t{96} << 20, huge = bytes > int64_t{256} << 20;
    return {large && !huge, large, huge};
}

} // namespace

} // namespace kd

using namespace kd;

extern "C" int kd_verify_drafts(int dtype, int64_t* tokens, int64_t* accepted, const void* target, const void* draft,
                                const int64_t* drafted, const int64_t* counts, const double* uniforms, int64_t sequences,
                                int64_t drafts, int64_t vocab) {
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, "kd_verify_drafts: dtype must be f32 or f64");
    if (sequences < 0 || drafts < 0 || vocab < 1 || !fits_grid(sequences, kVerifyThreads) || drafts >= (int64_t{1} << 20) ||
        vocab >= (int64_t{1} << 31))
        return fail(KD_E_INVALID, "kd_verify_drafts: bad number of sequences, drafts or tokens");
    if (sequences == 0) return KD_OK;
    if (tokens == nullptr || accepted == nullptr || target == nullptr || counts == nullptr || uniforms == nullptr ||
        (drafted == nullptr && drafts > 0))
        return fail(KD_E_INVALID, "kd_verify_drafts: every operand but draft must be given");
    if (int rc = ensure_device()) return rc;
    // Few sequences: one CU takes 6 to 14 us for a long row, and sixteen for each sequence are worth a second launch (one launch /
    // two, us: 1 x 30000 9.5 / 10.4, 1 x 50257 12.9 / 10.4, 1 x 100000 21 / 10.3, 32 x 50257 14.4 / 11.1, 64 x 50257 14.7 / 15.2).
    // Their sums go through the backend's workspace, which may grow, and that is no call to make under capture.
    hipStreamCaptureStatus captured = hipStreamCaptureStatusNone;
    if (stream() != nullptr) KD_HIP(hipStreamIsCapturing(stream(), &captured));
    const bool split = vocab >= 40000 && sequences <= 32 && captured == hipStreamCaptureStatusNone;
    Workspace lease;
    if (split)
        if (int rc = workspace(lease, static_cast<size_t>(sequences) * 2 * kVerifyWaves * kVerifyWaves * sizeof(double))) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        const Verification<T> v{static_cast<const T*>(target), static_cast<const T*>(draft), drafted, counts, uniforms, drafts, vocab};
        const uint32_t groups = static_cast<uint32_t>(sequences);
        if (!split) {
            hipLaunchKernelGGL((verify_drafts_kernel<T>), dim3(groups), dim3(kVerifyThreads), 0, stream(), tokens, accepted, v);
            return;
        }
        double* sums = static_cast<double*>(lease.ptr);
        hipLaunchKernelGGL((verify_sums_kernel<T>), dim3(kVerifyWaves, groups), dim3(kVerifyThreads), 0, stream(), sums, accepted, v);
        hipLaunchKernelGGL((verify_entry_kernel<T>), dim3(groups), dim3(kVerifyWaves * kVerifyWaves), 0, stream(), tokens, accepted,
                           sums, v);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_distill_rows(int dtype, void* losses, void* stats, const void* logits, const int64_t* indices,
                               const void* teacher, int64_t rows, int64_t cols, int64_t kept, double temperature) {
    if (int rc = check_distill("kd_distill_rows", dtype, rows, cols, kept, temperature)) return rc;
    if (rows == 0) return KD_OK;
    if (losses == nullptr || stats == nullptr || logits == nullptr || indices == nullptr || teacher == nullptr)
        return fail(KD_E_INVALID, "kd_distill_rows: every operand must be given");
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        const auto launch_wide = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(rows)), dim3(row_threads(rows, cols)), 0, stream(),
                               static_cast<T*>(losses), static_cast<T*>(stats), static_cast<const T*>(logits), indices,
                               static_cast<const T*>(teacher), cols, static_cast<int>(kept), temperature);
        };
        if (cols <= kNarrow)
            hipLaunchKernelGGL((distill_narrow_rows_kernel<T>), dim3(static_cast<uint32_t>((rows + kNarrowRows - 1) / kNarrowRows)),
                               dim3(kNarrowRows * 64), 0, stream(), static_cast<T*>(losses), static_cast<T*>(stats),
                               static_cast<const T*>(logits), indices, static_cast<const T*>(teacher), rows, cols,
                               static_cast<int>(kept), temperature);
        else if (past_caches(rows * cols * static_cast<int64_t>(sizeof(T))).loss_loads)
            launch_wide(distill_rows_kernel<T, true>);
        else
            launch_wide(distill_rows_kernel<T, false>);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_distill_grad(int dtype, void* out, const void* logits, const void* stats, const int64_t* indices,
                               const void* teacher, const void* row_weights, int64_t rows, int64_t cols, int64_t kept,
                               double temperature) {
    if (int rc = check_distill("kd_distill_grad", dtype, rows, cols, kept, temperature)) return rc;
    if (rows == 0) return KD_OK;
    if (out == nullptr || logits == nullptr || stats == nullptr || indices == nullptr || teacher == nullptr ||
        row_weights == nullptr)
        return fail(KD_E_INVALID, "kd_distill_grad: every operand must be given");
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        if (cols <= kNarrow) {
            hipLaunchKernelGGL((distill_narrow_grad_kernel<T>), dim3(static_cast<uint32_t>((rows + kNarrowRows - 1) / kNarrowRows)),
                               dim3(kNarrowRows * 64), 0, stream(), static_cast<T*>(out), static_cast<const T*>(logits),
                               static_cast<const T*>(stats), indices, static_cast<const T*>(teacher),
                               static_cast<const T*>(row_weights), rows, cols, static_cast<int>(kept), temperature);
            return;
        }
        // few rows: parts of them to a workgroup, in whole rounds of it
        const int threads = row_threads(rows, cols);
        const int64_t round = int64_t{threads} * 4 * Piece<T>::kCount;
        const int64_t wanted = std::max<int64_t>(1, 2 * compute_units() / rows);
        const int64_t span = std::max<int64_t>(1, (cols + round * wanted - 1) / (round * wanted)) * round;
        const int64_t spans = (cols + span - 1) / span;
        int table = 2;
        while (table < 2 * kept) table *= 2;
        const auto launch_wide = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(rows * spans)), dim3(threads),
                               static_cast<uint32_t>(kept * (sizeof(T) + 4) + table * 4), stream(), static_cast<T*>(out),
                               static_cast<const T*>(logits), static_cast<const T*>(stats), indices, static_cast<const T*>(teacher),
                               static_cast<const T*>(row_weights), cols, static_cast<int>(kept), temperature, span,
                               static_cast<int>(spans), table);
        };
        const PastCaches past = past_caches(rows * cols * static_cast<int64_t>(sizeof(T)));
        if (past.grad_stores) launch_wide(distill_grad_kernel<T, true, true>);
        else if (past.grad_loads) launch_wide(distill_grad_kernel<T, true, false>);
        else launch_wide(distill_grad_kernel<T, false, false>);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}
