// kd_answers.hip - training on sampled answers and on pairs of them: the targets' log-probabilities with their gradient, the
// preference loss of pairs, and the clipped policy loss with its gradient.
#include <algorithm>
#include <initializer_list>

#include "kd_internal.h"
#include "kd_logits.h"
#include "kd_waves.h"

namespace kd {

namespace {

// exp(d / temperature) of d <= 0. f32: the hardware's power of two of d * (high + low); one f32 factor's rounding would shift
// every exponent of every row the same way, and a long answer's sum of log-probabilities adds that up. high is rounded down
// and low is positive, so that a d of -inf has two terms of -inf.
template <typename T> struct Tempered;
template <> struct Tempered<float> {
    float high, low;
    explicit Tempered(double temperature) {
        const double c = 1.4426950408889634074 / temperature;
        high = static_cast<float>(c);
        if (static_cast<double>(high) > c) high = std::nextafterf(high, 0.f);
        low = std::max(static_cast<float>(c - static_cast<double>(high)), 1e-30f);
    }
    __device__ __forceinline__ float exp(float d) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(d, high, d * low)); }
};
template <> struct Tempered<double> {
    double inverse;
    explicit Tempered(double temperature) : inverse(1.0 / temperature) {}
    __device__ __forceinline__ double exp(double d) const { return std::exp(d * inverse); }
};

__device__ __forceinline__ bool is_target(int64_t t, int64_t cols) { return t >= 0 && t < cols; }

// ---- pairs ----------------------------------------------------------------------------------------
//
// A pair's rows are some thousand numbers, and a chain: starts, the rows' terms, two sums, the loss, the rows' slopes. One launch
// of 4.5 us for 16 pairs of 128 tokens, 7.5 for 32 of 1000.

template <typename T> struct Pairs {
    T* losses;
    T* rewards;
    T* slopes;
    const double* logps;
    const double* reference;
    const int64_t* targets;
    const int64_t* starts;
    const T* weights;
    int64_t pairs, rows, cols;
    double beta, smoothing;
};

// log(1 / (1 + exp(-m))) without overflow.
__device__ __forceinline__ double log_sigmoid(double m) { return (m < 0 ? m : 0.0) - log1p(exp(-fabs(m))); }

// A workgroup a pair: the rows' terms by its threads, their sums in a fixed order.
template <typename T> __global__ __launch_bounds__(256) void preference_pairs_kernel(Pairs<T> a) {
    __shared__ double room[2][4];
    const int64_t p = blockIdx.x;
    int64_t at[3];
    for (int i = 0; i < 3; ++i) at[i] = min(max(a.starts[2 * p + i], int64_t{0}), a.rows);
    double sums[2] = {0, 0};
    for (int i = 0; i < 2; ++i) {
        for (int64_t r = at[i] + threadIdx.x; r < at[i + 1]; r += blockDim.x)
            if (is_target(a.targets[r], a.cols)) sums[i] += a.logps[r] - (a.reference != nullptr ? a.reference[r] : 0.0);
        sums[i] = wave_total(sums[i]);
        if (threadIdx.x % 64 == 0) room[i][threadIdx.x / 64] = sums[i];
    }
    __syncthreads();
    for (int i = 0; i < 2; ++i) sums[i] = a.beta * (((room[i][0] + room[i][1]) + room[i][2]) + room[i][3]);
    const double m = sums[0] - sums[1], up = log_sigmoid(m), down = log_sigmoid(-m);
    if (threadIdx.x == 0) {
        // a weight of 0 takes an infinite term away
        a.losses[p] = static_cast<T>(-(1 - a.smoothing) * up - (a.smoothing > 0 ? a.smoothing * down : 0.0));
        if (a.rewards != nullptr) {
            a.rewards[2 * p] = static_cast<T>(sums[0]);
            a.rewards[2 * p + 1] = static_cast<T>(sums[1]);
        }
    }
    const double slope = a.beta * static_cast<double>(a.weights[p]) * (a.smoothing * exp(up) - (1 - a.smoothing) * exp(down));
    for (int i = 0; i < 2; ++i)
        for (int64_t r = at[i] + threadIdx.x; r < at[i + 1]; r += blockDim.x)
            a.slopes[r] = is_target(a.targets[r], a.cols) ? static_cast<T>(i == 0 ? slope : -slope) : T(0);
    if (p == 0)
        for (int64_t r = threadIdx.x; r < at[0]; r += blockDim.x) a.slopes[r] = T(0);
    if (p == a.pairs - 1)
        for (int64_t r = at[2] + threadIdx.x; r < a.rows; r += blockDim.x) a.slopes[r] = T(0);
}

template <typename T> __global__ __launch_bounds__(256) void zero_kernel(T* out, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) out[i] = T(0);
}

// ---- the clipped policy loss ----------------------------------------------------------------------

template <typename T> struct Policy {
    const double* old_logps;
    const double* reference_logps;
    const T* advantages;
    const T* row_weights;
    double low, high, kl_weight;
};

// A row's loss and its derivative with respect to the log-probability, in lane l and, the same, in lane l + 32 of a wave: its
// two exponentials are one, of the lower and the upper half. It is exp(x) - 1, since a model close to its reference has a d of 1e-8,
// of which exp(d) - d - 1 would be rounding; the ratio's is taken of a positive number, where adding 1 costs half a step.
template <typename T>
__device__ __forceinline__ void policy_terms(const Policy<T>& a, int64_t row, double lp, double& loss, double& slope) {
    const double advantage = static_cast<double>(a.advantages[row]);
    const bool held_near = a.reference_logps != nullptr && a.kl_weight != 0;
    const double moved = a.old_logps != nullptr ? lp - a.old_logps[row] : lp == lp ? 0.0 : lp, d = held_near ? a.reference_logps[row] - lp : 0.0;
    const int lane = threadIdx.x % 64;
    const double both = expm1(lane < 32 ? fabs(moved) : d), far = 1 + __shfl(both, lane % 32), away = __shfl(both, lane % 32 + 32);
    const double ratio = moved < 0 ? 1 / far : far;
    loss = slope = 0;
    if (advantage != 0) {
        const double free = ratio * advantage, held = fmin(fmax(ratio, 1 - a.low), 1 + a.high) * advantage;
        if (held < free) {
            loss = -held;
        } else {
            loss = slope = -free;
        }
    }
    if (held_near) {
        loss += a.kl_weight * (away - d);
        slope -= a.kl_weight * away;
    }
}

// ---- rows -----------------------------------------------------------------------------------------
//
// The log-probability of a row's target, and with `policy` the row's loss and gradient. A row is read once and held in the
// registers of its team (a wave, or a workgroup): its largest logit, then the exponentials in the logits' places and their sum,
// then the gradient from them. What a team's registers do not hold of a long row is read twice more, from the caches for the most
// part: f32 600 x 151936 191 us (693 MB, 3.6 TB/s of what the call has to move), f64 600 x 50257 154 (458 MB, 3.0).
// Bound by the logits read and the gradient written, f32: 2048 rows of 50257 162 us (782 MB at 4.8 TB/s, the rate of a copy;
// vector ALU busy 0.26), 3333 x 6000 29 us; 4096 x 96 5.8 us, a launch and a chain of a target, its row, two sums and four f64 functions.
// f64: 301 x 10007 12.2 us.

template <typename T> struct AnswerRows {
    T* losses;
    T* grad;
    T* stats;
    double* logps;
    const T* logits;
    const int64_t* targets;
    int64_t rows, cols;
    double inverse;  // 1 / temperature
    Tempered<T> t;
    bool with_policy;
    Policy<T> policy;
};

// The gradient's factors of a row: -e * factor, and by more at the target.
template <typename T> struct Slope {
    T factor, by;
};
template <typename T> __device__ __forceinline__ Slope<T> slope_of(double slope, double sum, double inverse) {
    const double by = slope * inverse;
    if (slope == 0) return {0, 0};  // whatever the row holds
    return {static_cast<T>(by / sum), static_cast<T>(by)};
}
// What is written of a row beside its gradient, from its largest logit and the sum of exponentials; the gradient's factors. A lane
// and the one 32 above it have the same row; `lead` says which lanes write. A wave's f64 functions take as long as some hundred
// logits a lane, so they are few, and as far as rows share a wave they are theirs together.
template <typename T>
__device__ __forceinline__ Slope<T> finish_row(const AnswerRows<T>& a, int64_t row, T there, T most, double sum, bool lead) {
    const double lp = (static_cast<double>(there) - static_cast<double>(most)) * a.inverse - log(sum);
    double loss = 0, derivative = 0;
    Slope<T> slope{0, 0};
    if (a.with_policy) {
        policy_terms(a.policy, row, lp, loss, derivative);
        if (a.grad != nullptr) slope = slope_of<T>(derivative * static_cast<double>(a.policy.row_weights[row]), sum, a.inverse);
    }
    if (lead) {
        if (a.losses != nullptr) a.losses[row] = static_cast<T>(loss);
        if (a.logps != nullptr) a.logps[row] = lp;
        if (a.stats != nullptr) {
            a.stats[2 * row] = most;
            a.stats[2 * row + 1] = static_cast<T>(sum);
        }
    }
    return slope;
}
// The same for a row without a target.
template <typename T> __device__ __forceinline__ void empty_row(const AnswerRows<T>& a, int64_t row) {
    if (a.losses != nullptr) a.losses[row] = 0;
    if (a.logps != nullptr) a.logps[row] = 0;
    if (a.stats != nullptr) {
        a.stats[2 * row] = 0;
        a.stats[2 * row + 1] = 1;
    }
}

// The gradient of a piece whose exponentials are given.
template <bool Past, typename T>
__device__ __forceinline__ void store_grad(T* g, int64_t at, int64_t cols, Piece<T> p, int64_t target, const Slope<T>& s) {
    constexpr int kCount = Piece<T>::kCount;
#pragma unroll
    for (int j = 0; j < kCount; ++j) p.x[j] = s.factor == 0 && s.by == 0 ? T(0) : (at + j == target ? s.by : T(0)) - p.x[j] * s.factor;
    if (at + kCount <= cols) {
        store_piece<Past>(g + at, p);
    } else {
#pragma unroll
        for (int j = 0; j < kCount; ++j)
            if (at + j < cols) g[at + j] = p.x[j];
    }
}

// Short rows: a wave has `Rows` of them, `Pieces` a lane each.
constexpr int kShortThreads = 256;

template <typename T, int Pieces, int Rows, bool PastLoads, bool PastStores>
__global__ __launch_bounds__(kShortThreads) void answer_short_kernel(AnswerRows<T> a) {
    constexpr int kCount = Piece<T>::kCount, kStep = 64 * kCount;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64), lane = threadIdx.x % 64;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * (kShortThreads / 64) + wave) * Rows;
    if (first >= a.rows) return;
    const T lowest = static_cast<T>(-INFINITY);
    const int own = lane * kCount;
    // lane r and lane 32 + r: row r's
    const int64_t lane_row = min(first + lane % 32 % Rows, a.rows - 1), lane_target = a.targets[lane_row];
    int64_t target[Rows];
    Piece<T> v[Rows][Pieces];
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        target[r] = from_lane(lane_target, r);
        if (first + r >= a.rows || !is_target(target[r], a.cols)) target[r] = -1;
        const T* z = a.logits + (first + r) * a.cols;
#pragma unroll
        for (int i = 0; i < Pieces; ++i)
            if (target[r] >= 0) v[r][i] = load_piece<PastLoads>(z, own + i * kStep, a.cols, lowest);
    }
    const bool counted = is_target(lane_target, a.cols);
    const T there = counted ? a.logits[lane_row * a.cols + lane_target] : T(0);
    T lane_most = 0;
    double lane_sum = 1;
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        if (target[r] < 0) continue;
        T most = lowest;  // a NaN is passed over here and comes through its exponential
#pragma unroll
        for (int i = 0; i < Pieces; ++i)
#pragma unroll
            for (int j = 0; j < kCount; ++j) most = fmax(most, v[r][i].x[j]);
        most = wave_most(most);
        const T base = or_zero(most);
        double sum = 0;
#pragma unroll
        for (int i = 0; i < Pieces; ++i)
#pragma unroll
            for (int j = 0; j < kCount; ++j) {
                v[r][i].x[j] = a.t.exp(v[r][i].x[j] - base);
                sum += static_cast<double>(v[r][i].x[j]);
            }
        sum = wave_total(sum);
        if (lane % 32 % Rows == r) {
            lane_most = most;
            lane_sum = sum;
        }
    }
    Slope<T> lane_slope = finish_row(a, lane_row, there, lane_most, lane_sum, lane < Rows && counted && first + lane < a.rows);
    if (lane < Rows && !counted && first + lane < a.rows) empty_row(a, lane_row);
    if (a.grad == nullptr) return;
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
        if (first + r >= a.rows) continue;
        Slope<T> slope{from_lane(lane_slope.factor, r), from_lane(lane_slope.by, r)};
        if (target[r] < 0) slope = {0, 0};
        T* g = a.grad + (first + r) * a.cols;
#pragma unroll
        for (int i = 0; i < Pieces; ++i)
            if (own + i * kStep < a.cols) store_grad<PastStores>(g, own + i * kStep, a.cols, v[r][i], target[r], slope);
    }
}

// Longer rows: a workgroup has one. More: `Pieces` a thread are not all of it.
template <typename T, int Threads, int Pieces, bool More, bool PastLoads, bool PastStores>
__global__ __launch_bounds__(Threads) void answer_rows_kernel(AnswerRows<T> a) {
    constexpr int kWaves = Threads / 64, kCount = Piece<T>::kCount;
    __shared__ T room_most[16];
    __shared__ double room_sum[16];
    __shared__ Slope<T> room_slope;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64), lane = threadIdx.x % 64;
    const int64_t row = blockIdx.x, target = a.targets[row], own = static_cast<int64_t>(threadIdx.x) * kCount;
    constexpr int64_t kStep = Threads * kCount, kHeld = kStep * Pieces;
    T* g = a.grad + row * a.cols;
    if (!is_target(target, a.cols)) {
        if (a.grad != nullptr)
            for (int64_t at = own; at < a.cols; at += kStep) store_grad<PastStores>(g, at, a.cols, Piece<T>{}, -1, Slope<T>{0, 0});
        if (threadIdx.x == 0) empty_row(a, row);
        return;
    }
    const T* z = a.logits + row * a.cols;
    const T lowest = static_cast<T>(-INFINITY);
    Piece<T> v[Pieces];
#pragma unroll
    for (int i = 0; i < Pieces; ++i) v[i] = load_piece<PastLoads>(z, own + i * kStep, a.cols, lowest);
    const T there = z[target];
    T most = lowest;  // a NaN is passed over here and comes through its exponential
#pragma unroll
    for (int i = 0; i < Pieces; ++i)
#pragma unroll
        for (int j = 0; j < kCount; ++j) most = fmax(most, v[i].x[j]);
    // what is not held, four pieces at a time
    constexpr int kMore = 4;
    const auto rest = [&](auto&& use) {
        if constexpr (More)
            for (int64_t at = own + kHeld; at < a.cols; at += kMore * kStep) {
                Piece<T> p[kMore];
#pragma unroll
                for (int i = 0; i < kMore; ++i) p[i] = load_piece(z, at + i * kStep, a.cols, lowest);
#pragma unroll
                for (int i = 0; i < kMore; ++i)
                    if (at + i * kStep < a.cols) use(p[i], at + i * kStep);
            }
    };
    rest([&](const Piece<T>& p, int64_t) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) most = fmax(most, p.x[j]);
    });
    most = wave_most(most);
    if (lane == 0) room_most[wave] = most;
    __syncthreads();
    most = from_lane(most_of_16(room_most[lane % 16 < kWaves ? lane % 16 : 0]), 15);
    const T base = or_zero(most);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < Pieces; ++i)
#pragma unroll
        for (int j = 0; j < kCount; ++j) {
            v[i].x[j] = a.t.exp(v[i].x[j] - base);
            sum += static_cast<double>(v[i].x[j]);
        }
    rest([&](const Piece<T>& p, int64_t) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) sum += static_cast<double>(a.t.exp(p.x[j] - base));
    });
    sum = wave_total(sum);
    if (lane == 0) room_sum[wave] = sum;
    __syncthreads();
    sum = from_lane(sum_of_16(lane % 16 < kWaves ? room_sum[lane % 16] : 0.0), 15);
    // by turns, since the first waves of all workgroups share a SIMD
    if (wave == static_cast<int>(blockIdx.x % kWaves)) {
        const Slope<T> slope = finish_row(a, row, there, most, sum, lane == 0);
        if (lane == 0) room_slope = slope;
    }
    if (a.grad == nullptr) return;
    __syncthreads();
    const Slope<T> slope = room_slope;
#pragma unroll
    for (int i = 0; i < Pieces; ++i)
        if (own + i * kStep < a.cols) store_grad<PastStores>(g, own + i * kStep, a.cols, v[i], target, slope);
    rest([&](Piece<T>& p, int64_t at) {
#pragma unroll
        for (int j = 0; j < kCount; ++j) p.x[j] = a.t.exp(p.x[j] - base);
        store_grad<PastStores>(g, at, a.cols, p, target, slope);
    });
}

// Without a gradient no row is held: a workgroup reads a long one in rounds of four pieces a thread, and a CU's eight waves a SIMD
// have the next loads on their way while one computes. A wave takes its exponentials from the largest logit that it has seen: an f32
// exponential's error grows with the distance from its base, so a confident target has to be that base, whose exponential is
// exactly 1 (with the largest logit of a row's first round as the base of all, targets 12 to 39 above it were 4e-7 to 2e-6 off and above 0).
// A round that holds a larger one moves the sum there first, in f64, whose rounding does not count beside f32's; that is seldom: a
// wave's k-th round does so with a chance of 1 / k. 1433 rows of 50257 of 1908: 61 to 66 us, by the machine (288 MB at 4.4 to 4.7 TB/s); held
// in registers, one workgroup a CU, 69. f64: 500 x 50257 41 us (4.9 TB/s).
template <typename T>
__global__ __launch_bounds__(kMostThreads) void answer_forward_kernel(AnswerRows<T> a) {
    constexpr int kCount = Piece<T>::kCount, kPieces = 4;
    __shared__ T room_most[16];
    __shared__ double room_sum[16];
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64), lane = threadIdx.x % 64;
    const int waves = blockDim.x / 64;
    const int64_t row = blockIdx.x, target = a.targets[row];
    if (!is_target(target, a.cols)) {
        if (threadIdx.x == 0) empty_row(a, row);
        return;
    }
    const T* z = a.logits + row * a.cols;
    const T there = z[target], lowest = static_cast<T>(-INFINITY);
    const int64_t own = static_cast<int64_t>(threadIdx.x) * kCount, step = static_cast<int64_t>(blockDim.x) * kCount;
    T base = lowest;
    double sum = 0;
    // the same rounds for all lanes: what is behind the row's end is -inf
    for (int64_t from = 0; from < a.cols; from += kPieces * step) {
        Piece<T> p[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) p[i] = load_piece(z, from + own + i * step, a.cols, lowest);
        T most = base;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int j = 0; j < kCount; ++j) most = fmax(most, p[i].x[j]);  // passes over NaN, which the sum takes up
        if (__any(most > base)) {
            most = wave_most(most);
            if (base != lowest) sum *= exp((static_cast<double>(base) - static_cast<double>(most)) * a.inverse);
            base = most;
        }
        const T from_base = or_zero(base);
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int j = 0; j < kCount; ++j) sum += static_cast<double>(a.t.exp(p[i].x[j] - from_base));
    }
    sum = wave_total(sum);
    if (lane == 0) {
        room_most[wave] = base;
        room_sum[wave] = sum;
    }
    __syncthreads();
    if (wave != 0) return;
    const int w = lane % 16 < waves ? lane % 16 : 0;
    base = room_most[w];
    const T most = from_lane(most_of_16(base), 15);
    sum = lane % 16 < waves ? room_sum[w] : 0.0;
    if (base != most) sum *= exp((static_cast<double>(base) - static_cast<double>(most)) * a.inverse);
    sum = from_lane(sum_of_16(sum), 15);
    finish_row(a, row, there, most, sum, lane == 0);
}

// The gradient from a row's statistics: a team of `Threads` (of a workgroup of 256) takes a round of a row, the last rows first, whose logits the caches may still
// hold from kd_token_logps (1908 x 50257: 105 to 113 us; from the first row on 16 more).
template <typename T, int Threads, bool Past>
__global__ __launch_bounds__(256) void token_logps_grad_kernel(T* out, const T* logits, const T* stats, const int64_t* targets,
                                                               const T* slopes, int64_t rows, int64_t cols, double inverse,
                                                               Tempered<T> t, int spans) {
    constexpr int kCount = Piece<T>::kCount, kPieces = 4;
    constexpr int64_t kStep = Threads * kCount;
    const int team = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64) / (Threads / 64);
    const int64_t round = static_cast<int64_t>(blockIdx.x) * (256 / Threads) + team;
    const int64_t row = rows - 1 - round / spans, at = round % spans * kPieces * kStep + static_cast<int64_t>(threadIdx.x % Threads) * kCount;
    if (row < 0) return;
    const int64_t target = targets[row];
    const double own = is_target(target, cols) ? static_cast<double>(slopes[row]) : 0.0;
    const Slope<T> slope = slope_of<T>(own, static_cast<double>(stats[2 * row + 1]), inverse);
    const T base = or_zero(stats[2 * row]);
    const T* z = logits + row * cols;
    T* g = out + row * cols;
    Piece<T> p[kPieces] = {};
    if (own != 0)
#pragma unroll
        for (int i = 0; i < kPieces; ++i) p[i] = load_piece(z, at + i * kStep, cols, base);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        if (at + i * kStep >= cols) continue;
#pragma unroll
        for (int j = 0; j < kCount; ++j) p[i].x[j] = t.exp(p[i].x[j] - base);
        store_grad<Past>(g, at + i * kStep, cols, p[i], target, slope);
    }
}

// ---- checks ---------------------------------------------------------------------------------------

int check_rows(const std::string& name, int dtype, int64_t rows, int64_t cols, double temperature) {
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (rows < 0 || cols < 1 || !fits_grid(rows + 3, kMostThreads) || cols >= (int64_t{1} << 31))
        return fail(KD_E_INVALID, name + ": bad number of rows or columns");
    if (!(temperature >= 1e-6 && temperature <= 1e6))
        return fail(KD_E_INVALID, name + ": temperature must be between 1e-6 and 1e6");
    return KD_OK;
}

template <int N> using Int = std::integral_constant<int, N>;

// Threads and the 16-byte pieces that each of them holds, by the row's pieces: as many as leave the registers of two workgroups of
// 1024 to a CU up to 5 pieces, of one up to 13; halved teams that hold twice as much measured the same or slower (2000 x 10000 f32 35.0
// us both, 4000 x 5000 30).
template <typename T> void launch_rows(const AnswerRows<T>& a) {
    const int64_t pieces = (a.cols + Piece<T>::kCount - 1) / Piece<T>::kCount;
    // Logits that are read once go past the caches where they would drive the gradient out of them, and so does a gradient that
    // the last cache's 256 MiB cannot hold. f32 rows of 50257, us: neither / loads / stores / both:
    //   40 MB 18.5 / 20.3 / 19.8 / 21.7    100 MB 43.1 / 42.1 / 42.7 / 48.4    181 MB 86.5 / 73.0 / 85.4 / 82.8
    //   281 MB 119 / 107 / 120 / 120    412 MB 170 / 167 / 164 / 163
    const int64_t bytes = a.rows * a.cols * static_cast<int64_t>(sizeof(T));
    const bool past_loads = bytes > int64_t{128} << 20, past_stores = bytes > int64_t{320} << 20;
    if (a.grad == nullptr && pieces > 1024) {
        hipLaunchKernelGGL((answer_forward_kernel<T>), dim3(static_cast<uint32_t>(a.rows)), dim3(row_threads(a.rows, a.cols)), 0,
                           stream(), a);
        return;
    }
    const auto with = [&](auto kernel, int64_t groups, int threads) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(threads), 0, stream(), a);
    };
    const auto by_caches = [&](auto launch) {
        if (past_stores) launch(std::true_type{}, std::true_type{});
        else if (past_loads) launch(std::true_type{}, std::false_type{});
        else launch(std::false_type{}, std::false_type{});
    };
    if (pieces <= 256) {
        // Four rows share a wave's f64 functions where there are enough of them: 66667 x 300 44.6 us (one a wave 52.9), but 4096 x 96
        // 6.3 (5.5) and, with two rows, 33333 x 600 38.5 (36).
        const auto rows = [&](auto held, auto together) {
            by_caches([&](auto loads, auto stores) {
                constexpr int kTogether = decltype(together)::value, kGroup = kShortThreads / 64 * kTogether;
                with(answer_short_kernel<T, decltype(held)::value, kTogether, decltype(loads)::value, decltype(stores)::value>,
                     (a.rows + kGroup - 1) / kGroup, kShortThreads);
            });
        };
        const bool many = a.rows >= 64 * compute_units();
        if (pieces <= 64) many ? rows(Int<1>{}, Int<4>{}) : rows(Int<1>{}, Int<1>{});
        else if (pieces <= 128) many ? rows(Int<2>{}, Int<4>{}) : rows(Int<2>{}, Int<1>{});
        else rows(Int<4>{}, Int<1>{});
        return;
    }
    const auto row = [&](auto threads, auto held, auto more) {
        by_caches([&](auto loads, auto stores) {
            constexpr int kThreads = decltype(threads)::value;
            with(answer_rows_kernel<T, kThreads, decltype(held)::value, decltype(more)::value, decltype(loads)::value, decltype(stores)::value>,
                 a.rows, kThreads);
        });
    };
    if (pieces <= 512) row(Int<256>{}, Int<2>{}, std::false_type{});
    else if (pieces <= 1024) row(Int<256>{}, Int<4>{}, std::false_type{});
    else if (pieces <= 2048) row(Int<512>{}, Int<4>{}, std::false_type{});
    else if (pieces <= 4096) row(Int<1024>{}, Int<4>{}, std::false_type{});
    else if (pieces <= 5 * 1024) row(Int<1024>{}, Int<5>{}, std::false_type{});
    else if (pieces <= 8 * 1024) row(Int<1024>{}, Int<8>{}, std::false_type{});
    else if (pieces <= 13 * 1024) row(Int<1024>{}, Int<13>{}, std::false_type{});
    else row(Int<1024>{}, Int<14>{}, std::true_type{});
}

struct Operand {
    const void* at;
    int64_t count, size;  // of its elements
    int same = -1;        // of an input: the output that may stand in its very place, since it reads an element before it writes it
};
// Refuses an operand that is not aligned to its elements, and an output that has a byte in common with another operand.
int check_operands(const std::string& name, std::initializer_list<Operand> outs, std::initializer_list<Operand> ins) {
    const auto crosses = [](const Operand& a, const Operand& b) { return overlap(a.at, a.count * a.size, b.at, b.count * b.size); };
    for (const auto* operands : {&outs, &ins})
        for (const Operand& o : *operands)
            if (reinterpret_cast<uintptr_t>(o.at) % static_cast<uintptr_t>(o.size) != 0)
                return fail(KD_E_INVALID, name + ": an operand is not aligned to its elements");
    int place = 0;
    for (const Operand& out : outs) {
        for (const Operand& other : outs)
            if (&out != &other && crosses(out, other)) return fail(KD_E_INVALID, name + ": outputs overlap");
        for (const Operand& in : ins)
            if (!(in.same == place && out.at == in.at) && crosses(out, in)) return fail(KD_E_INVALID, name + ": an output overlaps an input");
        ++place;
    }
    return KD_OK;
}

} // namespace

} // namespace kd

using namespace kd;

extern "C" int kd_token_logps(int dtype, double* logps, void* stats, const void* logits, const int64_t* targets, int64_t rows,
                              int64_t cols, double temperature) {
    const std::string name("kd_token_logps");
    if (int rc = check_rows(name, dtype, rows, cols, temperature)) return rc;
    if (rows == 0) return KD_OK;
    if (logps == nullptr || stats == nullptr || logits == nullptr || targets == nullptr)
        return fail(KD_E_INVALID, name + ": every operand must be given");
    const int64_t size = dtype_size(dtype);
    if (int rc = check_operands(name, {{logps, rows, 8}, {stats, 2 * rows, size}}, {{logits, rows * cols, size}, {targets, rows, 8}})) return rc;
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        AnswerRows<T> a{nullptr, nullptr, static_cast<T*>(stats), logps, static_cast<const T*>(logits), targets, rows, cols, 1.0 / temperature,
                        Tempered<T>(temperature), false, {}};
        launch_rows(a);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_token_logps_grad(int dtype, void* out, const void* logits, const void* stats, const int64_t* targets,
                                   const void* slopes, int64_t rows, int64_t cols, double temperature) {
    const std::string name("kd_token_logps_grad");
    if (int rc = check_rows(name, dtype, rows, cols, temperature)) return rc;
    if (rows == 0) return KD_OK;
    if (out == nullptr || logits == nullptr || stats == nullptr || targets == nullptr || slopes == nullptr)
        return fail(KD_E_INVALID, name + ": every operand must be given");
    const int64_t size = dtype_size(dtype);
    if (int rc = check_operands(name, {{out, rows * cols, size}},
                                {{logits, rows * cols, size, 0}, {stats, 2 * rows, size}, {targets, rows, 8}, {slopes, rows, size}}))
        return rc;
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) -> int {
        using T = decltype(zero);
        // one round a team: with two 2 % slower, with four 20 % (1908 x 50257)
        const auto one = [&](auto kernel, int threads) -> int {
            const int64_t span = int64_t{threads} * 4 * Piece<T>::kCount, spans = (cols + span - 1) / span;
            const int64_t groups = (rows * spans + 256 / threads - 1) / (256 / threads);
            if (!fits_grid(groups, 256)) return fail(KD_E_INVALID, name + ": too many rows and columns");
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(256), 0, stream(), static_cast<T*>(out),
                               static_cast<const T*>(logits), static_cast<const T*>(stats), targets, static_cast<const T*>(slopes),
                               rows, cols, 1.0 / temperature, Tempered<T>(temperature), static_cast<int>(spans));
            return KD_OK;
        };
        // A gradient that goes past the caches leaves the logits in them. With kd_token_logps, f32 rows of 50257, us, through / past:
        // 50 MB 26.3 / 27.4, 130 MB 69 / 58, 231 MB 134 / 116, 369 MB 202 / 176.
        const bool past = rows * cols * static_cast<int64_t>(sizeof(T)) > int64_t{96} << 20;
        const bool brief = cols <= 64 * 4 * Piece<T>::kCount;  // a wave's round
        if (int rc = brief ? past ? one(token_logps_grad_kernel<T, 64, true>, 64) : one(token_logps_grad_kernel<T, 64, false>, 64)
                           : past ? one(token_logps_grad_kernel<T, 256, true>, 256) : one(token_logps_grad_kernel<T, 256, false>, 256))
            return rc;
        KD_LAUNCH_CHECK();
        return KD_OK;
    };
    return dtype == KD_F32 ? launch(0.f) : launch(0.0);
}

extern "C" int kd_preference_pairs(int dtype, void* losses, void* rewards, void* slopes, const double* logps,
                                   const double* reference, const int64_t* targets, const int64_t* starts, const void* weights,
                                   int64_t pairs, int64_t rows, int64_t cols, double beta, double smoothing) {
    const std::string name("kd_preference_pairs");
    if (int rc = check_rows(name, dtype, rows, cols, 1.0)) return rc;
    if (pairs < 0 || !fits_grid(pairs + 3, kMostThreads)) return fail(KD_E_INVALID, name + ": bad number of pairs");
    if (!(beta > 0 && beta <= 1e6)) return fail(KD_E_INVALID, name + ": beta must be above 0 and at most 1e6");
    if (!(smoothing >= 0 && smoothing < 0.5)) return fail(KD_E_INVALID, name + ": smoothing must be 0 or more and below 0.5");
    if (pairs == 0 && rows == 0) return KD_OK;
    if ((pairs > 0 && (losses == nullptr || starts == nullptr || weights == nullptr)) ||
        (rows > 0 && (slopes == nullptr || logps == nullptr || targets == nullptr)))
        return fail(KD_E_INVALID, name + ": every operand but rewards and reference must be given");
    const int64_t size = dtype_size(dtype), read = pairs > 0 ? rows : 0;  // without pairs the slopes alone are written
    const int same = dtype == KD_F64 ? 2 : -1;
    if (int rc = check_operands(name, {{losses, pairs, size}, {rewards, 2 * pairs, size}, {slopes, rows, size}},
                                {{logps, read, 8, same}, {reference, read, 8, same}, {targets, read, 8}, {starts, 2 * pairs + 1, 8}, {weights, pairs, size}}))
        return rc;
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        if (pairs == 0) {
            hipLaunchKernelGGL((zero_kernel<T>), dim3(static_cast<uint32_t>(std::min<int64_t>((rows + 255) / 256, 1024))), dim3(256), 0,
                               stream(), static_cast<T*>(slopes), rows);
            return;
        }
        const Pairs<T> a{static_cast<T*>(losses), static_cast<T*>(rewards), static_cast<T*>(slopes), logps, reference, targets,
                         starts, static_cast<const T*>(weights), pairs, rows, cols, beta, smoothing};
        hipLaunchKernelGGL((preference_pairs_kernel<T>), dim3(static_cast<uint32_t>(pairs)), dim3(256), 0, stream(), a);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_policy_rows(int dtype, void* losses, double* logps, void* grad, const void* logits, const int64_t* targets,
                              const kd_policy* policy, const void* row_weights, int64_t rows, int64_t cols) {
    const std::string name("kd_policy_rows");
    if (policy == nullptr) return fail(KD_E_INVALID, name + ": the policy must be given");
    if (int rc = check_rows(name, dtype, rows, cols, policy->temperature)) return rc;
    if (!(policy->clip_low >= 0 && policy->clip_low <= 1) || !(policy->clip_high >= 0 && policy->clip_high <= 1e6) ||
        !(policy->kl_weight >= 0 && policy->kl_weight <= 1e6))
        return fail(KD_E_INVALID, name + ": clip_low must be 0 to 1, clip_high and kl_weight 0 to 1e6");
    if (rows == 0) return KD_OK;
    if (losses == nullptr || logits == nullptr || targets == nullptr || policy->advantages == nullptr ||
        (grad != nullptr && row_weights == nullptr))
        return fail(KD_E_INVALID, name + ": losses, logits, targets, advantages and, for a gradient, row_weights must be given");
    const int64_t size = dtype_size(dtype);
    if (int rc = check_operands(name, {{losses, rows, size}, {logps, rows, 8}, {grad, rows * cols, size}},
                                {{logits, rows * cols, size, 2}, {targets, rows, 8}, {policy->old_logps, rows, 8, 1},
                                 {policy->reference_logps, rows, 8, 1}, {policy->advantages, rows, size, 0},
                                 {grad != nullptr ? row_weights : nullptr, rows, size, 0}}))
        return rc;
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        AnswerRows<T> a{static_cast<T*>(losses), static_cast<T*>(grad), nullptr, logps, static_cast<const T*>(logits), targets, rows,
                        cols, 1.0 / policy->temperature, Tempered<T>(policy->temperature), true,
                        {policy->old_logps, policy->reference_logps, static_cast<const T*>(policy->advantages),
                         static_cast<const T*>(row_weights), policy->clip_low, policy->clip_high, policy->kl_weight}};
        launch_rows(a);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}
