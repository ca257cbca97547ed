// kd_answers.hip - training on sampled answers and on pairs of them: the targets' log-probabilities with their gradient, the
// preference loss of pairs, and the clipped policy loss with its gradient.
#include <algorithm>

#include "kd_counter.h"
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

// A row's loss and its derivative with respect to the log-probability.
template <typename T> __device__ __forceinline__ void policy_terms(const Policy<T>& a, int64_t row, double lp, double& loss, double& slope) {
    const double advantage = static_cast<double>(a.advantages[row]);
    loss = slope = 0;
    if (advantage != 0) {
        const double ratio = a.old_logps != nullptr ? exp(lp - a.old_logps[row]) : lp == lp ? 1.0 : lp;
        const double free = ratio * advantage, held = fmin(fmax(ratio, 1 - a.low), 1 + a.high) * advantage;
        if (held < free) {
            loss = -held;
        } else {
            loss = slope = -free;
        }
    }
    if (a.reference_logps != nullptr && a.kl_weight != 0) {
        const double d = a.reference_logps[row] - lp, e = expm1(d);
        loss += a.kl_weight * (e - d);
        slope -= a.kl_weight * e;
    }
}

// ---- rows -----------------------------------------------------------------------------------------
//
// The log-probability of a row's target, and with `policy` the row's loss and gradient. A row is read once and held in the
// registers of its team (a wave, or a workgroup): its largest logit, then the exponentials in the logits' places and their sum,
// then the gradient from them. What a team's registers do not hold of a long row is read again, from the caches for the most part.
// Bound by the logits read and the gradient written.

template <typename T> struct AnswerRows {
    T* losses;
    T* grad;
    T* stats;
    double* logps;
    const T* logits;
    const int64_t* targets;
    int64_t rows, cols;
    double temperature;
    Tempered<T> t;
    bool with_policy;
    Policy<T> policy;
};

// What a team writes a row's gradient from: -e * factor, and by more at the target.
template <typename T> struct Slope {
    T factor, by;
};
template <typename T> __device__ __forceinline__ Slope<T> slope_of(double slope, double sum, double temperature) {
    const double by = slope / temperature;
    if (slope == 0) return {0, 0};  // whatever the row holds
    return {static_cast<T>(by / sum), static_cast<T>(by)};
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

constexpr int group_of(int threads) { return threads < 256 ? 256 : threads; }

template <typename T, int Threads, int Pieces, bool Past>
__global__ __launch_bounds__(group_of(Threads)) void answer_rows_kernel(AnswerRows<T> a) {
    constexpr int kWaves = Threads / 64, kTeams = group_of(Threads) / Threads, kCount = Piece<T>::kCount;
    static_assert(kTeams == 1 || kWaves == 1, "teams that leave early may not meet at barriers");
    __shared__ T room_most[16];
    __shared__ double room_sum[16];
    __shared__ Slope<T> room_slope;
    const int wave_at = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64), lane = threadIdx.x % 64;
    const int wave = wave_at % kWaves;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + wave_at / kWaves;
    if (row >= a.rows) return;
    const int64_t target = from_lane(a.targets[row], 0), own = static_cast<int64_t>(wave * 64 + lane) * kCount;
    constexpr int64_t kStep = Threads * kCount, kHeld = kStep * Pieces;
    T* g = a.grad != nullptr ? a.grad + row * a.cols : nullptr;
    if (!is_target(target, a.cols)) {
        if (g != nullptr)
            for (int64_t at = own; at < a.cols; at += kStep) store_grad<Past>(g, at, a.cols, Piece<T>{}, -1, Slope<T>{0, 0});
        if (wave == 0 && lane == 0) {
            if (a.losses != nullptr) a.losses[row] = 0;
            if (a.logps != nullptr) a.logps[row] = 0;
            if (a.stats != nullptr) {
                a.stats[2 * row] = 0;
                a.stats[2 * row + 1] = 1;
            }
        }
        return;
    }
    const T* z = a.logits + row * a.cols;
    const T lowest = static_cast<T>(-INFINITY);
    Piece<T> v[Pieces];
#pragma unroll
    for (int i = 0; i < Pieces; ++i) v[i] = load_piece<Past>(z, own + i * kStep, a.cols, lowest);
    const T there = z[target];
    T most = lowest;  // a NaN is passed over here and comes through its exponential
#pragma unroll
    for (int i = 0; i < Pieces; ++i)
#pragma unroll
        for (int j = 0; j < kCount; ++j) most = fmax(most, v[i].x[j]);
    for (int64_t at = own + kHeld; at < a.cols; at += kStep) {
        const Piece<T> p = load_piece(z, at, a.cols, lowest);
#pragma unroll
        for (int j = 0; j < kCount; ++j) most = fmax(most, p.x[j]);
    }
    most = wave_most(most);
    if constexpr (kWaves > 1) {
        if (lane == 0) room_most[wave] = most;
        __syncthreads();
        most = from_lane(most_of_16(room_most[lane % 16 < kWaves ? lane % 16 : 0]), 15);
    }
    const T base = or_zero(most);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < Pieces; ++i)
#pragma unroll
        for (int j = 0; j < kCount; ++j) {
            v[i].x[j] = a.t.exp(v[i].x[j] - base);
            sum += static_cast<double>(v[i].x[j]);
        }
    for (int64_t at = own + kHeld; at < a.cols; at += kStep) {
        const Piece<T> p = load_piece(z, at, a.cols, lowest);
#pragma unroll
        for (int j = 0; j < kCount; ++j) sum += static_cast<double>(a.t.exp(p.x[j] - base));
    }
    sum = wave_total(sum);
    if constexpr (kWaves > 1) {
        if (lane == 0) room_sum[wave] = sum;
        __syncthreads();
        sum = from_lane(sum_of_16(lane % 16 < kWaves ? room_sum[lane % 16] : 0.0), 15);
    }
    Slope<T> slope{0, 0};
    if (wave == 0) {
        const double lp = (static_cast<double>(there) - static_cast<double>(most)) / a.temperature - log(sum);
        double loss = 0, derivative = 0;
        if (a.with_policy) {
            policy_terms(a.policy, row, lp, loss, derivative);
            if (g != nullptr) slope = slope_of<T>(derivative * static_cast<double>(a.policy.row_weights[row]), sum, a.temperature);
        }
        if (lane == 0) {
            if (a.losses != nullptr) a.losses[row] = static_cast<T>(loss);
            if (a.logps != nullptr) a.logps[row] = lp;
            if (a.stats != nullptr) {
                a.stats[2 * row] = most;
                a.stats[2 * row + 1] = static_cast<T>(sum);
            }
            if (kWaves > 1) room_slope = slope;
        }
    }
    if (g == nullptr) return;
    if constexpr (kWaves > 1) {
        __syncthreads();
        slope = room_slope;
    }
#pragma unroll
    for (int i = 0; i < Pieces; ++i)
        if (own + i * kStep < a.cols) store_grad<Past>(g, own + i * kStep, a.cols, v[i], target, slope);
    for (int64_t at = own + kHeld; at < a.cols; at += kStep) {
        Piece<T> p = load_piece(z, at, a.cols, lowest);
#pragma unroll
        for (int j = 0; j < kCount; ++j) p.x[j] = a.t.exp(p.x[j] - base);
        store_grad<Past>(g, at, a.cols, p, target, slope);
    }
}

// The gradient from a row's statistics: a workgroup takes `span` columns of a row, the last rows first, whose logits the caches
// may still hold from kd_token_logps.
template <typename T, bool PastLoads, bool PastStores>
__global__ __launch_bounds__(256) void token_logps_grad_kernel(T* out, const T* logits, const T* stats, const int64_t* targets,
                                                               const T* slopes, int64_t rows, int64_t cols, double temperature,
                                                               Tempered<T> t, int64_t span, int spans) {
    constexpr int kCount = Piece<T>::kCount, kPieces = 4;
    const int64_t row = rows - 1 - blockIdx.x / spans, from = blockIdx.x % spans * span, to = min(from + span, cols);
    const int64_t target = targets[row];
    const double own = is_target(target, cols) ? static_cast<double>(slopes[row]) : 0.0;
    const Slope<T> slope = slope_of<T>(own, static_cast<double>(stats[2 * row + 1]), temperature);
    const T base = or_zero(stats[2 * row]);
    const T* z = logits + row * cols;
    T* g = out + row * cols;
    constexpr int64_t kStep = 256 * kCount;
    for (int64_t at = from + static_cast<int64_t>(threadIdx.x) * kCount; at < to; at += kPieces * kStep) {
        Piece<T> p[kPieces] = {};
        if (own != 0)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) p[i] = load_piece<PastLoads>(z, at + i * kStep, to, base);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (at + i * kStep >= to) continue;
#pragma unroll
            for (int j = 0; j < kCount; ++j) p[i].x[j] = t.exp(p[i].x[j] - base);
            store_grad<PastStores>(g, at + i * kStep, to, p[i], target, slope);
        }
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

// A team's threads and the 16-byte pieces that each of them holds, by the row's pieces.
template <typename T> void launch_rows(const AnswerRows<T>& a) {
    const int64_t pieces = (a.cols + Piece<T>::kCount - 1) / Piece<T>::kCount;
    const bool past = a.rows * a.cols * static_cast<int64_t>(sizeof(T)) > int64_t{96} << 20;
    const auto one = [&](auto kernel, int threads) {
        const int teams = group_of(threads) / threads;
        hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>((a.rows + teams - 1) / teams)), dim3(group_of(threads)), 0, stream(), a);
    };
    const auto both = [&](auto threads, auto held) {
        constexpr int kThreads = decltype(threads)::value, kPieces = decltype(held)::value;
        if (past) one(answer_rows_kernel<T, kThreads, kPieces, true>, kThreads);
        else one(answer_rows_kernel<T, kThreads, kPieces, false>, kThreads);
    };
    using std::integral_constant;
    if (pieces <= 64) both(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (pieces <= 256) both(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else if (pieces <= 1024) both(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else if (pieces <= 2048) both(integral_constant<int, 512>{}, integral_constant<int, 4>{});
    else if (pieces <= 4096) both(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
    else if (pieces <= 8192) both(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
    else if (pieces <= 13 * 1024) both(integral_constant<int, 1024>{}, integral_constant<int, 13>{});
    else both(integral_constant<int, 1024>{}, integral_constant<int, 20>{});
}

// Whether `out` is neither apart from the logits nor the logits themselves.
bool crosses(const void* out, const void* logits, int dtype, int64_t rows, int64_t cols) {
    const int64_t bytes = rows * cols * dtype_size(dtype);
    return out != logits && overlap(out, bytes, logits, bytes);
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
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        AnswerRows<T> a{nullptr, nullptr, static_cast<T*>(stats), logps, static_cast<const T*>(logits), targets, rows, cols, temperature,
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
    if (crosses(out, logits, dtype, rows, cols)) return fail(KD_E_INVALID, name + ": out overlaps the logits");
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) -> int {
        using T = decltype(zero);
        // parts of a row to a workgroup, in whole rounds of it
        const int64_t round = int64_t{256} * 4 * Piece<T>::kCount;
        const int64_t span = round * std::max<int64_t>(1, std::min<int64_t>((cols + round - 1) / round, 4));
        const int64_t spans = (cols + span - 1) / span;
        if (!fits_grid(rows * spans, 256)) return fail(KD_E_INVALID, name + ": too many rows and columns");
        const auto one = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(rows * spans)), dim3(256), 0, stream(), static_cast<T*>(out),
                               static_cast<const T*>(logits), static_cast<const T*>(stats), targets, static_cast<const T*>(slopes),
                               rows, cols, temperature, Tempered<T>(temperature), span, static_cast<int>(spans));
        };
        const PastCaches past = past_caches(rows * cols * static_cast<int64_t>(sizeof(T)));
        if (past.grad_stores) one(token_logps_grad_kernel<T, true, true>);
        else if (past.grad_loads) one(token_logps_grad_kernel<T, true, false>);
        else one(token_logps_grad_kernel<T, false, false>);
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
    if (grad != nullptr && crosses(grad, logits, dtype, rows, cols)) return fail(KD_E_INVALID, name + ": grad overlaps the logits");
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        AnswerRows<T> a{static_cast<T*>(losses), static_cast<T*>(grad), nullptr, logps, static_cast<const T*>(logits), targets, rows,
                        cols, policy->temperature, Tempered<T>(policy->temperature), true,
                        {policy->old_logps, policy->reference_logps, static_cast<const T*>(policy->advantages),
                         static_cast<const T*>(row_weights), policy->clip_low, policy->clip_high, policy->kl_weight}};
        launch_rows(a);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}
