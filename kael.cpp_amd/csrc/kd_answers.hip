// kd_answers.hip - training on sampled answers and on pairs of them: the targets' log-probabilities with their gradient, the
// preference loss of pairs, and the clipped policy loss with its gradient.
#include <algorithm>

#include "kd_counter.h"
#include "kd_internal.h"
#include "kd_logits.h"

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

// A row's largest logit and its sum of exp((z - largest) / temperature), by a workgroup or by its first wave; `room` holds two
// values a wave.
template <typename T> struct RowSum {
    T largest;
    double sum;
};
template <typename T>
__device__ __forceinline__ RowSum<T> join_rows(RowSum<T> own, const Tempered<T>& t, int lanes) {
    for (int m = lanes / 2; m > 0; m /= 2) {
        const T other = __shfl_xor(own.largest, m);
        const double sum = __shfl_xor(own.sum, m);
        const T most = max_na(own.largest, other);
        const T base = or_zero(most);
        own.sum = own.sum * static_cast<double>(t.exp(own.largest - base)) + sum * static_cast<double>(t.exp(other - base));
        own.largest = most;
    }
    return own;
}
template <typename T> __device__ __forceinline__ RowSum<T> row_sum(const T* z, int64_t cols, const Tempered<T>& t, RowSum<T>* room) {
    RowSum<T> own{static_cast<T>(-INFINITY), 0.0};
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
        const T v = z[c], most = max_na(own.largest, v), base = or_zero(most);
        own.sum = own.sum * static_cast<double>(t.exp(own.largest - base)) + static_cast<double>(t.exp(v - base));
        own.largest = most;
    }
    own = join_rows(own, t, 64);
    __syncthreads();
    if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = own;
    __syncthreads();
    own = room[0];
    for (int w = 1; w < static_cast<int>(blockDim.x) / 64; ++w) {
        const RowSum<T> o = room[w];
        const T most = max_na(own.largest, o.largest), base = or_zero(most);
        own.sum = own.sum * static_cast<double>(t.exp(own.largest - base)) + o.sum * static_cast<double>(t.exp(o.largest - base));
        own.largest = most;
    }
    return own;
}

template <typename T>
__device__ __forceinline__ double logp_of(T at, const RowSum<T>& s, double temperature) {
    return (static_cast<double>(at) - static_cast<double>(s.largest)) / temperature - log(s.sum);
}

__device__ __forceinline__ bool is_target(int64_t t, int64_t cols) { return t >= 0 && t < cols; }

template <typename T>
__global__ __launch_bounds__(256) void token_logps_kernel(double* logps, T* stats, const T* logits, const int64_t* targets, int64_t cols,
                                                          double temperature, Tempered<T> t) {
    __shared__ RowSum<T> room[4];
    const int64_t row = blockIdx.x, target = targets[row];
    if (!is_target(target, cols)) {
        if (threadIdx.x == 0) {
            logps[row] = 0;
            stats[2 * row] = 0;
            stats[2 * row + 1] = 1;
        }
        return;
    }
    const T* z = logits + row * cols;
    const RowSum<T> s = row_sum(z, cols, t, room);
    if (threadIdx.x == 0) {
        logps[row] = logp_of(z[target], s, temperature);
        stats[2 * row] = s.largest;
        stats[2 * row + 1] = static_cast<T>(s.sum);
    }
}

// slope / temperature ((c == target) - softmax_c) for a row; 0 for a slope of 0.
template <typename T>
__device__ __forceinline__ void write_grad(T* g, const T* z, int64_t cols, int64_t target, T largest, T sum, double slope,
                                           double temperature, const Tempered<T>& t) {
    const T by = static_cast<T>(slope / temperature), factor = static_cast<T>(slope / temperature / static_cast<double>(sum));
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x)
        g[c] = slope == 0 ? T(0) : (c == target ? by : T(0)) - t.exp(z[c] - largest) * factor;
}

template <typename T>
__global__ __launch_bounds__(256) void token_logps_grad_kernel(T* out, const T* logits, const T* stats, const int64_t* targets,
                                                               const T* slopes, int64_t cols, double temperature, Tempered<T> t) {
    const int64_t row = blockIdx.x, target = targets[row];
    const double slope = is_target(target, cols) ? static_cast<double>(slopes[row]) : 0.0;
    write_grad(out + row * cols, logits + row * cols, cols, target, stats[2 * row], stats[2 * row + 1], slope, temperature, t);
}

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
        sums[i] = wave_sum(sums[i]);
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
    double temperature, low, high, kl_weight;
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

template <typename T>
__global__ __launch_bounds__(256) void policy_rows_kernel(T* losses, double* logps, T* grad, const T* logits, const int64_t* targets,
                                                          int64_t cols, Policy<T> a, Tempered<T> t) {
    __shared__ RowSum<T> room[4];
    const int64_t row = blockIdx.x, target = targets[row];
    const T* z = logits + row * cols;
    RowSum<T> s{T(0), 1.0};
    double lp = 0, loss = 0, slope = 0;
    if (is_target(target, cols)) {
        s = row_sum(z, cols, t, room);
        lp = logp_of(z[target], s, a.temperature);
        policy_terms(a, row, lp, loss, slope);
        if (grad != nullptr) slope *= static_cast<double>(a.row_weights[row]);
    }
    __syncthreads();  // the target's logit is read before its place is written
    if (threadIdx.x == 0) {
        losses[row] = static_cast<T>(loss);
        if (logps != nullptr) logps[row] = lp;
    }
    if (grad != nullptr) write_grad(grad + row * cols, z, cols, target, s.largest, static_cast<T>(s.sum), slope, a.temperature, t);
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
        hipLaunchKernelGGL((token_logps_kernel<T>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, stream(), logps,
                           static_cast<T*>(stats), static_cast<const T*>(logits), targets, cols, temperature, Tempered<T>(temperature));
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
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL((token_logps_grad_kernel<T>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, stream(),
                           static_cast<T*>(out), static_cast<const T*>(logits), static_cast<const T*>(stats), targets,
                           static_cast<const T*>(slopes), cols, temperature, Tempered<T>(temperature));
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
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
        const Policy<T> a{policy->old_logps, policy->reference_logps, static_cast<const T*>(policy->advantages),
                          static_cast<const T*>(row_weights), policy->temperature, policy->clip_low, policy->clip_high,
                          policy->kl_weight};
        hipLaunchKernelGGL((policy_rows_kernel<T>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, stream(),
                           static_cast<T*>(losses), logps, static_cast<T*>(grad), static_cast<const T*>(logits), targets, cols, a,
                           Tempered<T>(policy->temperature));
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}
