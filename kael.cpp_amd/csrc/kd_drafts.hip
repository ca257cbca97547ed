// kd_drafts.hip - a draft model beside its target: verification of drafted tokens against the target's probabilities,
// and the distillation loss against the target's top logits with its gradient.
#include "kd_internal.h"

namespace kd {

namespace {

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) v += __shfl_xor(v, m);
    return v;
}

// ---- verification ---------------------------------------------------------------------------------

constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWaves = kVerifyThreads / 64;

// The weight of entry j: p - q where that is positive, p itself without a draft row; NaN stays NaN.
template <typename T> struct Weights {
    const T* p;
    const T* q;        // NULL: no draft row
    int64_t certain;   // q NULL: the entry whose q is 1, or -1
    __device__ __forceinline__ double operator()(int64_t j) const {
        double w = static_cast<double>(p[j]);
        if (q != nullptr) w -= static_cast<double>(q[j]);
        else if (j == certain) w -= 1.0;
        return w < 0 ? 0.0 : w;
    }
};

// One workgroup a sequence, a contiguous part of the vocabulary a wave.
template <typename T>
__global__ __launch_bounds__(kVerifyThreads) void verify_drafts_kernel(int64_t* __restrict__ tokens, int64_t* __restrict__ accepted,
                                                                       const T* __restrict__ target, const T* __restrict__ draft,
                                                                       const int64_t* __restrict__ drafted,
                                                                       const int64_t* __restrict__ counts,
                                                                       const double* __restrict__ uniforms, int64_t drafts,
                                                                       int64_t vocab) {
    __shared__ double sums[kVerifyWaves];
    const int64_t s = blockIdx.x;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t count = min(max(counts[s], int64_t{0}), drafts);
    const int64_t* x = drafted + s * drafts;
    const double* u = uniforms + s * (drafts + 1);
    int64_t kept = 0;
    for (bool open = true; open && kept < count;) {
        const int64_t i = kept + lane;
        bool good = false;
        if (i < count) {
            const int64_t token = x[i];
            if (token >= 0 && token < vocab) {
                const double p = static_cast<double>(target[(s * (drafts + 1) + i) * vocab + token]);
                const double q = draft != nullptr ? static_cast<double>(draft[(s * drafts + i) * vocab + token]) : 1.0;
                good = u[i] * q < p;
            }
        }
        const uint64_t all = __ballot(good);
        const int n = all == ~uint64_t{0} ? 64 : __ffsll(static_cast<unsigned long long>(~all)) - 1;
        open = n == 64;
        kept += n;
    }
    Weights<T> weight{target + (s * (drafts + 1) + kept) * vocab, nullptr, -1};
    if (kept < count) {
        if (draft != nullptr) weight.q = draft + (s * drafts + kept) * vocab;
        else weight.certain = x[kept];
    }
    const int64_t part = (vocab + kVerifyThreads - 1) / kVerifyThreads * 64;
    const int64_t from = min(wave * part, vocab), to = min(from + part, vocab);
    double total = 0;
    for (int again = 0; again < 2; ++again) {
        double sum = 0;
        for (int64_t j = from + lane; j < to; j += 64) sum += weight(j);
        sum = wave_sum(sum);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        total = 0;
        for (int w = 0; w < kVerifyWaves; ++w) total += sums[w];
        if (total > 0 || (weight.q == nullptr && weight.certain < 0)) break;
        // nothing is left of p - q (or it is NaN): the target's own probabilities
        weight.q = nullptr;
        weight.certain = -1;
        __syncthreads();
    }
    int64_t* out = tokens + s * (drafts + 1);
    for (int64_t i = threadIdx.x; i <= drafts; i += kVerifyThreads)
        if (i != kept) out[i] = i < kept ? x[i] : -1;
    if (threadIdx.x == 0) accepted[s] = kept;
    if (!(total > 0 && total < INFINITY)) {
        if (threadIdx.x == 0) out[kept] = -1;
        return;
    }
    // the wave whose part holds the point: the first whose running sum exceeds it, else the last with any weight
    const double point = u[drafts] * total;
    double before = 0;
    int holder = -1, last = 0;
    double before_holder = 0, before_last = 0;
    for (int w = 0; w < kVerifyWaves; ++w) {
        const double after = before + sums[w];
        if (sums[w] > 0) {
            last = w;
            before_last = before;
        }
        if (holder < 0 && after > point) {
            holder = w;
            before_holder = before;
        }
        before = after;
    }
    if (holder < 0) {
        holder = last;
        before_holder = before_last;
    }
    if (wave != holder) return;
    int64_t picked = -1;
    double run = before_holder;
    for (int64_t j0 = from; j0 < to; j0 += 64) {
        const int64_t j = j0 + lane;
        const double w = j < to ? weight(j) : 0.0;
        double sum = w;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double other = __shfl_up(sum, d);
            if (lane >= d) sum += other;
        }
        const uint64_t over = __ballot(w > 0 && run + sum > point);
        if (over != 0) {
            picked = j0 + __ffsll(static_cast<unsigned long long>(over)) - 1;
            break;
        }
        const uint64_t any = __ballot(w > 0);
        if (any != 0) picked = j0 + 63 - __clzll(static_cast<long long>(any));
        run += __shfl(sum, 63);
    }
    if (lane == 0) out[kept] = picked;
}

// ---- distillation ---------------------------------------------------------------------------------

constexpr int kMaxKept = 1024;
constexpr int kRowThreads = 256;

// The teacher's side of a row, by a whole workgroup: share[j] = pi_j (0 where the entry counts for nothing) and
// log pi_j = (t_j - largest) / T - log_sum. Returns whether the row has any entry.
struct Teacher {
    double largest, log_sum;
    bool any;
};

__device__ __forceinline__ double group_max(double v, double* scratch) {
    for (int m = 32; m > 0; m /= 2) v = max_na(v, __shfl_xor(v, m));
    __syncthreads();
    if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = v;
    __syncthreads();
    for (int w = 0; w < kRowThreads / 64; ++w) v = max_na(v, scratch[w]);
    return v;
}
__device__ __forceinline__ double group_sum(double v, double* scratch) {
    v = wave_sum(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kRowThreads / 64; ++w) v += scratch[w];
    return v;
}

template <typename T>
__device__ Teacher teacher_of(const T* t, const int64_t* index, int64_t cols, int kept, double temperature, double* scratch) {
    double largest = -INFINITY;
    for (int j = threadIdx.x; j < kept; j += kRowThreads)
        if (index[j] >= 0 && index[j] < cols) largest = max_na(largest, static_cast<double>(t[j]));
    largest = group_max(largest, scratch);
    double sum = 0;
    if (largest != -INFINITY)
        for (int j = threadIdx.x; j < kept; j += kRowThreads)
            if (index[j] >= 0 && index[j] < cols) sum += exp((static_cast<double>(t[j]) - largest) / temperature);
    sum = group_sum(sum, scratch);
    return {largest, log(sum), largest != -INFINITY};
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void distill_rows_kernel(T* __restrict__ losses, T* __restrict__ stats,
                                                                   const T* __restrict__ logits, const int64_t* __restrict__ indices,
                                                                   const T* __restrict__ teacher, int64_t cols, int kept,
                                                                   double temperature) {
    __shared__ double scratch[kRowThreads / 64];
    const int64_t row = blockIdx.x;
    const T* z = logits + row * cols;
    T largest = -INFINITY;
    for (int64_t c = threadIdx.x; c < cols; c += kRowThreads) largest = max_na(largest, z[c]);
    largest = static_cast<T>(group_max(static_cast<double>(largest), scratch));
    const T inverse = static_cast<T>(1 / temperature);
    double sum = 0;
    for (int64_t c = threadIdx.x; c < cols; c += kRowThreads) sum += static_cast<double>(std::exp((z[c] - largest) * inverse));
    sum = group_sum(sum, scratch);
    const int64_t* index = indices + row * kept;
    const T* t = teacher + row * kept;
    const Teacher side = teacher_of(t, index, cols, kept, temperature, scratch);
    double loss = 0;
    const double log_total = log(sum);
    if (side.any)
        for (int j = threadIdx.x; j < kept; j += kRowThreads) {
            const int64_t i = index[j];
            if (i < 0 || i >= cols || t[j] == -INFINITY) continue;
            const double log_share = (static_cast<double>(t[j]) - side.largest) / temperature - side.log_sum;
            const double log_student = (static_cast<double>(z[i]) - static_cast<double>(largest)) / temperature - log_total;
            const double share = exp(log_share);
            loss += share == 0 ? 0 : share * (log_share - log_student);
        }
    loss = group_sum(loss, scratch);
    if (threadIdx.x == 0) {
        losses[row] = static_cast<T>(temperature * temperature * loss);
        stats[2 * row] = largest;
        stats[2 * row + 1] = static_cast<T>(sum);
    }
}

template <typename T>
__global__ __launch_bounds__(kRowThreads) void distill_grad_kernel(T* out, const T* logits, const T* __restrict__ stats,
                                                                   const int64_t* __restrict__ indices,
                                                                   const T* __restrict__ teacher, const T* __restrict__ row_weights,
                                                                   int64_t cols, int kept, double temperature) {
    __shared__ double scratch[kRowThreads / 64];
    __shared__ int places[kMaxKept];
    __shared__ T shares[kMaxKept];
    const int64_t row = blockIdx.x;
    const int64_t* index = indices + row * kept;
    const T* t = teacher + row * kept;
    const Teacher side = teacher_of(t, index, cols, kept, temperature, scratch);
    for (int j = threadIdx.x; j < kept; j += kRowThreads) {
        const bool in = side.any && index[j] >= 0 && index[j] < cols;
        places[j] = in ? static_cast<int>(index[j]) : -1;
        shares[j] = in ? static_cast<T>(exp((static_cast<double>(t[j]) - side.largest) / temperature - side.log_sum)) : T(0);
    }
    const T largest = stats[2 * row], inverse = static_cast<T>(1 / temperature);
    const T weight = static_cast<T>(static_cast<double>(row_weights[row]) * temperature);
    const T factor = side.any ? weight / stats[2 * row + 1] : T(0);
    const T* z = logits + row * cols;
    T* g = out + row * cols;
    for (int64_t c = threadIdx.x; c < cols; c += kRowThreads) g[c] = std::exp((z[c] - largest) * inverse) * factor;
    __syncthreads();
    // the first entry of a place takes off the shares of all entries there
    for (int j = threadIdx.x; j < kept; j += kRowThreads) {
        const int place = places[j];
        if (place < 0) continue;
        bool first = true;
        for (int i = 0; i < j; ++i) first = first && places[i] != place;
        if (!first) continue;
        T share = 0;
        for (int i = j; i < kept; ++i) share += places[i] == place ? shares[i] : T(0);
        g[place] -= weight * share;
    }
}

int check_distill(const char* what, int dtype, int64_t rows, int64_t cols, int64_t kept, double temperature) {
    const std::string name(what);
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (rows < 0 || cols < 1 || rows >= (int64_t{1} << 31) || cols >= (int64_t{1} << 31))
        return fail(KD_E_INVALID, name + ": bad number of rows or columns");
    if (kept < 1 || kept > kMaxKept) return fail(KD_E_INVALID, name + ": 1 to 1024 kept entries");
    if (!(temperature > 0) || !std::isfinite(temperature)) return fail(KD_E_INVALID, name + ": temperature must be positive");
    return KD_OK;
}

} // namespace

} // namespace kd

using namespace kd;

extern "C" int kd_verify_drafts(int dtype, int64_t* tokens, int64_t* accepted, const void* target, const void* draft,
                                const int64_t* drafted, const int64_t* counts, const double* uniforms, int64_t sequences,
                                int64_t drafts, int64_t vocab) {
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, "kd_verify_drafts: dtype must be f32 or f64");
    if (sequences < 0 || drafts < 0 || vocab < 1 || sequences >= (int64_t{1} << 31) || drafts >= (int64_t{1} << 20) ||
        vocab >= (int64_t{1} << 31))
        return fail(KD_E_INVALID, "kd_verify_drafts: bad number of sequences, drafts or tokens");
    if (sequences == 0) return KD_OK;
    if (tokens == nullptr || accepted == nullptr || target == nullptr || counts == nullptr || uniforms == nullptr ||
        (drafted == nullptr && drafts > 0))
        return fail(KD_E_INVALID, "kd_verify_drafts: every operand but draft must be given");
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        hipLaunchKernelGGL((verify_drafts_kernel<T>), dim3(static_cast<uint32_t>(sequences)), dim3(kVerifyThreads), 0, stream(),
                           tokens, accepted, static_cast<const T*>(target), static_cast<const T*>(draft), drafted, counts,
                           uniforms, drafts, vocab);
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
        hipLaunchKernelGGL((distill_rows_kernel<T>), dim3(static_cast<uint32_t>(rows)), dim3(kRowThreads), 0, stream(),
                           static_cast<T*>(losses), static_cast<T*>(stats), static_cast<const T*>(logits), indices,
                           static_cast<const T*>(teacher), cols, static_cast<int>(kept), temperature);
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
        hipLaunchKernelGGL((distill_grad_kernel<T>), dim3(static_cast<uint32_t>(rows)), dim3(kRowThreads), 0, stream(),
                           static_cast<T*>(out), static_cast<const T*>(logits), static_cast<const T*>(stats), indices,
                           static_cast<const T*>(teacher), static_cast<const T*>(row_weights), cols, static_cast<int>(kept),
                           temperature);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}
