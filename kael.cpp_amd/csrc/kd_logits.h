// kd_logits.h - rows of logits as the kernels of kd_drafts.hip and kd_answers.hip read and write them: 16-byte pieces, a running
// maximum with its sum of exponentials, workgroups by the rows' length, and what goes past the caches.
#pragma once

#include "kd_internal.h"

namespace kd {

constexpr int kNarrow = 256;        // columns up to which a wave holds a row
constexpr int kNarrowRows = 4;      // rows of such a workgroup
constexpr int kMostThreads = 1024;

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

template <bool Past, typename T> __device__ __forceinline__ void store_piece(T* to, const Piece<T>& p) {
    u32x4 raw;
    __builtin_memcpy(&raw, &p, 16);
    if constexpr (Past) __builtin_nontemporal_store(raw, reinterpret_cast<u32x4*>(to));
    else *reinterpret_cast<u32x4*>(to) = raw;
}

// Threads of a row's workgroup: one wave for short rows, 1024 threads for long ones where there are too few to fill the card
// with 256.
inline int row_threads(int64_t rows, int64_t cols) {
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
inline PastCaches past_caches(int64_t bytes) {
    const bool large = bytes > int64_t{96} << 20, huge = bytes > int64_t{256} << 20;
    return {large && !huge, large, huge};
}

} // namespace kd
