// kd_logits.h - rows of logits as the kernels of kd_drafts.hip and kd_answers.hip read and write them: 16-byte pieces, and workgroups
// by the rows' length.
#pragma once

#include "kd_internal.h"

namespace kd {

constexpr int kMostThreads = 1024;

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

template <typename T> __device__ __forceinline__ T or_zero(T largest) { return largest == -INFINITY ? T(0) : largest; }

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

} // namespace kd
