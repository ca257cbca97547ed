// kd_counter.h - masks from a counter: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011). A block of four words is ten rounds of two 32 x 32 -> 64 bit products over a 128-bit counter; it
// belongs to four neighbouring columns of a row, so a kernel that holds those makes it where it needs it.
#pragma once

#include "kd_internal.h"

namespace kd {

// A kd_counter as the kernels take it, with the border that a kept word does not pass.
struct Mask {
    uint64_t seed;
    const int64_t* more_steps;
    uint32_t row, stream, step, last;  // last: the largest word that is kept
    double scale;                      // 1 / keep

    // The counter's last word: one load, the same for every lane.
    __device__ __forceinline__ uint32_t step_now() const {
        return step + (more_steps != nullptr ? static_cast<uint32_t>(*more_steps) : 0u);
    }
    // Whether columns 4 * block .. + 3 of the row are kept.
    __device__ __forceinline__ void kept(bool (&k)[4], uint32_t row_at, uint32_t block, uint32_t step_at) const {
        uint32_t c0 = block, c1 = row + row_at, c2 = stream, c3 = step_at;
        uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
        for (int turn = 0; turn < 10; ++turn) {
            const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
            c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
            c1 = static_cast<uint32_t>(p1);
            c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
            c3 = static_cast<uint32_t>(p0);
            k0 += 0x9E3779B9u;
            k1 += 0xBB67AE85u;
        }
        k[0] = c0 <= last;
        k[1] = c1 <= last;
        k[2] = c2 <= last;
        k[3] = c3 <= last;
    }
};

// Checks a mask's arguments and fills `mask` for keep < 1; a counter is not read for keep = 1.
inline int mask_of(Mask& mask, const char* what, const kd_counter* counter, double keep, int64_t rows, int64_t cols) {
    const std::string name(what);
    if (!(keep >= 0x1p-32 && keep <= 1.0)) return fail(KD_E_INVALID, name + ": keep must be between 2^-32 and 1");
    mask = {0, nullptr, 0, 0, 0, 0xffffffffu, 1.0};
    if (keep == 1.0) return KD_OK;
    if (counter == nullptr) return fail(KD_E_INVALID, name + ": a mask needs a counter");
    if (counter->row < 0 || counter->row > (int64_t{1} << 32) || rows > (int64_t{1} << 32) - counter->row ||
        cols > (int64_t{1} << 34))
        return fail(KD_E_INVALID, name + ": rows from 2^32 on, or columns from 2^34 on, have no mask");
    if (reinterpret_cast<uintptr_t>(counter->more_steps) % 8 != 0)
        return fail(KD_E_INVALID, name + ": more_steps must be aligned to 8 bytes");
    mask = {counter->seed, counter->more_steps, static_cast<uint32_t>(counter->row), counter->stream, counter->step,
            static_cast<uint32_t>(static_cast<uint64_t>(std::nearbyint(keep * 0x1p32)) - 1), 1.0 / keep};
    return KD_OK;
}

} // namespace kd
