// kd_block.hip - dropout with a mask from a counter, and the end of a transformer's block (a norm of its output, dropout, a
// gate, the residual sum, the norm ahead of the next block) with its backward pass.
#include <algorithm>
#include <iterator>

#include "kd_counter.h"
#include "kd_internal.h"
#include "kd_waves.h"

namespace kd {

namespace {

constexpr int kThreads = 256;

// Four neighbouring elements of a row, whose start is aligned to its elements only; a row's last ones may be fewer.
template <typename T> struct Quad {
    T v[4];
};
template <typename T> __device__ __forceinline__ Quad<T> load_quad(const T* row, int64_t c, int64_t cols) {
    Quad<T> q;
    if (c + 4 <= cols) {
        __builtin_memcpy(&q, row + c, sizeof q);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = c + e < cols ? row[c + e] : T(0);
    }
    return q;
}
template <typename T> __device__ __forceinline__ void store_quad(T* row, int64_t c, int64_t cols, const Quad<T>& q) {
    if (c + 4 <= cols) {
        __builtin_memcpy(row + c, &q, sizeof q);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < cols) row[c + e] = q.v[e];
    }
}

// ---- dropout --------------------------------------------------------------------------------------
//
// A thread takes four columns of a row, the ones that share a block of the counter's words: 20 wide products for 32 bytes moved
// in f32, half of what the vector ALU can do in that time. Bound by the bytes: 16384 x 4096 in f32 97 us, 5.5 TB/s, the rate of a
// copy (vector ALU busy 0.47); 4096 x 256 3.7 us, a launch.

template <typename T>
__global__ __launch_bounds__(kThreads) void counter_dropout_kernel(T* out, const T* in, int64_t rows, int64_t cols, int64_t quads,
                                                                   Mask mask) {
    const uint32_t step = mask.step_now();
    const T scale = static_cast<T>(mask.scale);
    const int64_t total = rows * quads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t row = i / quads, block = i - row * quads;
        Quad<T> q = load_quad(in + row * cols, 4 * block, cols);
        bool k[4];
        mask.kept(k, static_cast<uint32_t>(row), static_cast<uint32_t>(block), step);
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = k[e] ? q.v[e] * scale : T(0);
        store_quad(out + row * cols, 4 * block, cols, q);
    }
}

// ---- the end of a block ---------------------------------------------------------------------------
//
// Bound by the bytes: x and residual read once, h and y written once, from registers in between. A row's arithmetic is f64,
// whose operations cost what f32's do here (packed ones aside); a thread's dropout words are made while its loads are on their
// way. Rows of up to 512 belong to a wave, which needs no barrier, longer ones to a workgroup with one barrier a norm.
// f32, a layer norm with dropout: 4096 x 256 7.2 us, 32768 x 768 79 us, 32768 x 1024 102 us (5.2 TB/s), 8192 x 4096 105 us (5.1 TB/s); RMS norms on
// both sides with a gate: 8192 x 4096 100 to 120 us, vector ALU busy 0.59 of the cycles; one row of 768 2.9 us, 16 rows 3.6 us.

template <typename T> struct NormArgs {
    const T* weight;
    const T* bias;
    double eps;
    int kind;
};

// Mean and 1 / sqrt(mean square + eps) of a row.
struct RowStats {
    double mean, rate;
    __device__ __forceinline__ double unit(double v) const { return (v - mean) * rate; }
};

template <typename T> struct BlockArgs {
    const T* x;
    const T* residual;
    const T* gate;
    int64_t rows, cols, gate_step;  // gate_step: between the gate's rows, 0 for one row
    double residual_scale, block_scale;
    NormArgs<T> after, before;
    Mask mask;
    bool masked;
};

// A team of `threads` threads has a row: each thread the columns 4 * (thread + i * threads) .. + 3 for i < Quads.
struct Pair {
    double a, b;
};
constexpr int kMostWaves = 16;

template <int Quads> struct Team {
    int threads, waves, team, wave, lane;  // wave: its place in the team
    __device__ __forceinline__ explicit Team(int threads_) : threads(threads_), waves(threads_ / 64) {
        const int wave_at = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64);
        team = wave_at / waves;
        wave = wave_at % waves;
        lane = threadIdx.x % 64;
    }
    __device__ __forceinline__ int column(int i) const { return 4 * (wave * 64 + lane + i * threads); }
    // How many of a row's values the team's wave w holds.
    __device__ __forceinline__ int held(int w, int cols) const {
        int n = 0;
#pragma unroll
        for (int i = 0; i < Quads; ++i) n += min(max(cols - 4 * (w * 64 + i * threads), 0), 256);
        return n;
    }
    // Lane w < waves gets wave w's pair; one barrier, so a team's next exchange takes another room.
    __device__ __forceinline__ Pair exchange(Pair own, Pair* room) const {
        if (lane == 0) room[team * waves + wave] = own;
        __syncthreads();
        const int w = lane % kMostWaves;
        return w < waves ? room[team * waves + w] : Pair{0, 0};
    }
    __device__ __forceinline__ Pair sums(double a, double b, Pair* room) const {
        a = wave_total(a);
        b = wave_total(b);
        if (waves == 1) return {a, b};
        const Pair p = exchange({a, b}, room);
        return {from_lane(sum_of_16(p.a), 15), from_lane(sum_of_16(p.b), 15)};
    }
    __device__ __forceinline__ double sum(double a, Pair* room) const {
        a = wave_total(a);
        if (waves == 1) return a;
        return from_lane(sum_of_16(exchange({a, 0}, room).a), 15);
    }
    // A row's statistics from its waves' sums. For a layer norm those are of the distances from one of the wave's own values, the
    // pivot, and of their squares: a value lies within sqrt(n var) of the mean of n, so var from them loses a factor n of the
    // rounding at most, and a row of one value has a var of 0. The waves' means are joined in the same way about wave 0's.
    // of(w): how many values wave w has.
    template <typename F>
    __device__ __forceinline__ RowStats stats(int kind, double eps, int cols, double pivot, double s1, double s2, Pair* room, F of) const {
        const double share = 1.0 / static_cast<double>(cols);
        if (kind == KD_NORM_RMS) return {0.0, rsqrt(sum(s2, room) * share + eps)};
        s1 = wave_total(s1);
        s2 = wave_total(s2);
        const double n = static_cast<double>(of(wave)), by = n > 0 ? s1 / n : 0.0;
        double mean = pivot + by, squares = s2 - s1 * by;
        if (waves > 1) {
            const Pair p = exchange({mean, squares}, room);
            const int w = lane % kMostWaves;
            const double base = from_lane(p.a, 0), count = w < waves ? static_cast<double>(of(w)) : 0.0;
            const double d = count > 0 ? p.a - base : 0.0;
            s1 = from_lane(sum_of_16(count * d), 15);
            s2 = from_lane(sum_of_16((count > 0 ? p.b : 0.0) + count * d * d), 15);
            mean = base + s1 * share;
            squares = s2 - s1 * (s1 * share);
        }
        return {mean, rsqrt((squares < 0 ? 0.0 : squares) * share + eps)};
    }
    template <typename T>
    __device__ __forceinline__ RowStats stats(int kind, double eps, int cols, const Quad<T> (&v)[Quads], Pair* room) const {
        if (kind == KD_NORM_NONE) return {0.0, 1.0};
        const double pivot = kind == KD_NORM_LAYER ? from_lane(static_cast<double>(v[0].v[0]), 0) : 0.0;
        double s1 = 0, s2 = 0;
#pragma unroll
        for (int i = 0; i < Quads; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double d = column(i) + e < cols ? static_cast<double>(v[i].v[e]) - pivot : 0.0;
                s1 += d;
                s2 += d * d;
            }
        return stats(kind, eps, cols, pivot, s1, s2, room, [&](int w) { return held(w, cols); });
    }
};

// Whether a thread's values are kept, a bit each.
template <typename T, int Quads>
__device__ __forceinline__ uint32_t kept_bits(const BlockArgs<T>& a, const Team<Quads>& at, int64_t row, uint32_t step) {
    uint32_t bits = ~0u;
    if (a.masked) {
        bits = 0;
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            bool k[4];
            a.mask.kept(k, static_cast<uint32_t>(row), static_cast<uint32_t>(at.column(i) / 4), step);
#pragma unroll
            for (int e = 0; e < 4; ++e) bits |= (k[e] ? 1u : 0u) << (4 * i + e);
        }
    }
    return bits;
}

// A row's quads for a kernel whose rows are of whole quads, or of any length. A whole quad is loaded without a branch: behind the
// row's end it is the last one again, which nothing counts or stores.
// Offsets in a row are 32 bits without a sign, beside a row's start in scalar registers: one register an address.
template <typename T> __device__ __forceinline__ const T* place_in(const T* row, int c) {
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(T)));
}
template <typename T> __device__ __forceinline__ T* place_in(T* row, int c) {
    return reinterpret_cast<T*>(reinterpret_cast<char*>(row) + static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(T)));
}
template <bool Whole, typename T> __device__ __forceinline__ Quad<T> take_quad(const T* row, int c, int cols) {
    if constexpr (Whole) {
        Quad<T> q;
        __builtin_memcpy(&q, place_in(row, min(c, cols - 4)), sizeof q);
        return q;
    } else {
        return load_quad(place_in(row, c), 0, cols - c);
    }
}
template <bool Whole, typename T> __device__ __forceinline__ Quad<T> quad_or(const T* p, int c, int cols, T otherwise) {
    if (p != nullptr) return take_quad<Whole>(p, c, cols);
    return {otherwise, otherwise, otherwise, otherwise};
}
template <bool Whole, typename T> __device__ __forceinline__ void give_quad(T* row, int c, int cols, const Quad<T>& q) {
    if constexpr (Whole) {
        if (c < cols) __builtin_memcpy(place_in(row, c), &q, sizeof q);
    } else {
        store_quad(place_in(row, c), 0, cols - c, q);
    }
}

// The same past the caches.
template <bool Whole, typename T> __device__ __forceinline__ void give_quad_past(T* row, int c, int cols, const Quad<T>& q) {
    typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (Whole ? c < cols : c + 4 <= cols) {
        Four four;
        __builtin_memcpy(&four, &q, sizeof q);
        __builtin_nontemporal_store(four, reinterpret_cast<Four*>(place_in(row, c)));
    } else if constexpr (!Whole) {
        store_quad(place_in(row, c), 0, cols - c, q);
    }
}

// Keeps the compiler from holding the f64 forms of a loop's f32 constants, twice the registers, all through the loop.
__device__ __forceinline__ void converted_late(Quad<float>& q) {
#pragma unroll
    for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(q.v[e]));
}
__device__ __forceinline__ void converted_late(Quad<double>&) {}

// A row is read once, held in registers and written once. Held: the workgroup takes rows one after another, with the norms'
// weights and the gate in registers all through (from the L2 they are more bytes than the row) and the next row on its way.
// Most: the workgroup's threads at most, all of them a row's, as many waves as the row needs (All: that is all of them, which the
// compiler then knows); 64: a workgroup of four such rows, whose waves leave when they are done and so may not meet at barriers.
template <typename T, int Most, int Quads, bool Whole, bool Held, bool All>
__global__ __launch_bounds__(Most == 64 ? 256 : Most) void block_rows_kernel(T* h, T* y, double* stats, BlockArgs<T> a) {
    constexpr int kTeams = Most == 64 ? 4 : 1;
    __shared__ Pair room[2][2][kMostWaves];  // by turns: a row's waves may be ahead of the last ones of the row before
    const Team<Quads> at(All ? Most : blockDim.x);
    const int cols = static_cast<int>(a.cols);
    const uint32_t step = a.mask.step_now();
    Quad<T> after_w[Quads], after_b[Quads], before_w[Quads], before_b[Quads], gate[Quads];
    const auto load_after = [&](int i, int64_t row) {
        after_w[i] = quad_or<Whole>(a.after.weight, at.column(i), cols, T(1));
        after_b[i] = quad_or<Whole>(a.after.bias, at.column(i), cols, T(0));
        gate[i] = quad_or<Whole>(a.gate != nullptr ? a.gate + row * a.gate_step : nullptr, at.column(i), cols, T(1));
    };
    const auto load_before = [&](int i) {
        before_w[i] = quad_or<Whole>(a.before.weight, at.column(i), cols, T(1));
        before_b[i] = quad_or<Whole>(a.before.bias, at.column(i), cols, T(0));
    };
    if constexpr (Held)
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            load_after(i, 0);
            load_before(i);
        }
    Quad<T> next_v[Quads], next_r[Quads];
    const auto load_row = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            next_v[i] = take_quad<Whole>(a.x + row * a.cols, at.column(i), cols);
            next_r[i] = quad_or<Whole>(a.residual != nullptr ? a.residual + row * a.cols : nullptr, at.column(i), cols, T(0));
        }
    };
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kTeams;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + at.team;
    if (row >= a.rows) return;
    load_row(row);
    for (int turn = 0; row < a.rows; row += stride, turn ^= 1) {
        const int64_t base = row * a.cols;
        Quad<T> v[Quads], r[Quads];
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            v[i] = next_v[i];
            r[i] = next_r[i];
        }
        if constexpr (Held) {
            if (row + stride < a.rows) load_row(row + stride);
#pragma unroll
            for (int i = 0; i < Quads; ++i) {
                converted_late(after_w[i]);
                converted_late(after_b[i]);
                converted_late(before_w[i]);
                converted_late(before_b[i]);
                converted_late(gate[i]);
                if (a.gate_step != 0) gate[i] = take_quad<Whole>(a.gate + row * a.gate_step, at.column(i), cols);
            }
        }
        const uint32_t bits = kept_bits(a, at, row, step);
        const RowStats after = at.stats(a.after.kind, a.after.eps, cols, v, room[turn][0]);
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            const int c = at.column(i);
            if constexpr (!Held) load_after(i, row);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                double n = static_cast<double>(v[i].v[e]);
                if (a.after.kind != KD_NORM_NONE)
                    n = after.unit(n) * static_cast<double>(after_w[i].v[e]) + static_cast<double>(after_b[i].v[e]);
                n = bits >> (4 * i + e) & 1 ? n * a.mask.scale : 0.0;
                v[i].v[e] = static_cast<T>(a.block_scale * static_cast<double>(gate[i].v[e]) * n +
                                           a.residual_scale * static_cast<double>(r[i].v[e]));
            }
            if (h != nullptr) give_quad<Whole>(h + base, c, cols, v[i]);
        }
        RowStats before{0.0, 1.0};
        if (a.before.kind != KD_NORM_NONE && (y != nullptr || stats != nullptr)) {
            before = at.stats(a.before.kind, a.before.eps, cols, v, room[turn][1]);
            if (y != nullptr)
#pragma unroll
                for (int i = 0; i < Quads; ++i) {
                    const int c = at.column(i);
                    if constexpr (!Held) load_before(i);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[i].v[e] = static_cast<T>(before.unit(static_cast<double>(v[i].v[e])) * static_cast<double>(before_w[i].v[e]) +
                                                   static_cast<double>(before_b[i].v[e]));
                    give_quad<Whole>(y + base, c, cols, v[i]);
                }
        }
        if (stats != nullptr && at.wave == 0 && at.lane == 0) {
            stats[4 * row] = after.mean;
            stats[4 * row + 1] = after.rate;
            stats[4 * row + 2] = before.mean;
            stats[4 * row + 3] = before.rate;
        }
        if constexpr (!Held) break;
    }
}

// Any row length, and more rows than a launch of a workgroup for each can have: a workgroup reads a row again in each pass, from the
// caches for the most part. 1500 x 20000 with both norms and a gate 208 to 220 us (2.2 to 2.3 TB/s of what the call has to move), one row
// of 20000 24 us.
constexpr int kWideThreads = 1024, kWideStep = 4 * kWideThreads;

// How many values of a row of any length a wave of such a workgroup has.
__device__ __forceinline__ int wide_held(int wave, int cols) {
    return cols / kWideStep * 256 + min(max(cols % kWideStep - 256 * wave, 0), 256);
}
// A row's statistics, from quads that `value(c)` gives.
template <typename F>
__device__ __forceinline__ RowStats wide_stats(int kind, double eps, int cols, const Team<1>& at, Pair* room, F value) {
    if (kind == KD_NORM_NONE) return {0.0, 1.0};
    double pivot = 0, s1 = 0, s2 = 0;
    for (int c = at.column(0); c < cols; c += kWideStep) {
        const auto q = value(c);
        if (kind == KD_NORM_LAYER && c == at.column(0)) pivot = from_lane(static_cast<double>(q.v[0]), 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double d = c + e < cols ? static_cast<double>(q.v[e]) - pivot : 0.0;
            s1 += d;
            s2 += d * d;
        }
    }
    return at.stats(kind, eps, cols, pivot, s1, s2, room, [&](int w) { return wide_held(w, cols); });
}

// Four values of x after their norm, and whether dropout keeps them.
struct Branch {
    double u[4], n[4];
    bool kept[4];
};
template <typename T>
__device__ __forceinline__ Branch branch_at(const BlockArgs<T>& a, const RowStats& s, int64_t row, int c, int cols, uint32_t step, bool x_read) {
    Branch b{{}, {}, {true, true, true, true}};
    if (a.masked) a.mask.kept(b.kept, static_cast<uint32_t>(row), static_cast<uint32_t>(c / 4), step);
    if (!x_read) return b;
    const Quad<T> x = take_quad<false>(a.x + row * a.cols, c, cols);
    const Quad<T> w = quad_or<false>(a.after.weight, c, cols, T(1)), bias = quad_or<false>(a.after.bias, c, cols, T(0));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        b.u[e] = s.unit(static_cast<double>(x.v[e]));
        b.n[e] = a.after.kind != KD_NORM_NONE ? b.u[e] * static_cast<double>(w.v[e]) + static_cast<double>(bias.v[e]) : b.u[e];
    }
    return b;
}
template <typename T> __device__ __forceinline__ Quad<T> gate_at(const BlockArgs<T>& a, int64_t row, int c, int cols) {
    return quad_or<false>(a.gate != nullptr ? a.gate + row * a.gate_step : nullptr, c, cols, T(1));
}

template <typename T>
__global__ __launch_bounds__(kWideThreads) void block_rows_wide_kernel(T* h, T* y, double* stats, BlockArgs<T> a) {
    __shared__ Pair room[2][2][kMostWaves];
    const Team<1> at(kWideThreads);
    const uint32_t step = a.mask.step_now();
    const int cols = static_cast<int>(a.cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const int64_t base = row * a.cols;
        const RowStats after = wide_stats(a.after.kind, a.after.eps, cols, at, room[turn][0],
                                          [&](int c) { return take_quad<false>(a.x + base, c, cols); });
        const auto sum = [&](int c) {
            const Branch b = branch_at(a, after, row, c, cols, step, true);
            const Quad<T> gate = gate_at(a, row, c, cols), r = quad_or<false>(a.residual != nullptr ? a.residual + base : nullptr, c, cols, T(0));
            Quad<T> q;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                q.v[e] = static_cast<T>(a.block_scale * static_cast<double>(gate.v[e]) * (b.kept[e] ? b.n[e] * a.mask.scale : 0.0) +
                                        a.residual_scale * static_cast<double>(r.v[e]));
            return q;
        };
        // h may take x's or the residual's place, so from then on it is read there; each thread reads what it has written
        if (h != nullptr)
            for (int c = at.column(0); c < cols; c += kWideStep) give_quad<false>(h + base, c, cols, sum(c));
        const auto h_at = [&](int c) { return h != nullptr ? take_quad<false>(h + base, c, cols) : sum(c); };
        RowStats before{0.0, 1.0};
        if (a.before.kind != KD_NORM_NONE && (y != nullptr || stats != nullptr)) {
            before = wide_stats(a.before.kind, a.before.eps, cols, at, room[turn][1], h_at);
            if (y != nullptr)
                for (int c = at.column(0); c < cols; c += kWideStep) {
                    Quad<T> q = h_at(c);
                    const Quad<T> w = quad_or<false>(a.before.weight, c, cols, T(1)), b = quad_or<false>(a.before.bias, c, cols, T(0));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        q.v[e] = static_cast<T>(before.unit(static_cast<double>(q.v[e])) * static_cast<double>(w.v[e]) + static_cast<double>(b.v[e]));
                    give_quad<false>(y + base, c, cols, q);
                }
        }
        if (stats != nullptr && threadIdx.x == 0) {
            stats[4 * row] = after.mean;
            stats[4 * row + 1] = after.rate;
            stats[4 * row + 2] = before.mean;
            stats[4 * row + 3] = before.rate;
        }
    }
}

// ---- its backward pass ----------------------------------------------------------------------------
//
// With v the standardized rows of h, u those of x, w the norms' weights: p = grad_y w, G = grad_h + rate (p - mean p -
// v mean(p v)), d = block_scale gate G dropout, q = d w, grad_x = rate (q - mean q - u mean(q u)); the means without v and u
// only for KD_NORM_LAYER. Summed over the rows: grad_y v, grad_y, d u, d, and block_scale a G for one row of gate.
//
// Bound by the bytes: x, h, grad_h and grad_y read once, two gradients written once, where a team's registers hold a row and LDS its
// sums: rows of up to 4096. The parts' sums are 5 % more where each team has many rows, and a second kernel adds them in order, so that no
// result depends on what runs first. f32: 8192 x 4096, both norms and a gate, 170 to 217 + 6 us (805 MB at 3.7 to 4.7 TB/s, vector ALU busy
// 0.70); a layer norm alone 148 + 5; 32768 x 1024 160 + 5; 4096 x 256 10.5 + 3.8, where it is a chain of launch, loads and two
// exchanges. With all sums the row's kernel and the sums' take 204 to 217 + 97 to 106 us for 4096 x 8192, 311 to 332 + 129 to 147 for 8192 x 5120.

enum Sum { kAfterWeight, kAfterBias, kBeforeWeight, kBeforeBias, kGate, kSums };

template <typename T> struct BackArgs {
    BlockArgs<T> b;
    const T* h;
    const double* stats;
    const T* grad_h;
    const T* grad_y;  // NULL: nothing comes through the second norm
    T* x;
    T* residual;
    T* gate;          // a row for each row
    T* sums[kSums];

    __device__ __forceinline__ RowStats after(int64_t row) const { return {stats[4 * row], stats[4 * row + 1]}; }
    __device__ __forceinline__ RowStats before(int64_t row) const { return {stats[4 * row + 2], stats[4 * row + 3]}; }
};

// Any row length: the gradients of the rows, a workgroup each, and the means of p and p v, [rows][2], for the sums over rows.
template <typename T> __global__ __launch_bounds__(kWideThreads) void block_back_wide_kernel(double* means, BackArgs<T> a) {
    __shared__ Pair room[2][2][kMostWaves];
    const Team<1> at(kWideThreads);
    const uint32_t step = a.b.mask.step_now();
    const int cols = static_cast<int>(a.b.cols);
    const double share = 1.0 / cols;
    const bool normed = a.b.after.kind != KD_NORM_NONE && a.x != nullptr, x_read = normed || a.gate != nullptr;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.b.rows; row += gridDim.x, turn ^= 1) {
        const int64_t base = row * a.b.cols;
        const RowStats before = a.before(row), after = a.after(row);
        double mean = 0, along = 0, back_mean = 0, back_along = 0;
        if (a.grad_y != nullptr) {
            for (int c = at.column(0); c < cols; c += kWideStep) {
                const Quad<T> grad_y = take_quad<false>(a.grad_y + base, c, cols), h = take_quad<false>(a.h + base, c, cols);
                const Quad<T> w = quad_or<false>(a.b.before.weight, c, cols, T(1));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c + e >= cols) continue;
                    const double p = static_cast<double>(grad_y.v[e]) * static_cast<double>(w.v[e]);
                    mean += p;
                    along += p * before.unit(static_cast<double>(h.v[e]));
                }
            }
            const Pair s = at.sums(mean, along, room[turn][0]);
            mean = a.b.before.kind == KD_NORM_LAYER ? s.a * share : 0.0;
            along = s.b * share;
        }
        if (means != nullptr && threadIdx.x == 0) {
            means[2 * row] = mean;
            means[2 * row + 1] = along;
        }
        if (a.x == nullptr && a.residual == nullptr && a.gate == nullptr) continue;
        // G and what it gives of the block's output, for four columns
        const auto through = [&](int c, const Branch& b, double(&g)[4], double(&d)[4]) {
            const Quad<T> grad_h = quad_or<false>(a.grad_h != nullptr ? a.grad_h + base : nullptr, c, cols, T(0));
            const Quad<T> gate = gate_at(a.b, row, c, cols);
            Quad<T> grad_y{}, h{}, w{};
            if (a.grad_y != nullptr) {
                grad_y = take_quad<false>(a.grad_y + base, c, cols);
                h = take_quad<false>(a.h + base, c, cols);
                w = quad_or<false>(a.b.before.weight, c, cols, T(1));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g[e] = static_cast<double>(grad_h.v[e]);
                if (a.grad_y != nullptr)
                    g[e] += before.rate * (static_cast<double>(grad_y.v[e]) * static_cast<double>(w.v[e]) - mean -
                                           before.unit(static_cast<double>(h.v[e])) * along);
                d[e] = b.kept[e] ? a.b.block_scale * static_cast<double>(gate.v[e]) * g[e] * a.b.mask.scale : 0.0;
            }
        };
        if (normed) {
            for (int c = at.column(0); c < cols; c += kWideStep) {
                const Branch b = branch_at(a.b, after, row, c, cols, step, true);
                const Quad<T> w = quad_or<false>(a.b.after.weight, c, cols, T(1));
                double g[4], d[4];
                through(c, b, g, d);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (c + e >= cols) continue;
                    const double q = d[e] * static_cast<double>(w.v[e]);
                    back_mean += q;
                    back_along += q * b.u[e];
                }
            }
            const Pair s = at.sums(back_mean, back_along, room[turn][1]);
            back_mean = a.b.after.kind == KD_NORM_LAYER ? s.a * share : 0.0;
            back_along = s.b * share;
        }
        // outputs may take the place of what is read at the same element
        for (int c = at.column(0); c < cols; c += kWideStep) {
            const Branch b = branch_at(a.b, after, row, c, cols, step, x_read);
            const Quad<T> w = quad_or<false>(a.b.after.weight, c, cols, T(1));
            double g[4], d[4];
            through(c, b, g, d);
            Quad<T> to_x, to_residual, to_gate;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                to_residual.v[e] = static_cast<T>(a.b.residual_scale * g[e]);
                to_gate.v[e] = static_cast<T>(b.kept[e] ? a.b.block_scale * (b.n[e] * a.b.mask.scale) * g[e] : 0.0);
                to_x.v[e] = static_cast<T>(normed ? after.rate * (d[e] * static_cast<double>(w.v[e]) - back_mean - b.u[e] * back_along) : d[e]);
            }
            if (a.residual != nullptr) give_quad<false>(a.residual + base, c, cols, to_residual);
            if (a.gate != nullptr) give_quad<false>(a.gate + base, c, cols, to_gate);
            if (a.x != nullptr) give_quad<false>(a.x + base, c, cols, to_x);
        }
    }
}

// The sums over a segment of rows: [segment][sum][cols]. A workgroup takes 256 columns, four a lane, and its waves share the rows.
// All segments go from the last rows to the first ones, since the last cache may still hold the last ones from the rows' kernel (4096 x 8192,
// both norms and a gate, 122 us from the first row on, 111 so, 104 where the gradients went past the caches as well).
template <typename T, bool Whole>
__global__ __launch_bounds__(kThreads) void block_columns_kernel(T* parts, const double* means, BackArgs<T> a) {
    constexpr int kWaves = kThreads / 64;
    __shared__ double room[kWaves][4][64];
    const uint32_t step = a.b.mask.step_now();
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64);
    const int c = static_cast<int>(blockIdx.x) * 256 + 4 * lane, cols = static_cast<int>(a.b.cols);
    const bool normed = a.b.after.kind != KD_NORM_NONE, gate_sum = a.sums[kGate] != nullptr, x_read = normed || gate_sum;
    const Quad<T> before_w = quad_or<Whole>(a.b.before.weight, c, cols, T(1)), after_w = quad_or<Whole>(a.b.after.weight, c, cols, T(1));
    const Quad<T> after_b = quad_or<Whole>(a.b.after.bias, c, cols, T(0));
    Quad<T> gate = quad_or<Whole>(a.b.gate, c, cols, T(1));
    double sums[kSums][4] = {};
    if (c < cols)
        for (int64_t row = a.b.rows - 1 - (static_cast<int64_t>(wave) * gridDim.y + blockIdx.y); row >= 0;
             row -= static_cast<int64_t>(kWaves) * gridDim.y) {
            const int64_t base = row * a.b.cols;
            const RowStats before = a.before(row), after = a.after(row);
            const double mean = means[2 * row], along = means[2 * row + 1];
            Quad<T> x{}, h{}, grad_y{};
            const Quad<T> grad_h = quad_or<Whole>(a.grad_h != nullptr ? a.grad_h + base : nullptr, c, cols, T(0));
            if (a.grad_y != nullptr) {
                grad_y = take_quad<Whole>(a.grad_y + base, c, cols);
                h = take_quad<Whole>(a.h + base, c, cols);
            }
            if (x_read) x = take_quad<Whole>(a.b.x + base, c, cols);
            if (a.b.gate_step != 0) gate = take_quad<Whole>(a.b.gate + row * a.b.gate_step, c, cols);
            bool kept[4] = {true, true, true, true};
            if (a.b.masked) a.b.mask.kept(kept, static_cast<uint32_t>(row), static_cast<uint32_t>(c / 4), step);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                double g = static_cast<double>(grad_h.v[e]);
                if (a.grad_y != nullptr) {
                    const double own = static_cast<double>(grad_y.v[e]), v = before.unit(static_cast<double>(h.v[e]));
                    g += before.rate * (own * static_cast<double>(before_w.v[e]) - mean - v * along);
                    sums[kBeforeWeight][e] += own * v;
                    sums[kBeforeBias][e] += own;
                }
                const double through = kept[e] ? a.b.block_scale * a.b.mask.scale * g : 0.0;
                const double u = after.unit(static_cast<double>(x.v[e]));
                if (gate_sum)
                    sums[kGate][e] += kept[e] ? through * (normed ? u * static_cast<double>(after_w.v[e]) + static_cast<double>(after_b.v[e]) : u) : 0.0;
                const double d = kept[e] ? through * static_cast<double>(gate.v[e]) : 0.0;
                if (normed) {
                    sums[kAfterWeight][e] += d * u;
                    sums[kAfterBias][e] += d;
                }
            }
        }
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
        if (a.sums[k] == nullptr) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) room[wave][e][lane] = sums[k][e];
        __syncthreads();
        if (wave == 0 && c < cols) {
            Quad<T> q;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                double total = room[0][e][lane];
                for (int w = 1; w < kWaves; ++w) total += room[w][e][lane];
                q.v[e] = static_cast<T>(total);
            }
            give_quad<Whole>(parts + (blockIdx.y * kSums + k) * a.b.cols, c, cols, q);
        }
    }
}

// A long row's gradients, by a workgroup that holds it: what the sums over rows would take of the registers is left to
// block_columns_kernel, which reads the rows again (4096 x 8192: 167 + 80 us for a layer norm; in one kernel, which spilled, 421 to 480).
// Four quads a thread, rows past 8192, spill too: 24 to 34 of the 128 registers that 16 waves may have.
template <typename T, int Quads, bool Whole, bool Past>
__global__ __launch_bounds__(1024) void block_back_row_kernel(double* means, BackArgs<T> a) {
    __shared__ Pair room[2][kMostWaves];
    const Team<Quads> at(blockDim.x);
    const int64_t row = blockIdx.x, base = row * a.b.cols;
    const int cols = static_cast<int>(a.b.cols);
    const double share = 1.0 / cols;
    const auto give = [&](T* out, int c, const Quad<T>& q) {
        if constexpr (Past) give_quad_past<Whole>(out, c, cols, q);
        else give_quad<Whole>(out, c, cols, q);
    };
    const RowStats before = a.before(row), after = a.after(row);
    Quad<T> grad_h[Quads], grad_y[Quads], h[Quads];
    double g[Quads][4], mean = 0, along = 0;
#pragma unroll
    for (int i = 0; i < Quads; ++i) {
        const int c = at.column(i);
        if (a.grad_y != nullptr) {
            grad_y[i] = take_quad<Whole>(a.grad_y + base, c, cols);
            h[i] = take_quad<Whole>(a.h + base, c, cols);
        }
        grad_h[i] = quad_or<Whole>(a.grad_h != nullptr ? a.grad_h + base : nullptr, c, cols, T(0));
    }
    const uint32_t bits = kept_bits(a.b, at, row, a.b.mask.step_now());
    if (a.grad_y != nullptr) {
        double p_sum = 0, pv_sum = 0;
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            const Quad<T> w = quad_or<Whole>(a.b.before.weight, at.column(i), cols, T(1));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (at.column(i) + e >= cols) continue;
                const double p = static_cast<double>(grad_y[i].v[e]) * static_cast<double>(w.v[e]);
                p_sum += p;
                pv_sum += p * before.unit(static_cast<double>(h[i].v[e]));
            }
        }
        const Pair s = at.sums(p_sum, pv_sum, room[0]);
        mean = a.b.before.kind == KD_NORM_LAYER ? s.a * share : 0.0;
        along = s.b * share;
    }
    if (means != nullptr && threadIdx.x == 0) {
        means[2 * row] = mean;
        means[2 * row + 1] = along;
    }
    if (a.x == nullptr && a.residual == nullptr && a.gate == nullptr) return;
    const bool normed = a.b.after.kind != KD_NORM_NONE && a.x != nullptr, x_read = normed || a.gate != nullptr;
    double q_sum = 0, qu_sum = 0;
    Quad<T> x[Quads];
#pragma unroll
    for (int i = 0; i < Quads; ++i) {
        const int c = at.column(i);
        if (x_read) x[i] = take_quad<Whole>(a.b.x + base, c, cols);
        const Quad<T> before_w = quad_or<Whole>(a.b.before.weight, c, cols, T(1)), after_w = quad_or<Whole>(a.b.after.weight, c, cols, T(1));
        const Quad<T> gate = quad_or<Whole>(a.b.gate != nullptr ? a.b.gate + row * a.b.gate_step : nullptr, c, cols, T(1));
        Quad<T> to_residual, to_gate;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            double own = static_cast<double>(grad_h[i].v[e]);
            if (a.grad_y != nullptr)
                own += before.rate * (static_cast<double>(grad_y[i].v[e]) * static_cast<double>(before_w.v[e]) - mean -
                                      before.unit(static_cast<double>(h[i].v[e])) * along);
            to_residual.v[e] = static_cast<T>(a.b.residual_scale * own);
            const double through = bits >> (4 * i + e) & 1 ? a.b.block_scale * a.b.mask.scale * own : 0.0;
            g[i][e] = bits >> (4 * i + e) & 1 ? through * static_cast<double>(gate.v[e]) : 0.0;
            if (x_read) {
                const double u = after.unit(static_cast<double>(x[i].v[e]));
                if (a.gate != nullptr) {
                    const Quad<T> b = quad_or<Whole>(a.b.after.bias, c, cols, T(0));
                    const double n = a.b.after.kind != KD_NORM_NONE ? u * static_cast<double>(after_w.v[e]) + static_cast<double>(b.v[e]) : u;
                    to_gate.v[e] = static_cast<T>(bits >> (4 * i + e) & 1 ? through * n : 0.0);
                }
                if (normed && c + e < cols) {
                    const double q = g[i][e] * static_cast<double>(after_w.v[e]);
                    q_sum += q;
                    qu_sum += q * u;
                }
            }
        }
        if (a.residual != nullptr) give(a.residual + base, c, to_residual);
        if (a.gate != nullptr) give(a.gate + base, c, to_gate);
    }
    if (a.x == nullptr) return;
    double back_mean = 0, back_along = 0;
    if (normed) {
        const Pair s = at.sums(q_sum, qu_sum, room[1]);
        back_mean = a.b.after.kind == KD_NORM_LAYER ? s.a * share : 0.0;
        back_along = s.b * share;
    }
#pragma unroll
    for (int i = 0; i < Quads; ++i) {
        const int c = at.column(i);
        const Quad<T> after_w = quad_or<Whole>(normed ? a.b.after.weight : nullptr, c, cols, T(1));
        Quad<T> to;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            double d = g[i][e];
            if (normed)
                d = after.rate * (d * static_cast<double>(after_w.v[e]) - back_mean - after.unit(static_cast<double>(x[i].v[e])) * back_along);
            to.v[e] = static_cast<T>(d);
        }
        give(a.x + base, c, to);
    }
}

// A team's rows one after another, each read once: the rows' gradients and the sums over the team's rows. Those lie in LDS,
// [team][wanted sum][cols up to a quad], where each thread adds to the places of its own columns: in registers they took 20 a
// quad (40 in f64), and the row spilled. Held: the norms' weights and the gate stay in registers, and a row is loaded while
// the one before it is worked on. One workgroup a CU: 128 registers a lane for its 16 waves in f32; f64 takes 8 waves, which may have
// 195 each (two workgroups of 128 that read the weights anew: 8192 x 2048 246 us instead of 176).
template <typename T> constexpr int kBackThreads = std::is_same_v<T, float> ? 1024 : 512;

struct SumPlaces {
    int at[kSums];  // a sum's place in LDS, -1 if it is not wanted
    int wanted;
};
template <typename T> __device__ __forceinline__ void add_quad(T* place, const Quad<T>& q) {
    Quad<T> own;
    T* p = static_cast<T*>(__builtin_assume_aligned(place, 16));
    __builtin_memcpy(&own, p, sizeof own);
#pragma unroll
    for (int e = 0; e < 4; ++e) own.v[e] += q.v[e];
    __builtin_memcpy(p, &own, sizeof own);
}

// A quad of a row of any length without a branch: one behind the row's end, or over it, is loaded from the last four values, and `settled`
// moves them to their places once they are there. What is in the other places nothing counts or stores.
template <typename T> __device__ __forceinline__ Quad<T> raw_quad(const T* row, int c, int cols) {
    Quad<T> q;
    if (cols >= 4) {
        __builtin_memcpy(&q, place_in(row, min(c, cols - 4)), sizeof q);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = row[min(c + e, cols - 1)];
    }
    return q;
}
template <typename T> __device__ __forceinline__ void settled(Quad<T>& q, int c, int cols) {
    const int by = cols < 4 ? 0 : c - min(c, cols - 4);
    const bool one = by & 1, two = by & 2;
    const T v0 = one ? q.v[1] : q.v[0], v1 = one ? q.v[2] : q.v[1], v2 = one ? q.v[3] : q.v[2];
    q = {two ? v2 : v0, two ? q.v[3] : v1, v2, q.v[3]};
}

// kLate: f64 rows that are not of whole quads, whose quads are two loads each (6610 x 454 57 us with branches, 47 without; in f32 the
// moves cost more than the branches, 7000 x 4095 174 and 192).
template <typename T, int Quads, bool Whole> struct BackRow {
    static constexpr bool kLate = !Whole && sizeof(T) == 8;
    __device__ __forceinline__ static Quad<T> take(const T* row, int c, int cols) {
        if constexpr (kLate) return raw_quad(row, c, cols);
        else return take_quad<Whole>(row, c, cols);
    }
    Quad<T> x[Quads], h[Quads], grad_h[Quads], grad_y[Quads];
    RowStats after, before;
    __device__ __forceinline__ void load(const BackArgs<T>& a, const Team<Quads>& at, int64_t row, bool x_read) {
        const int64_t base = row * a.b.cols;
        const int cols = static_cast<int>(a.b.cols);
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            const int c = at.column(i);
            if (x_read) x[i] = take(a.b.x + base, c, cols);
            if (a.grad_y != nullptr) {
                h[i] = take(a.h + base, c, cols);
                grad_y[i] = take(a.grad_y + base, c, cols);
            }
            if (a.grad_h != nullptr) grad_h[i] = take(a.grad_h + base, c, cols);
            else grad_h[i] = {};
        }
        // the same for a wave's lanes and constant in this kernel: scalar loads to scalar registers
        const auto* s = (const __attribute__((address_space(4))) double*)(a.stats + 4 * row);
        after = {s[0], s[1]};
        before = {s[2], s[3]};
    }
    __device__ __forceinline__ void settle(const Team<Quads>& at, int cols) {
        if constexpr (kLate)
#pragma unroll
            for (int i = 0; i < Quads; ++i) {
                settled(x[i], at.column(i), cols);
                settled(h[i], at.column(i), cols);
                settled(grad_h[i], at.column(i), cols);
                settled(grad_y[i], at.column(i), cols);
            }
    }
    __device__ __forceinline__ void converted_late() {
#pragma unroll
        for (int i = 0; i < Quads; ++i) {
            kd::converted_late(x[i]);
            kd::converted_late(h[i]);
            kd::converted_late(grad_h[i]);
            kd::converted_late(grad_y[i]);
        }
    }
};

// Threads: a team's, 0: as many as are given.
template <typename T, int Threads, int Quads, bool Held, bool Whole>
__global__ __launch_bounds__(kBackThreads<T>) void block_back_kernel(T* parts, BackArgs<T> a, int threads, int64_t rows_per_team, SumPlaces places) {
    extern __shared__ __attribute__((aligned(16))) char shared[];
    __shared__ Pair room[2][2][kMostWaves];  // by turns: a row's waves may be ahead of the last ones of the row before
    const Team<Quads> at(Threads != 0 ? Threads : threads);
    const int group = Threads != 0 ? kBackThreads<T> : static_cast<int>(blockDim.x), teams = group / at.threads;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * teams + at.team) * rows_per_team, end = min(a.b.rows, first + rows_per_team);
    const int cols = static_cast<int>(a.b.cols);
    const double share = 1.0 / cols;
    const uint32_t step = a.b.mask.step_now();
    const bool normed = a.b.after.kind != KD_NORM_NONE, gate_sum = a.sums[kGate] != nullptr;
    const bool branch = gate_sum || a.gate != nullptr, x_read = normed || branch;
    Quad<T> before_w[Quads], after_w[Quads], after_b[Quads], gate[Quads];
    const auto load_weights = [&](int i, int64_t row) {
        const int c = at.column(i);
        before_w[i] = quad_or<Whole>(a.b.before.weight, c, cols, T(1));
        after_w[i] = quad_or<Whole>(a.b.after.weight, c, cols, T(1));
        after_b[i] = quad_or<Whole>(branch ? a.b.after.bias : nullptr, c, cols, T(0));
        gate[i] = quad_or<Whole>(a.b.gate != nullptr ? a.b.gate + row * a.b.gate_step : nullptr, c, cols, T(1));
    };
    if constexpr (Held)
#pragma unroll
        for (int i = 0; i < Quads; ++i) load_weights(i, 0);
    const int padded = (cols + 3) & ~3;
    T* sums = reinterpret_cast<T*>(shared) + at.team * places.wanted * padded;
    const auto sum_place = [&](Sum k, int c) { return sums + places.at[k] * padded + c; };
    for (int k = 0; k < places.wanted; ++k)
#pragma unroll
        for (int i = 0; i < Quads; ++i)
            if (at.column(i) < cols) __builtin_memset(sums + k * padded + at.column(i), 0, 4 * sizeof(T));
    BackRow<T, Quads, Whole> now, next;
    if (Held && first < end) next.load(a, at, first, x_read);
    for (int64_t n = 0; n < rows_per_team; ++n) {
        const int64_t row = first + n, base = row * a.b.cols;
        const bool here = row < end;  // the same for all threads of a team; the teams meet at the barriers
        if constexpr (Held) {
            now = next;
            if (row + 1 < end) next.load(a, at, row + 1, x_read);
        } else if (here) {
            now.load(a, at, row, x_read);
        }
        if constexpr (Held) {
#pragma unroll
            for (int i = 0; i < Quads; ++i) {
                converted_late(before_w[i]);
                converted_late(after_w[i]);
                converted_late(after_b[i]);
                converted_late(gate[i]);
            }
        }
        double p_sum = 0, pv_sum = 0;
        uint32_t bits = 0;
        if (here) {
            bits = kept_bits(a.b, at, row, step);
            now.settle(at, cols);
            if (a.grad_y != nullptr) {
#pragma unroll
                for (int i = 0; i < Quads; ++i) {
                    Quad<T> by_weight;
                    if constexpr (!Held) before_w[i] = quad_or<Whole>(a.b.before.weight, at.column(i), cols, T(1));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const double g = static_cast<double>(now.grad_y[i].v[e]), p = g * static_cast<double>(before_w[i].v[e]);
                        const double v = now.before.unit(static_cast<double>(now.h[i].v[e]));
                        if (at.column(i) + e < cols) {
                            p_sum += p;
                            pv_sum += p * v;
                        }
                        by_weight.v[e] = static_cast<T>(g * v);
                    }
                    if (at.column(i) < cols) {
                        if (places.at[kBeforeWeight] >= 0) add_quad(sum_place(kBeforeWeight, at.column(i)), by_weight);
                        if (places.at[kBeforeBias] >= 0) add_quad(sum_place(kBeforeBias, at.column(i)), now.grad_y[i]);
                    }
                }
            }
        }
        double mean = 0, along = 0;
        if (a.grad_y != nullptr) {
            if (a.b.before.kind == KD_NORM_LAYER) {
                const Pair s = at.sums(p_sum, pv_sum, room[n & 1][0]);
                mean = s.a * share;
                along = s.b * share;
            } else {
                along = at.sum(pv_sum, room[n & 1][0]) * share;
            }
        }
        double q_sum = 0, qu_sum = 0, d[Quads][4];
        if (here) {
            now.converted_late();
#pragma unroll
            for (int i = 0; i < Quads; ++i) {
                const int c = at.column(i);
                if constexpr (!Held) load_weights(i, row);
                else if (a.b.gate_step != 0) gate[i] = take_quad<Whole>(a.b.gate + row * a.b.gate_step, c, cols);
                Quad<T> to_residual, to_gate, by_weight, by_bias;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    double g = static_cast<double>(now.grad_h[i].v[e]);
                    if (a.grad_y != nullptr)
                        g += now.before.rate * (static_cast<double>(now.grad_y[i].v[e]) * static_cast<double>(before_w[i].v[e]) - mean -
                                                now.before.unit(static_cast<double>(now.h[i].v[e])) * along);
                    to_residual.v[e] = static_cast<T>(a.b.residual_scale * g);
                    const bool kept = bits >> (4 * i + e) & 1;
                    d[i][e] = kept ? a.b.block_scale * static_cast<double>(gate[i].v[e]) * g * a.b.mask.scale : 0.0;
                    double u = 0;
                    if (x_read) u = now.after.unit(static_cast<double>(now.x[i].v[e]));
                    if (branch) {
                        const double b = normed ? u * static_cast<double>(after_w[i].v[e]) + static_cast<double>(after_b[i].v[e]) : u;
                        const double own = kept ? a.b.block_scale * (b * a.b.mask.scale) * g : 0.0;
                        to_gate.v[e] = static_cast<T>(own);
                    }
                    if (normed && c + e < cols) {
                        by_weight.v[e] = static_cast<T>(d[i][e] * u);
                        by_bias.v[e] = static_cast<T>(d[i][e]);
                        const double q = d[i][e] * static_cast<double>(after_w[i].v[e]);
                        q_sum += q;
                        qu_sum += q * u;
                    }
                }
                if (c < cols) {
                    if (places.at[kAfterWeight] >= 0) add_quad(sum_place(kAfterWeight, c), by_weight);
                    if (places.at[kAfterBias] >= 0) add_quad(sum_place(kAfterBias, c), by_bias);
                    if (gate_sum) add_quad(sum_place(kGate, c), to_gate);
                }
                if (a.residual != nullptr) give_quad<Whole>(a.residual + base, c, cols, to_residual);
                if (a.gate != nullptr) give_quad<Whole>(a.gate + base, c, cols, to_gate);
            }
        }
        if (normed) {
            if (a.b.after.kind == KD_NORM_LAYER) {
                const Pair s = at.sums(q_sum, qu_sum, room[n & 1][1]);
                mean = s.a * share;
                along = s.b * share;
            } else {
                mean = 0;
                along = at.sum(qu_sum, room[n & 1][1]) * share;
            }
        }
        if (here && a.x != nullptr) {
            now.converted_late();
#pragma unroll
            for (int i = 0; i < Quads; ++i) {
                Quad<T> to;
                if constexpr (!Held) after_w[i] = quad_or<Whole>(a.b.after.weight, at.column(i), cols, T(1));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    double g = d[i][e];
                    if (normed)
                        g = now.after.rate * (g * static_cast<double>(after_w[i].v[e]) - mean -
                                              now.after.unit(static_cast<double>(now.x[i].v[e])) * along);
                    to.v[e] = static_cast<T>(g);
                }
                give_quad<Whole>(a.x + base, at.column(i), cols, to);
            }
        }
    }
    // the teams' sums in order
    __syncthreads();
    for (int k = 0; k < kSums; ++k) {
        if (places.at[k] < 0) continue;
        T* out = parts + (static_cast<int64_t>(blockIdx.x) * kSums + k) * cols;
        const T* own = reinterpret_cast<const T*>(shared) + places.at[k] * padded;
        for (int c = threadIdx.x; c < cols; c += group) {
            double total = static_cast<double>(own[c]);
            for (int t = 1; t < teams; ++t) total += static_cast<double>(own[t * places.wanted * padded + c]);
            out[c] = static_cast<T>(total);
        }
    }
}

// The segments' sums in order: a workgroup takes 64 columns of one sum, its 16 waves a run of segments each.
constexpr int kJoinWaves = 16;
template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void block_join_kernel(BackArgs<T> a, const T* parts, int64_t segments) {
    __shared__ double room[kJoinWaves][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    T* out = a.sums[blockIdx.y];
    if (out == nullptr) return;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane, cols = a.b.cols;
    const int64_t run = (segments + kJoinWaves - 1) / kJoinWaves, end = min(segments, (wave + 1) * run);
    double sum = 0;
    if (c < cols) {
        const T* own = parts + blockIdx.y * cols + c;
        int64_t at = wave * run;
        for (; at + 8 <= end; at += 8) {  // eight loads in flight
            T part[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) part[i] = own[(at + i) * kSums * cols];
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += static_cast<double>(part[i]);
        }
        for (; at < end; ++at) sum += static_cast<double>(own[at * kSums * cols]);
    }
    room[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || c >= cols) return;
    for (int w = 1; w < kJoinWaves; ++w) sum += room[w][lane];
    out[c] = static_cast<T>(sum);
}

// ---- plans and checks -----------------------------------------------------------------------------

template <int N> using Int = std::integral_constant<int, N>;

// How a backward pass is divided. threads: a row's team, 0 for rows that registers do not hold; teams: of a workgroup; segments:
// parts of the rows whose sums are kept apart.
struct BackPlan {
    int threads, quads;
    int64_t teams, rows_per_team, segments;
    int64_t most;  // segments that no smaller number of rows passes, so that a workspace serves those too
};
// Threads of a team that holds a row in `quads` quads a thread: as many waves as that takes, so that none is idle (32768 x 768 176 us in teams of
// four waves, three of them at work, 158 in teams of three; 20000 x 1280 207 and 150).
int team_threads(int64_t cols, int quads) { return static_cast<int>((cols + 256 * quads - 1) / (256 * quads) * 64); }
int most_threads(int dtype) { return dtype == KD_F32 ? kBackThreads<float> : kBackThreads<double>; }
// Bytes of LDS that `wanted` sums take for `teams`.
int64_t sums_bytes(int dtype, int64_t cols, int64_t teams, int wanted) { return teams * wanted * ((cols + 3) / 4 * 4) * dtype_size(dtype); }
BackPlan wide_plan(int64_t rows, int64_t cols) {
    // Workgroups of 256 columns, of 16 rows at least, and four for each CU at most, as many as it has at once: with one round more of a few
    // of them, a layer norm alone / both norms and a gate, 8192 x 5120 took 162 / 205 us instead of 106 / 138, 2000 x 20000 174 / 216
    // instead of 112 / 138.
    const int64_t wanted = int64_t{4} * compute_units() / ((cols + 255) / 256);
    const int64_t segments = std::clamp<int64_t>(wanted, 1, (rows + 15) / 16);
    return {0, 0, 0, 0, segments, segments};
}
BackPlan back_plan(int dtype, int64_t rows, int64_t cols, int wanted) {
    if (cols > 4096) return wide_plan(rows, cols);
    const int quads = cols <= 4 * most_threads(dtype) ? 1 : 2, threads = team_threads(cols, quads);
    const int64_t teams = most_threads(dtype) / threads;
    if (sums_bytes(dtype, cols, teams, wanted) > 159 * 1024) return wide_plan(rows, cols);
    const int64_t all = teams * compute_units();
    // a CU has one workgroup at a time: as few rounds as parts of 32 rows allow, all of them full
    const int64_t rounds = (rows + 32 * all - 1) / (32 * all), each = (rows + rounds * all - 1) / (rounds * all);
    return {threads, quads, teams, each, (rows + teams * each - 1) / (teams * each),
            std::min(rounds * compute_units(), (rows + teams - 1) / teams)};
}
// What the passes of any number of sums need at most.
int64_t room_of(int dtype, int64_t rows, int64_t cols) {
    if (rows == 0 || cols == 0) return 0;
    int64_t most = 0;
    for (int wanted = 1; wanted <= kSums; ++wanted) {
        const BackPlan plan = back_plan(dtype, rows, cols, wanted);
        most = std::max(most, (plan.threads == 0 ? rows * 16 : 0) + plan.most * kSums * cols * dtype_size(dtype));
    }
    return most;
}

constexpr int64_t kMostCols = int64_t{1} << 28;  // offsets in a row are 32 bits
bool fits(int64_t rows, int64_t cols) { return rows <= (int64_t{1} << 40) && cols <= (int64_t{1} << 40) && (cols == 0 || rows <= (int64_t{1} << 46) / cols); }

template <typename T> NormArgs<T> norm_of(const kd_norm& n) {
    if (n.kind == KD_NORM_NONE) return {nullptr, nullptr, 0.0, KD_NORM_NONE};
    return {static_cast<const T*>(n.weight), static_cast<const T*>(n.bias), n.eps, n.kind};
}

template <typename T> BlockArgs<T> args_of(const kd_block& b, const Mask& mask) {
    BlockArgs<T> a;
    a.x = static_cast<const T*>(b.x);
    a.residual = static_cast<const T*>(b.residual);
    a.gate = static_cast<const T*>(b.gate);
    a.rows = b.rows;
    a.cols = b.cols;
    a.gate_step = b.gate_rows == b.rows && b.gate_rows != 1 ? b.cols : 0;
    a.residual_scale = b.residual_scale;
    a.block_scale = b.block_scale;
    a.after = norm_of<T>(b.after);
    a.before = norm_of<T>(b.before);
    a.mask = mask;
    a.masked = b.keep < 1.0;
    return a;
}

int check_block(const char* what, int dtype, const kd_block* b, Mask& mask) {
    const std::string name(what);
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (b == nullptr) return fail(KD_E_INVALID, name + ": the block must be given");
    if (b->rows < 0 || b->cols < 0 || b->cols > kMostCols || !fits(b->rows, b->cols)) return fail(KD_E_INVALID, name + ": bad number of rows or columns");
    for (const kd_norm* n : {&b->after, &b->before}) {
        if (n->kind != KD_NORM_NONE && n->kind != KD_NORM_LAYER && n->kind != KD_NORM_RMS)
            return fail(KD_E_INVALID, name + ": no such norm");
        if (n->kind != KD_NORM_NONE && !(n->eps >= 0 && n->eps < INFINITY))
            return fail(KD_E_INVALID, name + ": eps must be finite and not negative");
    }
    if (!std::isfinite(b->residual_scale) || !std::isfinite(b->block_scale))
        return fail(KD_E_INVALID, name + ": the scales must be finite");
    if (b->gate != nullptr ? b->gate_rows != 1 && b->gate_rows != b->rows : b->gate_rows != 0)
        return fail(KD_E_INVALID, name + ": gate_rows is 1 or rows with a gate, 0 without one");
    return mask_of(mask, what, &b->counter, b->keep, b->rows, b->cols);
}

} // namespace

} // namespace kd

using namespace kd;

extern "C" int kd_counter_dropout(int dtype, void* out, const void* in, int64_t rows, int64_t cols, double keep,
                                  const kd_counter* counter) {
    const char* what = "kd_counter_dropout";
    const std::string name(what);
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (rows < 0 || cols < 0 || !fits(rows, cols)) return fail(KD_E_INVALID, name + ": bad number of rows or columns");
    Mask mask;
    if (int rc = mask_of(mask, what, counter, keep, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return KD_OK;
    if (out == nullptr || in == nullptr) return fail(KD_E_INVALID, name + ": in and out must be given");
    const int64_t bytes = rows * cols * dtype_size(dtype);
    if (out != in && overlap(out, bytes, in, bytes)) return fail(KD_E_INVALID, name + ": out overlaps in");
    if (overlap(out, bytes, mask.more_steps, 8)) return fail(KD_E_INVALID, name + ": out overlaps more_steps");
    if (int rc = ensure_device()) return rc;
    const int64_t quads = (cols + 3) / 4;
    const uint32_t groups = static_cast<uint32_t>(
        std::min<int64_t>((rows * quads + kThreads - 1) / kThreads, int64_t{compute_units()} * 32));
    if (dtype == KD_F32)
        hipLaunchKernelGGL((counter_dropout_kernel<float>), dim3(groups), dim3(kThreads), 0, stream(), static_cast<float*>(out),
                           static_cast<const float*>(in), rows, cols, quads, mask);
    else
        hipLaunchKernelGGL((counter_dropout_kernel<double>), dim3(groups), dim3(kThreads), 0, stream(), static_cast<double*>(out),
                           static_cast<const double*>(in), rows, cols, quads, mask);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_block_rows(int dtype, void* h, void* y, double* stats, const kd_block* block) {
    const std::string name("kd_block_rows");
    Mask mask;
    if (int rc = check_block("kd_block_rows", dtype, block, mask)) return rc;
    const kd_block& b = *block;
    if (y != nullptr && b.before.kind == KD_NORM_NONE) return fail(KD_E_INVALID, name + ": y needs a norm");
    if (b.rows == 0 || b.cols == 0) return KD_OK;
    if (b.x == nullptr) return fail(KD_E_INVALID, name + ": x must be given");
    if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) return fail(KD_E_INVALID, name + ": stats must be aligned to 8 bytes");
    const int64_t bytes = b.rows * b.cols * dtype_size(dtype), row_bytes = b.cols * dtype_size(dtype);
    for (void* out : {h, y})
        for (const void* in : {b.x, b.residual})
            if (out != in && overlap(out, bytes, in, bytes)) return fail(KD_E_INVALID, name + ": an output overlaps an input");
    for (void* out : {h, y, static_cast<void*>(stats)}) {
        const int64_t size = out == stats ? b.rows * 32 : bytes;
        if (overlap(out, size, mask.more_steps, 8)) return fail(KD_E_INVALID, name + ": an output overlaps more_steps");
        if (overlap(out, size, b.gate, b.gate_rows * row_bytes)) return fail(KD_E_INVALID, name + ": an output overlaps the gate");
        for (const kd_norm* n : {&b.after, &b.before})
            for (const void* in : {n->weight, n->bias})
                if (n->kind != KD_NORM_NONE && overlap(out, size, in, row_bytes))
                    return fail(KD_E_INVALID, name + ": an output overlaps a norm's weights");
    }
    if (overlap(h, bytes, y, bytes) || overlap(stats, b.rows * 32, h, bytes) || overlap(stats, b.rows * 32, y, bytes) ||
        overlap(stats, b.rows * 32, b.x, bytes) || overlap(stats, b.rows * 32, b.residual, bytes))
        return fail(KD_E_INVALID, name + ": outputs overlap");
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) {
        using T = decltype(zero);
        const BlockArgs<T> a = args_of<T>(b, mask);
        const auto one = [&](auto kernel, int threads, int64_t groups) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(threads), 0, stream(), static_cast<T*>(h),
                               static_cast<T*>(y), stats, a);
        };
        const auto rows = [&](auto most, auto quads, auto held, int threads, int64_t groups) {
            constexpr int kMost = decltype(most)::value, kQuads = decltype(quads)::value;
            constexpr bool kHeld = decltype(held)::value;
            if (b.cols % 4 != 0) {
                one(block_rows_kernel<T, kMost, kQuads, false, kHeld, kMost == 64>, threads, groups);
            } else if constexpr (kMost == 64) {
                one(block_rows_kernel<T, kMost, kQuads, true, kHeld, true>, threads, groups);
            } else {
                if (threads == kMost) one(block_rows_kernel<T, kMost, kQuads, true, kHeld, true>, threads, groups);
                else one(block_rows_kernel<T, kMost, kQuads, true, kHeld, false>, threads, groups);
            }
        };
        // Workgroups a CU that hold the weights: as many as fit its registers, `waves` a CU. They hold them where the weights are more bytes than x and
        // residual, and where each has two rows or more, in f64 (2000 x 2263 46 / 53) eight; us, weights read / held, both
        // norms and a gate: 32768 x 768 95 / 83, 16384 x 2048 122 / 105, 16384 x 2560 187 / 138, 8192 x 4096 121 / 106; a layer norm ahead of
        // the next block alone: 78 / 84, 104 / 108, 143 / 135, 104 / 111.
        const auto choose = [&](auto most, auto quads, int waves) {
            const int weights = 2 * (b.after.kind != KD_NORM_NONE) + 2 * (b.before.kind != KD_NORM_NONE) + (b.gate_rows == 1);
            const int threads = team_threads(b.cols, decltype(quads)::value);
            const int64_t groups = int64_t{waves * 64 / threads} * compute_units();
            if (weights > 2 && b.rows >= (sizeof(T) == 4 ? 2 : 8) * groups) rows(most, quads, std::true_type{}, threads, groups);
            else rows(most, quads, std::false_type{}, threads, b.rows);
        };
        // Quads a thread: so few registers that a CU has two workgroups of rows at least, but few enough threads that the barriers wait for few; one row a CU,
        // of many threads, where there are no more rows. us, a layer norm with dropout / both norms and a gate: 16384 x 2560 two quads 148 / 194,
        // three 141 / 137; 7000 x 6144 two 132 / 164, three 138 / 177, four 174 / 212; 4096 x 8192 two 124 / 163, four 115 / 142.
        // rows that a launch of a workgroup for each (or for four short ones) can have
        const int64_t limit = b.cols <= 512 ? int64_t{1} << 25 : b.cols <= 2048 ? int64_t{1} << 23 : int64_t{1} << 21;
        if (b.rows > limit || b.cols > 16384)
            one(block_rows_wide_kernel<T>, kWideThreads, std::min<int64_t>(b.rows, int64_t{compute_units()} * 16));
        else if (b.cols <= 256) rows(Int<64>{}, Int<1>{}, std::false_type{}, 256, (b.rows + 3) / 4);
        else if (b.cols <= 512) rows(Int<64>{}, Int<2>{}, std::false_type{}, 256, (b.rows + 3) / 4);
        else if (b.cols <= 1024) choose(Int<256>{}, Int<1>{}, 20);
        else if (b.cols <= 2048) choose(Int<512>{}, Int<2>{}, sizeof(T) == 4 ? 12 : 8);
        else if (b.cols <= 4096) {
            if constexpr (sizeof(T) == 4) {
                if (b.cols <= 12 * 256) choose(Int<256>{}, Int<3>{}, 8);
                else choose(Int<512>{}, Int<2>{}, 12);
            } else {
                choose(Int<512>{}, Int<2>{}, 8);
            }
        }
        else if (b.cols <= 6144 || (b.cols <= 8192 && b.rows <= compute_units()))
            rows(Int<1024>{}, Int<2>{}, std::false_type{}, team_threads(b.cols, 2), b.rows);
        else if (b.cols <= 8192) rows(Int<512>{}, Int<4>{}, std::false_type{}, team_threads(b.cols, 4), b.rows);
        else if (b.cols <= 12288) rows(Int<1024>{}, Int<3>{}, std::false_type{}, team_threads(b.cols, 3), b.rows);
        else rows(Int<1024>{}, Int<4>{}, std::false_type{}, team_threads(b.cols, 4), b.rows);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_block_rows_workspace(int64_t* bytes, int dtype, int64_t rows, int64_t cols) {
    const std::string name("kd_block_rows_workspace");
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (bytes == nullptr || rows < 0 || cols < 0 || cols > kMostCols || !fits(rows, cols)) return fail(KD_E_INVALID, name + ": bad arguments");
    *bytes = room_of(dtype, rows, cols);
    return KD_OK;
}

extern "C" int kd_block_rows_backward(int dtype, const kd_block_grads* grads, const kd_block* block, const void* h,
                                      const double* stats, const void* grad_h, const void* grad_y, void* workspace,
                                      int64_t workspace_bytes) {
    const std::string name("kd_block_rows_backward");
    Mask mask;
    if (int rc = check_block("kd_block_rows_backward", dtype, block, mask)) return rc;
    const kd_block& b = *block;
    if (grads == nullptr) return fail(KD_E_INVALID, name + ": the gradients must be given");
    if (grad_y != nullptr && b.before.kind == KD_NORM_NONE) return fail(KD_E_INVALID, name + ": grad_y needs a norm");
    if (((grads->after_weight != nullptr || grads->after_bias != nullptr) && b.after.kind == KD_NORM_NONE) ||
        ((grads->before_weight != nullptr || grads->before_bias != nullptr) && b.before.kind == KD_NORM_NONE))
        return fail(KD_E_INVALID, name + ": no norm, no gradient of its weight or bias");
    if (grads->gate != nullptr && b.gate == nullptr) return fail(KD_E_INVALID, name + ": no gate, no gradient of it");
    if (b.cols == 0) return KD_OK;
    const bool shared_gate = grads->gate != nullptr && b.gate_rows == 1;
    void* const sums[kSums] = {grads->after_weight, grads->after_bias, grads->before_weight, grads->before_bias,
                               shared_gate ? grads->gate : nullptr};
    const bool summed = std::any_of(sums, sums + kSums, [](void* p) { return p != nullptr; });
    const bool by_row = grads->x != nullptr || grads->residual != nullptr || (grads->gate != nullptr && !shared_gate);
    if (!summed && (!by_row || b.rows == 0)) return KD_OK;
    int64_t needed = 0;
    if (b.rows > 0) {
        if (stats == nullptr || reinterpret_cast<uintptr_t>(stats) % 8 != 0)
            return fail(KD_E_INVALID, name + ": stats must be given, aligned to 8 bytes");
        if (b.x == nullptr && (b.after.kind != KD_NORM_NONE || grads->gate != nullptr))
            return fail(KD_E_INVALID, name + ": x must be given");
        if (h == nullptr && grad_y != nullptr) return fail(KD_E_INVALID, name + ": h must be given");
        const int64_t bytes = b.rows * b.cols * dtype_size(dtype), row_bytes = b.cols * dtype_size(dtype);
        struct Memory {
            const void* at;
            int64_t bytes;
        };
        needed = room_of(dtype, b.rows, b.cols);
        const bool x_read = b.after.kind != KD_NORM_NONE || grads->gate != nullptr;
        const Memory outs[] = {{grads->x, bytes}, {grads->residual, bytes}, {grads->gate, b.gate_rows * row_bytes},
                               {grads->after_weight, row_bytes}, {grads->after_bias, row_bytes},
                               {grads->before_weight, row_bytes}, {grads->before_bias, row_bytes},
                               {summed ? workspace : nullptr, needed}};
        const Memory ins[] = {{x_read ? b.x : nullptr, bytes}, {grad_h, bytes}, {grad_y, bytes},
                              {grad_y != nullptr ? h : nullptr, bytes}, {b.gate, b.gate_rows * row_bytes}, {stats, b.rows * 32},
                              {b.after.kind != KD_NORM_NONE ? b.after.weight : nullptr, row_bytes},
                              {b.after.kind != KD_NORM_NONE && grads->gate != nullptr ? b.after.bias : nullptr, row_bytes},
                              {b.before.kind != KD_NORM_NONE ? b.before.weight : nullptr, row_bytes}, {mask.more_steps, 8}};
        for (int i = 0; i < static_cast<int>(std::size(outs)); ++i) {
            for (int j = 0; j < i; ++j)
                if (overlap(outs[i].at, outs[i].bytes, outs[j].at, outs[j].bytes)) return fail(KD_E_INVALID, name + ": outputs overlap");
            for (int j = 0; j < static_cast<int>(std::size(ins)); ++j) {
                // an element's own place
                const bool same = outs[i].at == ins[j].at && ((i == 0 && j <= 2) || (i == 1 && (j == 1 || j == 2)));
                if (!same && overlap(outs[i].at, outs[i].bytes, ins[j].at, ins[j].bytes))
                    return fail(KD_E_INVALID, name + ": an output overlaps an input");
            }
        }
        if (summed && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < needed))
            return fail(KD_E_INVALID, name + ": the summed gradients need " + std::to_string(needed) + " bytes of workspace");
    }
    if (int rc = ensure_device()) return rc;
    const auto launch = [&](auto zero) -> int {
        using T = decltype(zero);
        BackArgs<T> a{args_of<T>(b, mask), static_cast<const T*>(h), stats, static_cast<const T*>(grad_h),
                      static_cast<const T*>(grad_y), static_cast<T*>(grads->x), static_cast<T*>(grads->residual),
                      shared_gate ? nullptr : static_cast<T*>(grads->gate), {}};
        for (int k = 0; k < kSums; ++k) a.sums[k] = static_cast<T*>(sums[k]);
        SumPlaces places;
        places.wanted = 0;
        for (int k = 0; k < kSums; ++k) places.at[k] = sums[k] != nullptr ? places.wanted++ : -1;
        const BackPlan plan = b.rows > 0 ? back_plan(dtype, b.rows, b.cols, places.wanted) : BackPlan{};
        const int64_t column_groups = (b.cols + 63) / 64;
        if (!fits_grid(column_groups, kJoinWaves * 64) || !fits_grid(plan.segments, kBackThreads<float>) ||
            (plan.threads == 0 && plan.segments > 65535))
            return fail(KD_E_INVALID, name + ": too many rows or columns");
        const uint32_t groups = static_cast<uint32_t>(std::min<int64_t>(b.rows, int64_t{compute_units()} * 16));
        double* means = static_cast<double*>(workspace);
        T* parts = summed ? reinterpret_cast<T*>(means + (plan.threads == 0 ? 2 * b.rows : 0)) : nullptr;
        if (b.rows > 0 && plan.threads == 0) {
            const auto rows_of = [&](const BackArgs<T>& which, double* to) {
                const auto one = [&](auto kernel, int quads) {
                    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(b.rows)), dim3(team_threads(b.cols, quads)), 0, stream(), to, which);
                };
                const auto by_whole = [&](auto quads, auto past) {
                    constexpr int kQuads = decltype(quads)::value;
                    constexpr bool kPast = decltype(past)::value;
                    if (b.cols % 4 == 0) one(block_back_row_kernel<T, kQuads, true, kPast>, kQuads);
                    else one(block_back_row_kernel<T, kQuads, false, kPast>, kQuads);
                };
                // Gradients go past the caches where they and the inputs are more than the last one's 256 MiB: the sums' kernel finds
                // more of its inputs there. Both kernels, us, through / past: both norms and a gate, f32 4096 x 8192 335 / 320, 8192 x 5120
                // 480 / 470, f64 2000 x 8192 293 / 281; a layer norm alone, f32 4096 x 8192 258 / 247, 8192 x 5120 346 / 348.
                const bool past = to != nullptr && 6 * b.rows * b.cols * static_cast<int64_t>(sizeof(T)) > int64_t{256} << 20;
                const auto by_past = [&](auto quads) {
                    if (past) by_whole(quads, std::true_type{});
                    else by_whole(quads, std::false_type{});
                };
                if (b.rows > int64_t{1} << 21 || b.cols > (sizeof(T) == 4 ? 16384 : 8192)) {
                    hipLaunchKernelGGL((block_back_wide_kernel<T>), dim3(groups), dim3(kWideThreads), 0, stream(), to, which);
                    return;
                }
                if (b.cols <= 8192) by_past(Int<2>{});
                else if constexpr (sizeof(T) == 4) by_past(Int<4>{});
            };
            // gradients in the place of what the sums read are written last
            const auto in_place = [](const void* out, const void* in) { return out != nullptr && out == in; };
            const bool first = !summed || in_place(grads->residual, grad_h) || in_place(grads->residual, grad_y) || in_place(grads->x, b.x) ||
                               in_place(grads->x, grad_h) || in_place(grads->x, grad_y);
            if (summed) {
                BackArgs<T> which = a;
                if (first) which.x = which.residual = which.gate = nullptr;
                rows_of(which, means);
                const dim3 grid(static_cast<uint32_t>((b.cols + 255) / 256), static_cast<uint32_t>(plan.segments));
                if (b.cols % 4 == 0) hipLaunchKernelGGL((block_columns_kernel<T, true>), grid, dim3(kThreads), 0, stream(), parts, means, a);
                else hipLaunchKernelGGL((block_columns_kernel<T, false>), grid, dim3(kThreads), 0, stream(), parts, means, a);
            }
            if (first && by_row) rows_of(a, nullptr);
        }
        if (plan.threads != 0) {
            const auto one = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(plan.segments)), dim3(static_cast<uint32_t>(plan.teams * plan.threads)),
                                   static_cast<uint32_t>(sums_bytes(dtype, b.cols, plan.teams, places.wanted)), stream(), parts, a, plan.threads,
                                   plan.rows_per_team, places);
            };
            // what the compiler knows of a team saves 3 %
            const auto by_whole = [&](auto threads, auto quads) {
                constexpr int kTeam = decltype(threads)::value, kQuads = decltype(quads)::value;
                constexpr bool kHeld = kQuads == 1;
                if (b.cols % 4 == 0) one(block_back_kernel<T, kTeam, kQuads, kHeld, true>);
                else one(block_back_kernel<T, kTeam, kQuads, kHeld, false>);
            };
            if (plan.quads == 2) {
                if constexpr (sizeof(T) == 8) by_whole(Int<0>{}, Int<2>{});
            } else if (plan.threads == 64) by_whole(Int<64>{}, Int<1>{});
            else if (plan.threads == 256) by_whole(Int<256>{}, Int<1>{});
            else if (plan.threads == 512) by_whole(Int<512>{}, Int<1>{});
            else if (plan.threads == 1024) {
                if constexpr (sizeof(T) == 4) by_whole(Int<1024>{}, Int<1>{});
            } else by_whole(Int<0>{}, Int<1>{});
        }
        if (summed)
            hipLaunchKernelGGL((block_join_kernel<T>), dim3(static_cast<uint32_t>(column_groups), kSums), dim3(kJoinWaves * 64), 0,
                               stream(), a, parts, plan.segments);
        KD_LAUNCH_CHECK();
        return KD_OK;
    };
    return dtype == KD_F32 ? launch(0.f) : launch(0.0);
}
