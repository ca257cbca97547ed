// kd_block.hip - dropout with a mask from a counter, and the end of a transformer's block (a norm of its output, dropout, a
// gate, the residual sum, the norm ahead of the next block) with its backward pass.
#include <algorithm>

#include "kd_counter.h"
#include "kd_internal.h"

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

template <typename T> struct NormArgs {
    const T* weight;
    const T* bias;
    double eps;
    int kind;
    __device__ __forceinline__ double weight_at(int64_t c) const { return weight != nullptr ? static_cast<double>(weight[c]) : 1.0; }
    __device__ __forceinline__ double bias_at(int64_t c) const { return bias != nullptr ? static_cast<double>(bias[c]) : 0.0; }
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

// Count, mean and sum of squared distances from the mean. A part's sums are taken about one of its own values p, which lies
// within sqrt(n var) of the mean, so the difference below loses at most a factor n of the rounding; parts are joined by Chan,
// Golub and LeVeque's formula ("Algorithms for computing the sample variance", 1983).
struct Moments {
    double n, mean, squares;
    __device__ __forceinline__ void join(const Moments& o) {
        const double total = n + o.n, d = o.mean - mean;
        if (o.n == 0) return;
        if (n == 0) {
            *this = o;
            return;
        }
        mean += d * (o.n / total);
        squares += o.squares + d * d * (n * o.n / total);
        n = total;
    }
};
struct MomentSums {
    double n = 0, p = 0, s1 = 0, s2 = 0;
    __device__ __forceinline__ void add(double v) {
        if (n == 0) p = v;
        const double d = v - p;
        n += 1;
        s1 += d;
        s2 += d * d;
    }
    __device__ __forceinline__ Moments moments() const {
        return n > 0 ? Moments{n, p + s1 / n, s2 - s1 * (s1 / n)} : Moments{0, 0, 0};
    }
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 32; m > 0; m /= 2) v += __shfl_xor(v, m);
    return v;
}

// Sums over the workgroup, the waves' in order; `room` holds a value a wave.
__device__ __forceinline__ double group_sum(double v, double* room) {
    const int waves = blockDim.x / 64;
    v = wave_sum(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = v;
    __syncthreads();
    double total = 0;
    for (int w = 0; w < waves; ++w) total += room[w];
    return total;
}

__device__ __forceinline__ Moments group_moments(Moments m, Moments* room) {
    const int waves = blockDim.x / 64;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        Moments o;
        o.n = __shfl_xor(m.n, d);
        o.mean = __shfl_xor(m.mean, d);
        o.squares = __shfl_xor(m.squares, d);
        m.join(o);
    }
    __syncthreads();
    if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = m;
    __syncthreads();
    Moments total = room[0];
    for (int w = 1; w < waves; ++w) total.join(room[w]);
    return total;
}

// The statistics of a row that `value(c)` gives.
template <typename F> __device__ __forceinline__ RowStats row_stats(int kind, double eps, int64_t cols, Moments* room, F value) {
    if (kind == KD_NORM_NONE) return {0.0, 1.0};
    MomentSums sums;
    if (kind == KD_NORM_LAYER) {
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) sums.add(value(c));
        const Moments m = group_moments(sums.moments(), room);
        return {m.mean, 1.0 / sqrt(m.squares / static_cast<double>(cols) + eps)};
    }
    double squares = 0;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
        const double v = value(c);
        squares += v * v;
    }
    return {0.0, 1.0 / sqrt(group_sum(squares, reinterpret_cast<double*>(room)) / static_cast<double>(cols) + eps)};
}

// The block's output at column c of a row, after its norm and dropout.
template <typename T>
__device__ __forceinline__ double branch_at(const BlockArgs<T>& a, const RowStats& s, int64_t row, int64_t c, uint32_t step) {
    double v = static_cast<double>(a.x[row * a.cols + c]);
    if (a.after.kind != KD_NORM_NONE) v = s.unit(v) * a.after.weight_at(c) + a.after.bias_at(c);
    if (a.masked) {
        bool k[4];
        a.mask.kept(k, static_cast<uint32_t>(row), static_cast<uint32_t>(c / 4), step);
        const bool one = c % 4 == 0 ? k[0] : c % 4 == 1 ? k[1] : c % 4 == 2 ? k[2] : k[3];
        v = one ? v * a.mask.scale : 0.0;
    }
    return v;
}
template <typename T> __device__ __forceinline__ double gate_at(const BlockArgs<T>& a, int64_t row, int64_t c) {
    return a.gate != nullptr ? static_cast<double>(a.gate[row * a.gate_step + c]) : 1.0;
}

// Any row length: a workgroup a row, which is read again in each pass.
template <typename T>
__global__ __launch_bounds__(kThreads) void block_rows_wide_kernel(T* h, T* y, double* stats, BlockArgs<T> a) {
    __shared__ Moments room[kThreads / 64];
    const uint32_t step = a.mask.step_now();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t base = row * a.cols;
        const RowStats after = row_stats(a.after.kind, a.after.eps, a.cols, room,
                                         [&](int64_t c) { return static_cast<double>(a.x[base + c]); });
        const auto sum = [&](int64_t c) {
            double v = a.block_scale * gate_at(a, row, c) * branch_at(a, after, row, c, step);
            if (a.residual != nullptr) v += a.residual_scale * static_cast<double>(a.residual[base + c]);
            return static_cast<T>(v);
        };
        // h may take x's or the residual's place, so from then on it is read there; each thread reads what it has written
        if (h != nullptr)
            for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) h[base + c] = sum(c);
        const auto h_at = [&](int64_t c) { return static_cast<double>(h != nullptr ? h[base + c] : sum(c)); };
        RowStats before{0.0, 1.0};
        if (a.before.kind != KD_NORM_NONE && (y != nullptr || stats != nullptr)) {
            before = row_stats(a.before.kind, a.before.eps, a.cols, room, h_at);
            if (y != nullptr)
                for (int64_t c = threadIdx.x; c < a.cols; c += kThreads)
                    y[base + c] = static_cast<T>(before.unit(h_at(c)) * a.before.weight_at(c) + a.before.bias_at(c));
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
    // p and p v at column c
    __device__ __forceinline__ double weighted(int64_t base, int64_t c) const {
        return static_cast<double>(grad_y[base + c]) * b.before.weight_at(c);
    }
    // G, from the means of p and p v
    __device__ __forceinline__ double total(int64_t base, int64_t c, const RowStats& s, double mean, double along) const {
        double g = grad_h != nullptr ? static_cast<double>(grad_h[base + c]) : 0.0;
        if (grad_y != nullptr) g += s.rate * (weighted(base, c) - mean - s.unit(static_cast<double>(h[base + c])) * along);
        return g;
    }
    __device__ __forceinline__ bool kept(int64_t row, int64_t c, uint32_t step) const {
        if (!b.masked) return true;
        bool k[4];
        b.mask.kept(k, static_cast<uint32_t>(row), static_cast<uint32_t>(c / 4), step);
        return c % 4 == 0 ? k[0] : c % 4 == 1 ? k[1] : c % 4 == 2 ? k[2] : k[3];
    }
};

// The means of p and p v of a row.
template <typename T>
__device__ __forceinline__ void before_means(const BackArgs<T>& a, int64_t row, double* room, double& mean, double& along) {
    mean = along = 0;
    if (a.grad_y == nullptr) return;
    const int64_t base = row * a.b.cols;
    const RowStats s = a.before(row);
    for (int64_t c = threadIdx.x; c < a.b.cols; c += blockDim.x) {
        const double p = a.weighted(base, c);
        mean += p;
        along += p * s.unit(static_cast<double>(a.h[base + c]));
    }
    along = group_sum(along, room) / static_cast<double>(a.b.cols);
    mean = a.b.before.kind == KD_NORM_LAYER ? group_sum(mean, room) / static_cast<double>(a.b.cols) : 0.0;
}

// Any row length: the gradients of the rows, a workgroup each.
template <typename T> __global__ __launch_bounds__(kThreads) void block_back_wide_kernel(BackArgs<T> a) {
    __shared__ double room[kThreads / 64];
    const uint32_t step = a.b.mask.step_now();
    const int64_t cols = a.b.cols;
    for (int64_t row = blockIdx.x; row < a.b.rows; row += gridDim.x) {
        const int64_t base = row * cols;
        const RowStats before = a.before(row), after = a.after(row);
        double mean, along, back_mean = 0, back_along = 0;
        before_means(a, row, room, mean, along);
        const auto through = [&](int64_t c, double g) {
            return a.kept(row, c, step) ? a.b.block_scale * gate_at(a.b, row, c) * g * a.b.mask.scale : 0.0;
        };
        const bool normed = a.b.after.kind != KD_NORM_NONE && a.x != nullptr;
        if (normed) {
            for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
                const double q = through(c, a.total(base, c, before, mean, along)) * a.b.after.weight_at(c);
                back_mean += q;
                back_along += q * after.unit(static_cast<double>(a.b.x[base + c]));
            }
            back_along = group_sum(back_along, room) / static_cast<double>(cols);
            back_mean = a.b.after.kind == KD_NORM_LAYER ? group_sum(back_mean, room) / static_cast<double>(cols) : 0.0;
        }
        // outputs may take the place of what is read at the same element
        for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
            const double g = a.total(base, c, before, mean, along);
            const double branch = a.gate != nullptr ? branch_at(a.b, after, row, c, step) : 0.0;
            double d = through(c, g);
            if (normed)
                d = after.rate * (d * a.b.after.weight_at(c) - back_mean - after.unit(static_cast<double>(a.b.x[base + c])) * back_along);
            if (a.residual != nullptr) a.residual[base + c] = static_cast<T>(a.b.residual_scale * g);
            if (a.gate != nullptr) a.gate[base + c] = static_cast<T>(a.b.block_scale * branch * g);
            if (a.x != nullptr) a.x[base + c] = static_cast<T>(d);
        }
    }
}

// The means that the sums over rows need: [rows][2].
template <typename T> __global__ __launch_bounds__(kThreads) void block_means_kernel(double* means, BackArgs<T> a) {
    __shared__ double room[kThreads / 64];
    for (int64_t row = blockIdx.x; row < a.b.rows; row += gridDim.x) {
        double mean, along;
        before_means(a, row, room, mean, along);
        if (threadIdx.x == 0) {
            means[2 * row] = mean;
            means[2 * row + 1] = along;
        }
    }
}

// The sums over a segment of rows: [segment][sum][cols]. A workgroup takes 64 columns, its waves share the rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void block_columns_kernel(double* parts, const double* means, BackArgs<T> a,
                                                                 int64_t rows_per_segment) {
    __shared__ double room[kThreads / 64][kSums][64];
    const uint32_t step = a.b.mask.step_now();
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane, cols = a.b.cols;
    const int64_t from = blockIdx.y * rows_per_segment, to = min(a.b.rows, from + rows_per_segment);
    double sums[kSums] = {};
    if (c < cols)
        for (int64_t row = from + wave; row < to; row += kThreads / 64) {
            const int64_t base = row * cols;
            const RowStats before = a.before(row), after = a.after(row);
            const double g = a.total(base, c, before, means[2 * row], means[2 * row + 1]);
            if (a.grad_y != nullptr) {
                const double own = static_cast<double>(a.grad_y[base + c]);
                sums[kBeforeWeight] += own * before.unit(static_cast<double>(a.h[base + c]));
                sums[kBeforeBias] += own;
            }
            if (a.sums[kGate] != nullptr) sums[kGate] += a.b.block_scale * branch_at(a.b, after, row, c, step) * g;
            if (a.b.after.kind != KD_NORM_NONE) {
                const double d = a.kept(row, c, step) ? a.b.block_scale * gate_at(a.b, row, c) * g * a.b.mask.scale : 0.0;
                sums[kAfterWeight] += d * after.unit(static_cast<double>(a.b.x[base + c]));
                sums[kAfterBias] += d;
            }
        }
#pragma unroll
    for (int k = 0; k < kSums; ++k) room[wave][k][lane] = sums[k];
    __syncthreads();
    if (wave == 0 && c < cols)
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            double total = room[0][k][lane];
            for (int w = 1; w < kThreads / 64; ++w) total += room[w][k][lane];
            parts[(blockIdx.y * kSums + k) * cols + c] = total;
        }
}

// The segments' sums in order: a workgroup takes 64 columns of one sum, its 16 waves a run of segments each.
constexpr int kJoinWaves = 16;
template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void block_join_kernel(BackArgs<T> a, const double* parts, int64_t segments) {
    __shared__ double room[kJoinWaves][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    T* out = a.sums[blockIdx.y];
    if (out == nullptr) return;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane, cols = a.b.cols;
    const int64_t run = (segments + kJoinWaves - 1) / kJoinWaves;
    double sum = 0;
    if (c < cols)
        for (int64_t s = wave * run; s < min(segments, (wave + 1) * run); ++s) sum += parts[(s * kSums + blockIdx.y) * cols + c];
    room[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || c >= cols) return;
    for (int w = 1; w < kJoinWaves; ++w) sum += room[w][lane];
    out[c] = static_cast<T>(sum);
}

// ---- plans and checks -----------------------------------------------------------------------------

// Segments of rows whose sums are kept apart: enough to fill the card, at most 64 MiB of them.
int64_t segments_of(int64_t rows, int64_t cols) {
    const int64_t most = std::max<int64_t>(1, (int64_t{64} << 20) / (cols * kSums * 8));
    return std::max<int64_t>(1, std::min({(rows + 15) / 16, int64_t{1024}, most}));
}
int64_t means_bytes(int64_t rows) { return rows * 16; }

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
    if (b->rows < 0 || b->cols < 0 || !fits(b->rows, b->cols)) return fail(KD_E_INVALID, name + ": bad number of rows or columns");
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
    const int64_t bytes = b.rows * b.cols * dtype_size(dtype), row_bytes = b.cols * dtype_size(dtype);
    for (void* out : {h, y})
        for (const void* in : {b.x, b.residual})
            if (out != in && overlap(out, bytes, in, bytes)) return fail(KD_E_INVALID, name + ": an output overlaps an input");
    for (void* out : {h, y, static_cast<void*>(stats)}) {
        const int64_t size = out == stats ? b.rows * 32 : bytes;
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
        const uint32_t groups = static_cast<uint32_t>(std::min<int64_t>(b.rows, int64_t{compute_units()} * 32));
        hipLaunchKernelGGL((block_rows_wide_kernel<T>), dim3(groups), dim3(kThreads), 0, stream(), static_cast<T*>(h),
                           static_cast<T*>(y), stats, a);
    };
    if (dtype == KD_F32) launch(0.f);
    else launch(0.0);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_block_rows_workspace(int64_t* bytes, int dtype, int64_t rows, int64_t cols) {
    const std::string name("kd_block_rows_workspace");
    if (dtype != KD_F32 && dtype != KD_F64) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32 or f64");
    if (bytes == nullptr || rows < 0 || cols < 0 || !fits(rows, cols)) return fail(KD_E_INVALID, name + ": bad arguments");
    *bytes = rows == 0 || cols == 0 ? 0 : means_bytes(rows) + segments_of(rows, cols) * kSums * cols * 8;
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
        if (stats == nullptr) return fail(KD_E_INVALID, name + ": stats must be given");
        if (b.x == nullptr && (b.after.kind != KD_NORM_NONE || grads->gate != nullptr))
            return fail(KD_E_INVALID, name + ": x must be given");
        if (h == nullptr && grad_y != nullptr) return fail(KD_E_INVALID, name + ": h must be given");
        const int64_t bytes = b.rows * b.cols * dtype_size(dtype), row_bytes = b.cols * dtype_size(dtype);
        struct Memory {
            const void* at;
            int64_t bytes;
        };
        needed = means_bytes(b.rows) + segments_of(b.rows, b.cols) * kSums * b.cols * 8;
        const bool x_read = b.after.kind != KD_NORM_NONE || grads->gate != nullptr;
        const Memory outs[] = {{grads->x, bytes}, {grads->residual, bytes}, {grads->gate, b.gate_rows * row_bytes},
                               {grads->after_weight, row_bytes}, {grads->after_bias, row_bytes},
                               {grads->before_weight, row_bytes}, {grads->before_bias, row_bytes},
                               {summed ? workspace : nullptr, needed}};
        const Memory ins[] = {{x_read ? b.x : nullptr, bytes}, {grad_h, bytes}, {grad_y, bytes},
                              {grad_y != nullptr ? h : nullptr, bytes}, {b.gate, b.gate_rows * row_bytes}, {stats, b.rows * 32},
                              {b.after.kind != KD_NORM_NONE ? b.after.weight : nullptr, row_bytes},
                              {b.before.kind != KD_NORM_NONE ? b.before.weight : nullptr, row_bytes}};
        for (int i = 0; i < 8; ++i) {
            for (int j = 0; j < i; ++j)
                if (overlap(outs[i].at, outs[i].bytes, outs[j].at, outs[j].bytes)) return fail(KD_E_INVALID, name + ": outputs overlap");
            for (int j = 0; j < 8; ++j) {
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
        const uint32_t groups = static_cast<uint32_t>(std::min<int64_t>(b.rows, int64_t{compute_units()} * 32));
        if (summed) {
            const int64_t column_groups = (b.cols + 63) / 64;
            if (!fits_grid(column_groups, kJoinWaves * 64)) return fail(KD_E_INVALID, name + ": too many columns");
            double* means = static_cast<double*>(workspace);
            double* parts = means + 2 * b.rows;
            int64_t segments = 0;
            if (b.rows > 0) {
                segments = segments_of(b.rows, b.cols);
                const int64_t per_segment = (b.rows + segments - 1) / segments;
                segments = (b.rows + per_segment - 1) / per_segment;
                hipLaunchKernelGGL((block_means_kernel<T>), dim3(groups), dim3(kThreads), 0, stream(), means, a);
                hipLaunchKernelGGL((block_columns_kernel<T>), dim3(static_cast<uint32_t>(column_groups), static_cast<uint32_t>(segments)),
                                   dim3(kThreads), 0, stream(), parts, means, a, per_segment);
            }
            hipLaunchKernelGGL((block_join_kernel<T>), dim3(static_cast<uint32_t>(column_groups), kSums), dim3(kJoinWaves * 64), 0,
                               stream(), a, parts, segments);
        }
        if (by_row && b.rows > 0) hipLaunchKernelGGL((block_back_wide_kernel<T>), dim3(groups), dim3(kThreads), 0, stream(), a);
        KD_LAUNCH_CHECK();
        return KD_OK;
    };
    return dtype == KD_F32 ? launch(0.f) : launch(0.0);
}
