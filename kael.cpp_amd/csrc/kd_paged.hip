// kd_paged.hip - the paged 8-bit key / value cache: appending rotated keys and values, reading them back, and the
// attention of ragged new queries over them.
//
// A cached value is one signed byte times the f32 scale of its page and kv head. Keys lie token by token, values feature by
// feature with a page's tokens side by side, so that both are read in 16-byte pieces along the axis that the
// attention's products sum over. Everything that a caller's arrays can say wrongly (a table entry that is no page, a
// start or a length out of range) is checked here against the sizes that the host passed.
#include <algorithm>
#include <type_traits>

#include "kd_internal.h"

namespace kd {

namespace {

struct Paged {
    int8_t* keys;
    int8_t* values;
    float* key_scales;
    float* value_scales;
    const int64_t* table;
    const int64_t* starts;
    const int64_t* lengths;
    int64_t pages;
    int kv_heads, head_dim;
    int page_shift;  // page_size = 1 << page_shift
    int sequences, columns, tokens;
};

// A sequence's rows: `count` from `row` on, the first of them at position `position` (may be below 0).
struct Rows {
    int row, count;
    int64_t position;
};

__device__ __forceinline__ int start_of(const Paged& c, int s) {
    const int64_t v = c.starts[s];
    return static_cast<int>(v < 0 ? 0 : v > c.tokens ? c.tokens : v);
}

__device__ __forceinline__ Rows rows_of(const Paged& c, int s) {
    const int row = start_of(c, s), end = start_of(c, s + 1);
    const int count = max(end - row, 0);
    // a length beyond any table is as good as 2^40, so that no sum below overflows
    int64_t length = c.lengths[s];
    length = length < 0 ? 0 : length > (int64_t{1} << 40) ? int64_t{1} << 40 : length;
    return {row, count, length - count};
}

// The page of table column `column` of sequence s, or -1.
__device__ __forceinline__ int64_t page_of(const Paged& c, int s, int64_t column) {
    if (column < 0 || column >= c.columns) return -1;
    const int64_t page = c.table[static_cast<int64_t>(s) * c.columns + column];
    return page >= 0 && page < c.pages ? page : -1;
}

// Work is handed out by slots: sequence s owns the slots base(start, s) .. base(next start, s + 1) - 1, base ascending. Which
// sequence a slot belongs to (s < 0 for none) is found by a whole wave, every lane of which has to call this: in one round
// of loads with the sequence's rows for up to 64 sequences, and 64 at a time beyond (two rounds up to 4096).
struct Found {
    int s;
    int64_t base;
    Rows rows;
};

// Lane `lane`'s value (the lane the same for the whole wave), in a scalar register.
__device__ __forceinline__ int64_t from_lane(int64_t x, int lane) {
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(x), lane);
    return static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane)) << 32 | low;
}
__device__ __forceinline__ Rows from_lane(const Rows& rows, int lane) {
    return {__builtin_amdgcn_readlane(rows.row, lane), __builtin_amdgcn_readlane(rows.count, lane), from_lane(rows.position, lane)};
}

template <class Base> __device__ __forceinline__ Found find_sequence(const Paged& c, int64_t slot, const Base& base) {
    const int lane = threadIdx.x % 64;
    if (c.sequences <= 64) {
        const int s = min(lane, c.sequences - 1);
        const Rows rows = rows_of(c, s);
        const int64_t own = base(rows.row, s);
        const int n = __popcll(__ballot(lane < c.sequences && own <= slot));
        if (n == 0) return {-1, 0, {}};
        return {n - 1, from_lane(own, n - 1), from_lane(rows, n - 1)};
    }
    int low = 0, count = c.sequences;
    while (count > 1) {
        const int step = (count + 63) / 64;
        const int at = low + lane * step;
        const int n = __popcll(__ballot(lane * step < count && base(start_of(c, at < c.sequences ? at : 0), at) <= slot));
        if (n == 0) return {-1, 0, {}};
        low += (n - 1) * step;
        count = min(step, count - (n - 1) * step);
    }
    const Rows rows = from_lane(rows_of(c, low), 0);
    return {low, base(rows.row, low), rows};
}

// Walks on from a sequence that begins at or before `token` to the one that holds it; s is c.sequences where none does.
__device__ __forceinline__ void walk_to(const Paged& c, int token, int& s, Rows& rows) {
    while (s < c.sequences && token >= rows.row + rows.count) {
        ++s;
        if (s < c.sequences) rows = rows_of(c, s);
    }
}

// The new tokens of one page, as the workgroup of `slot` sees them: slots held .. held + count - 1 of table column `column`.
struct PageSlots {
    int s;
    int row;        // batch row of the first of them
    int64_t first;  // its position
    int64_t page;   // -1 for none
    int held, count;
    bool leads;     // the first slot of its sequence
    Rows rows;
};

// A sequence's new tokens touch at most (count + 2 size - 2) / size pages; base(s + 1) - base(s) is at least that.
__host__ __device__ inline int64_t page_base(int64_t start, int64_t s, int shift) {
    return (start + s * ((int64_t{2} << shift) - 2)) >> shift;
}

__device__ __forceinline__ PageSlots page_slots(const Paged& c, int64_t slot) {
    const Found f = find_sequence(c, slot, [&](int64_t start, int64_t s) { return page_base(start, s, c.page_shift); });
    PageSlots p{f.s, 0, 0, -1, 0, 0, false, f.rows};
    if (f.s < 0) return p;
    const int64_t begin = max(f.rows.position, int64_t{0}), end = f.rows.position + f.rows.count;
    const int64_t column = (begin >> c.page_shift) + (slot - f.base);
    const int64_t from = max(begin, column << c.page_shift), to = min(end, (column + 1) << c.page_shift);
    p.leads = slot == f.base;
    if (from >= to) return p;
    p.page = page_of(c, f.s, column);
    p.row = f.rows.row + static_cast<int>(from - f.rows.position);
    p.first = from;
    p.held = static_cast<int>(from - (column << c.page_shift));
    p.count = static_cast<int>(to - from);
    return p;
}

// ---- append ---------------------------------------------------------------------------------------
//
// Bound by the bytes of q, k and v for prompts, by the chain of dependent loads (starts and lengths, table, scale, rows) for
// single tokens. One launch: a workgroup takes one page of one kv head, its keys or its values, so that the page's scale
// has one owner, and the workgroups behind those take the queries. Rotated and quantised in f64, where the products of two
// f32 are exact and a rounding to the wrong side of a tie takes a value within 2^-45 of it: f64 costs less here than the bytes.
// Keys and values are read twice, for the scale and for the codes, the second time mostly from behind the L2 (42 of 52 MB in the
// case below): a page held in registers or LDS in between left fewer workgroups on a CU and took longer. 6347 tokens of 32 + 2 x 8 heads of 128: 71 us, 274 MB at
// 3.9 TB/s; 64 single tokens of 12 heads of 64: 6.9 us.

struct Rotation {
    const float* cosines;
    const float* sines;
    int64_t positions;
    int half;  // pairs; 0 rotates nothing
    bool interleaved;
};

struct Strided {
    const float* data;
    int64_t row, head;
};

constexpr int kUnit = 8;  // features of a thread: four pairs, or eight that are not rotated

// Past: the load takes no place in the caches.
typedef float v4f __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store4(float* p, const v4f& x) { *reinterpret_cast<v4f*>(p) = x; }
template <bool Vector, bool Past = false> __device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
    if constexpr (Vector && Past) {
        const v4f v = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(p));
        x[0] = v[0], x[1] = v[1], x[2] = v[2], x[3] = v[3];
    } else if constexpr (Vector) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = p[i];
    }
}

// Where unit u of a row has its two runs of four features. Without Vector a unit is eight features that follow each other.
template <bool Vector> __device__ __forceinline__ void unit_places(int u, const Rotation& r, int& low, int& high) {
    low = kUnit * u;
    high = low + 4;
    if (Vector && !r.interleaved && low < 2 * r.half) {
        low = 4 * u;
        high = low + r.half;
    }
}

// The unit of the row x, rotated by `position`'s angles, in f64. Vector: pairs never cross a unit and everything is 16-byte
// aligned; otherwise each feature finds its partner.
template <bool Vector, bool Past = false>
__device__ __forceinline__ void rotated_unit(const float* x, int low, int high, int64_t position, const Rotation& r, double (&y)[kUnit]) {
    float a[4], b[4];
    load4<Vector, Past>(x + low, a);
    load4<Vector, Past>(x + high, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = a[i];
        y[4 + i] = b[i];
    }
    if (low >= 2 * r.half) return;
    const bool known = position >= 0 && position < r.positions;  // queries may stand below position 0
    if constexpr (Vector) {
        float c[4] = {NAN, NAN, NAN, NAN}, s[4] = {NAN, NAN, NAN, NAN};
        if (known) {
            const int64_t at = position * r.half + (r.interleaved ? low / 2 : low);
            load4<true>(r.cosines + at, c);
            load4<true>(r.sines + at, s);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // pair i of the unit: its features 2 i and 2 i + 1, or feature i of either run
            const double p = r.interleaved ? (i < 2 ? a[2 * i % 4] : b[2 * i % 4]) : a[i];
            const double q = r.interleaved ? (i < 2 ? a[(2 * i + 1) % 4] : b[(2 * i + 1) % 4]) : b[i];
            const double turned = p * c[i] - q * s[i], other = q * c[i] + p * s[i];
            if (r.interleaved) {
                y[2 * i] = turned;
                y[2 * i + 1] = other;
            } else {
                y[i] = turned;
                y[4 + i] = other;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const int d = low + i;
            if (d >= 2 * r.half) break;
            const int pair = r.interleaved ? d / 2 : d % r.half;
            const bool second = r.interleaved ? d % 2 != 0 : d >= r.half;
            const double p = x[r.interleaved ? 2 * pair : pair], q = x[r.interleaved ? 2 * pair + 1 : pair + r.half];
            const double c = known ? r.cosines[position * r.half + pair] : NAN, s = known ? r.sines[position * r.half + pair] : NAN;
            y[i] = second ? q * c + p * s : p * c - q * s;
        }
    }
}

__device__ __forceinline__ uint32_t code_of(double x, double inverse) {
    const double r = rint(x * inverse);
    return r != r ? 0u : static_cast<uint32_t>(static_cast<int>(fmin(fmax(r, -127.0), 127.0))) & 0xffu;
}

constexpr int kAppendThreads = 256;
constexpr int64_t kPastBytes = int64_t{32} << 20;  // of queries, from which on they are loaded past the caches

template <int D, bool Vector, bool Past>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(Paged c, Rotation rotation, Strided k, Strided v,
                                                                      Strided q, float* __restrict__ q_out, int heads,
                                                                      int64_t cache_groups, int q_tokens) {
    constexpr int dim = D, units = D / kUnit;
    const int threads = blockDim.x;
    if (static_cast<int64_t>(blockIdx.x) >= cache_groups) {
        // the queries of q_tokens tokens
        const int64_t token0 = (static_cast<int64_t>(blockIdx.x) - cache_groups) * q_tokens;
        Found f = find_sequence(c, token0, [&](int64_t start, int64_t) { return start; });
        if (f.s < 0) f = {0, 0, rows_of(c, 0)};
        const uint32_t per_token = static_cast<uint32_t>(heads) * units;
        for (uint32_t i = threadIdx.x; i < q_tokens * per_token; i += threads) {
            const int64_t token = token0 + i / per_token;
            if (token >= c.tokens) return;
            int s = f.s;
            Rows rows = f.rows;
            walk_to(c, static_cast<int>(token), s, rows);
            if (s >= c.sequences || token < rows.row) continue;
            const uint32_t h = i % per_token / units;
            int low, high;
            unit_places<Vector>(i % units, rotation, low, high);
            const int64_t position = rows.position + (token - rows.row);
            double y[kUnit];
            rotated_unit<Vector, Past>(q.data + token * q.row + h * q.head, low, high, position, rotation, y);
            float* out = q_out + (token * heads + h) * dim;
            const auto at = [&](int j) { return position < 0 ? NAN : static_cast<float>(y[j]); };
            store4(out + low, v4f{at(0), at(1), at(2), at(3)});
            store4(out + high, v4f{at(4), at(5), at(6), at(7)});
        }
        return;
    }
    const uint32_t group = c.kv_heads * 2;
    const int h = static_cast<int>(blockIdx.x % group) / 2;
    const bool keys = blockIdx.x % 2 == 0;
    const int size = 1 << c.page_shift;
    const PageSlots p = page_slots(c, blockIdx.x / group);
    if (p.page < 0) return;
    const int64_t at = p.page * c.kv_heads + h;
    int8_t* codes = (keys ? c.keys : c.values) + at * size * dim;
    float* scales = keys ? c.key_scales : c.value_scales;
    const float old = p.held > 0 ? scales[at] : 0.f;
    const Strided in = keys ? k : v;
    const float* x = in.data + static_cast<int64_t>(p.row) * in.row + h * in.head;
    // keys: a unit of a token; values: a feature of 16 tokens that begin at a multiple of 16 slots
    const int key_units = p.count * units;
    const int chunk0 = p.held / 16, value_units = ((p.held + p.count + 15) / 16 - chunk0) * dim;
    double most = 0;
    if (keys) {
        for (int i = threadIdx.x; i < key_units; i += threads) {
            const int token = i / units;
            int low, high;
            unit_places<Vector>(i % units, rotation, low, high);
            double y[kUnit];
            rotated_unit<Vector>(x + token * in.row, low, high, p.first + token, rotation, y);
#pragma unroll
            for (int j = 0; j < kUnit; ++j) most = max_na(most, fabs(y[j]));
        }
    } else {
        float largest = 0;
        for (int i = threadIdx.x; i < value_units; i += threads) {
            const int slot0 = (chunk0 + i / dim) * 16;
            float y[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int token = slot0 + j - p.held;
                y[j] = token >= 0 && token < p.count ? x[token * in.row + i % dim] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) largest = max_na(largest, fabsf(y[j]));
        }
        most = largest;
    }
    __shared__ double wave_most[kAppendThreads / 64];
#pragma unroll
    for (int m = 32; m > 0; m /= 2) most = max_na(most, __shfl_xor(most, m));
    if (threads > 64) {
        if (threadIdx.x % 64 == 0) wave_most[threadIdx.x / 64] = most;
        __syncthreads();
        for (int w = 0; w < threads / 64; ++w) most = max_na(most, wave_most[w]);
    }
    const float scale = most < INFINITY ? max_na(old, static_cast<float>(most / 127)) : NAN;
    if (threadIdx.x == 0) scales[at] = scale;
    const double inverse = scale > 0 ? 1.0 / scale : 0.0;  // 0 for NaN too
    if (keys) {
        for (int i = threadIdx.x; i < key_units; i += threads) {
            const int token = i / units;
            int low, high;
            unit_places<Vector>(i % units, rotation, low, high);
            double y[kUnit];
            rotated_unit<Vector, Past>(x + token * in.row, low, high, p.first + token, rotation, y);
            uint32_t word[2] = {};
#pragma unroll
            for (int j = 0; j < kUnit; ++j) word[j / 4] |= code_of(y[j], inverse) << (8 * (j % 4));
            int8_t* to = codes + (p.held + token) * dim;
            *reinterpret_cast<uint32_t*>(to + low) = word[0];
            *reinterpret_cast<uint32_t*>(to + high) = word[1];
        }
    } else {
        for (int i = threadIdx.x; i < value_units; i += threads) {
            const int slot0 = (chunk0 + i / dim) * 16, d = i % dim;
            int8_t* to = codes + d * size + slot0;
            const int from = max(p.held - slot0, 0), end = min(p.held + p.count - slot0, 16);
            const float* row = x + static_cast<int64_t>(slot0 - p.held) * in.row + d;
            if (from == 0 && end == 16) {
                float y[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) y[j] = row[j * in.row];
                uint4 words = make_uint4(0, 0, 0, 0);
                uint32_t* word = &words.x;
#pragma unroll
                for (int j = 0; j < 16; ++j) word[j / 4] |= code_of(y[j], inverse) << (8 * (j % 4));
                *reinterpret_cast<uint4*>(to) = words;
            } else {
                for (int j = from; j < end; ++j) to[j] = static_cast<int8_t>(code_of(row[j * in.row], inverse));
            }
        }
    }
    if (scale > old) {
        const double ratio = static_cast<double>(old) / scale;
        for (int i = threadIdx.x; i < p.held * dim; i += threads) {
            int8_t* code = codes + (keys ? i : i / p.held * size + i % p.held);
            *code = static_cast<int8_t>(rint(*code * ratio));
        }
    }
}

// ---- read -----------------------------------------------------------------------------------------
//
// The append's division into pages: four codes a thread and a 16-byte store for the keys, a feature's 16 tokens a thread for
// the values, so that codes are read in whole pieces and rows written in whole lines. Bound by the bytes, the rows' above all:
// 67 MB in 14 us. Rows stored past the caches take less time alone (79 MB of them 17 us instead of 27) and cost their reader more than that
// (with a sum of keys and values behind it 49.3 / 47.3, 102 MB 61.1 / 59.3, 52 MB 31.5 / 31.5), so they are not.

__global__ __launch_bounds__(256) void paged_read_kernel(Paged c, float* __restrict__ k, float* __restrict__ v) {
    const uint32_t group = c.kv_heads * 2;
    const int h = static_cast<int>(blockIdx.x % group) / 2;
    const bool keys = blockIdx.x % 2 == 0;
    float* out = keys ? k : v;
    if (out == nullptr) return;
    const int dim = c.head_dim, size = 1 << c.page_shift, threads = blockDim.x;
    const PageSlots p = page_slots(c, blockIdx.x / group);
    if (p.s < 0) return;
    const int64_t row_size = static_cast<int64_t>(c.kv_heads) * dim;
    out += h * dim;
    const auto clear = [&](int row, int count) {  // of any number of rows: 2^27 have 2^31 pieces
        const int shift = dim == 64 ? 4 : 5;
        for (int64_t i = threadIdx.x; i < int64_t{count} << shift; i += threads)
            *reinterpret_cast<float4*>(out + (row + (i >> shift)) * row_size + (i & ((1 << shift) - 1)) * 4) = make_float4(0, 0, 0, 0);
    };
    // rows before position 0 have no page
    if (p.leads && p.rows.position < 0) clear(p.rows.row, static_cast<int>(min(int64_t{p.rows.count}, -p.rows.position)));
    if (p.count == 0) return;
    if (p.page < 0) {
        clear(p.row, p.count);
        return;
    }
    const int64_t at = p.page * c.kv_heads + h;
    out += p.row * row_size;
    if (keys) {
        const float scale = c.key_scales[at];
        const int8_t* codes = c.keys + (at * size + p.held) * dim;
        for (int i = threadIdx.x; i < p.count * (dim / 4); i += threads) {
            const char4 x = *reinterpret_cast<const char4*>(codes + 4 * i);
            store4(out + i / (dim / 4) * row_size + i % (dim / 4) * 4, v4f{x.x * scale, x.y * scale, x.z * scale, x.w * scale});
        }
    } else {
        const float scale = c.value_scales[at];
        const int8_t* codes = c.values + at * size * dim;
        const int chunk0 = p.held / 16, chunks = (p.held + p.count + 15) / 16 - chunk0;
        for (int i = threadIdx.x; i < chunks * dim; i += threads) {
            const int slot0 = (chunk0 + i / dim) * 16, d = i % dim;
            const uint4 words = *reinterpret_cast<const uint4*>(codes + d * size + slot0);
            const uint32_t* word = &words.x;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int token = slot0 + j - p.held;
                const float x = static_cast<float>(static_cast<int8_t>(word[j / 4] >> (8 * (j % 4)))) * scale;
                float* to = out + token * row_size + d;
                if (token >= 0 && token < p.count) *to = x;
            }
        }
    }
}

// ---- attention ------------------------------------------------------------------------------------
//
// Scores and weighted sums run on the signed 8-bit matrix cores, whose sums are exact: the cached codes go in as they
// are, and the other operand as four signed digits of base 256. A query row is q = 2^(e - 30) * x with x whole, e the
// exponent of its largest feature (x is exact for features of at least 2^-6 of that one, and off by 2^-30 of it at
// most otherwise); a weight exp(score - max) times its value scale likewise, against the largest of a row's block. Four products a
// tile and twice bf16's rate are as many cycles as two bf16 products, where three would be needed for f32's bits, and the
// codes need no conversion.
//
// A wave holds 16 rows (queries x the heads that share the kv head) as columns and takes 64 keys at a time:
//   scores: 4 tiles of 16 keys, S^T = K . Q^T (16x16x64): lane l ends with column l % 16 and, the tiles' rows being dealt
//     out so, the 16 keys of chunk g = l / 16; a chunk lies in one page, so a lane has one page, key scale and value scale;
//   weights: their digits are the B operand of the second product as they stand, no lane exchanges anything;
//   sums: O^T += V^T . P^T, the values' pages holding a feature's 16 tokens side by side.
// The next block's codes are loaded while the present one is worked on, and the table entries of the one after it.
//
// Where there are fewer rows, a row takes S = 2 or 4 columns, each of them 4 / S of its digits: a tile is S times fewer products,
// and the columns that join a score's digits share its row's keys out between them, so that a lane computes 16 / S
// weights; their digits go back to the columns that multiply with them by exchanges within four lanes.
//
// Bound by the codes' bytes for many sequences (4 x 40000 keys of 128, 32 heads over 8: 47 us, 5.5 TB/s; 64 x 4000 of 64, one row,
// 52 us, 5.7 TB/s), by the loads' latency for 9 to 32 rows (17 x 20000 of 64, 24 rows: vector ALU
// busy 0.42 of the cycles, matrix cores 0.10, waves waiting 0.31), by the chain of loads (starts, table, codes) and 50 GB/s a CU for few.

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kRowTile = 16;
constexpr int kTileRows = 64;  // rows of a workgroup
constexpr int kKeyBlock = 64;

// Sequence s has base(s + 1) - base(s) >= ceil(count * group / rows) tiles of `rows` rows.
__host__ __device__ inline int64_t tile_base(int64_t start, int64_t s, int group, int rows = kTileRows) { return start * group / rows + s; }

template <int Control> __device__ __forceinline__ int in_quad(int x) { return __builtin_amdgcn_mov_dpp(x, Control, 0xf, 0xf, true); }
constexpr int kNextLane = 0xb1, kOtherPair = 0x4e;  // lane ^ 1, lane ^ 2 (quad_perm)

// x of the lanes l, l ^ 16, l ^ 32 and l ^ 48 put together, in every one of them.
template <class Op> __device__ __forceinline__ int over_chunks(int x, const Op& op) {
    const auto near = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = op(static_cast<int>(near[0]), static_cast<int>(near[1]));
    const auto far = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return op(static_cast<int>(far[0]), static_cast<int>(far[1]));
}
__device__ __forceinline__ float chunks_max(float x) {
    return __int_as_float(over_chunks(__float_as_int(x), [](int a, int b) {
        return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
    }));
}
__device__ __forceinline__ float chunks_sum(float x) {
    return __int_as_float(over_chunks(__float_as_int(x), [](int a, int b) {
        return __float_as_int(__int_as_float(a) + __int_as_float(b));
    }));
}

// The digits of four whole numbers x of size at most 2^30 from x + kDigitBias: byte r of digits[p] is digit p of x[r], in
// -128 .. 127. The bias adds 128 to the lower three digits, whose bytes then are those of the sum; flipping their top bits
// takes it off again.
constexpr int kDigitBias = 0x00808080;
__device__ __forceinline__ void digits_of(const int (&biased)[4], int (&digits)[4]) {
    const uint32_t y0 = biased[0], y1 = biased[1], y2 = biased[2], y3 = biased[3];
    const uint32_t low01 = __builtin_amdgcn_perm(y1, y0, 0x05010400u), low23 = __builtin_amdgcn_perm(y3, y2, 0x05010400u);
    const uint32_t high01 = __builtin_amdgcn_perm(y1, y0, 0x07030602u), high23 = __builtin_amdgcn_perm(y3, y2, 0x07030602u);
    digits[0] = static_cast<int>(__builtin_amdgcn_perm(low23, low01, 0x05040100u) ^ 0x80808080u);
    digits[1] = static_cast<int>(__builtin_amdgcn_perm(low23, low01, 0x07060302u) ^ 0x80808080u);
    digits[2] = static_cast<int>(__builtin_amdgcn_perm(high23, high01, 0x05040100u) ^ 0x80808080u);
    digits[3] = static_cast<int>(__builtin_amdgcn_perm(high23, high01, 0x07060302u));
}

// The digits' four sums as one number: each is below 2^21 in size, so the pairs are exact.
__device__ __forceinline__ float joined(const v4i (&sum)[4], int r) {
    return static_cast<float>((sum[3][r] << 8) + sum[2][r]) * 65536.f + static_cast<float>((sum[1][r] << 8) + sum[0][r]);
}

// The digits of a lane's 16 U features of a query row (0 where the row is not real) and the factor that a score's whole number
// times its key's scale takes: scale * 2^(e - 30) * log2(e), positive, the scale's sign being in the digits; NaN where the
// row is not finite.
template <int U> __device__ __forceinline__ float query_digits(float (&features)[16 * U], bool real, double scale, v4i (&digits)[4][U]) {
    int bits = 0;
#pragma unroll
    for (int d = 0; d < 16 * U; ++d) {
        features[d] = real ? features[d] : 0.f;
        bits = max(bits, __float_as_int(features[d]) & 0x7fffffff);
    }
    bits = over_chunks(bits, [](int a, int b) { return max(a, b); });
    const int e = __builtin_amdgcn_frexp_expf(__int_as_float(bits));  // 0 for 0; unused where not finite
    const float sign = scale < 0 ? -1.f : 1.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            int y[4], d4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = static_cast<int>(rintf(ldexpf(features[16 * u + 4 * t + i] * sign, 30 - e))) + kDigitBias;
            digits_of(y, d4);
#pragma unroll
            for (int p = 0; p < 4; ++p) digits[p][u][t] = d4[p];
        }
    return bits < 0x7f800000 ? static_cast<float>(ldexp(fabs(scale) * 1.4426950408889634074, e - 30)) : NAN;
}

// The exponent e of the largest of a row's weighted value scales, whose bits are `top`, at least `least`: 2^(e - 30) is the unit of
// whole weights and 2^(e - 13) that of f16 ones, and neither may fall below f32's least number.
constexpr int kLeastWhole = 30 - 149, kLeastHalf = 13 - 149;
// The unit is not below that of 2^-96 of the largest value scale, so that the scale in units stays finite.
constexpr int kFarBelow = 96 << 23;
__device__ __forceinline__ int unit_exponent(int top, int least) {
    return max(__builtin_amdgcn_frexp_expf(__int_as_float(top)), least);
}

// A row's maximum is a rounded product, and a weight's exponent the fused product less that maximum: the largest weight is
// 2^(that rounding), 2^(1/16) at most for maxima below this. From here on the products are rounded ahead of the subtraction, so
// that it is 1 again and none is larger.
constexpr float kFarScore = 0x1p20f;
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// What a row's factor and a key's scale make of a score's whole number. Infinity is NaN: times a number below 0 it would be
// -infinity, a weight of nothing.
__device__ __forceinline__ float score_factor(float query, float key_scale) {
    const float factor = query * key_scale;
    return factor < INFINITY ? factor : NAN;
}

struct Split {
    int count;    // parts that a row's keys are split into
    int part;     // keys of a part, a multiple of 64; the last part goes to the end
    float* sums;  // [row][count][D], then [row][count][2] of the maximum (base 2) and the sum
};

// The one of S values that column `sub` of a row's S takes.
template <int S> __device__ __forceinline__ int taken(int sub, int a, int b, int c, int d) {
    if constexpr (S == 2) return sub == 0 ? a : b;
    else return sub & 2 ? (sub & 1 ? d : c) : sub & 1 ? b : a;
}
// x of a row's S columns put together, in each of them.
template <int S, class T, class Op> __device__ __forceinline__ T over_row(T x, const Op& op) {
    if constexpr (S > 1) x = op(x, __builtin_bit_cast(T, in_quad<kNextLane>(__builtin_bit_cast(int, x))));
    if constexpr (S > 2) x = op(x, __builtin_bit_cast(T, in_quad<kOtherPair>(__builtin_bit_cast(int, x))));
    return x;
}
struct MostOf {
    __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumOf {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
constexpr MostOf most_of;
constexpr SumOf sum_of;

template <int D, int Waves, int S>
__global__ __launch_bounds__(Waves * 64, D == 64 ? 4 : 2) void paged_attention_kernel(Paged c, float* __restrict__ out, Strided q,
                                                                                      int heads, FastDiv by_group, double scale,
                                                                                      Split split) {
    constexpr int U = D / 64, J = 4 / S;
    constexpr int kRowTile = 16 / S, kTileRows = 4 * kRowTile;
    constexpr int kLd = D + 4;
    __shared__ __attribute__((aligned(16))) float os[Waves][kRowTile][kLd];
    __shared__ float ms[Waves][kRowTile], ls[Waves][kRowTile];
    const int group = static_cast<int>(by_group.divisor);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int column = lane % 16, chunk = lane / 16;
    const int sub = column % S;
    const int part = blockIdx.y, kv = static_cast<int>(blockIdx.x % c.kv_heads);
    // the last rows see most keys and go first
    const int64_t tile = (gridDim.x - 1 - blockIdx.x) / c.kv_heads;
    const Found found = find_sequence(c, tile, [&](int64_t start, int64_t at) { return tile_base(start, at, group, kTileRows); });
    if (found.s < 0) return;
    const Rows rows = found.rows;
    // tokens * heads is below 2^31, and so are the rows of a kv head
    const int64_t tile_at = (tile - found.base) * kTileRows;
    const int row_end = rows.count * group;
    if (tile_at < 0 || tile_at >= row_end) return;
    const int row0 = static_cast<int>(tile_at);
    const int here = min(row_end - row0, kTileRows);
    // row tiles of the workgroup (1, 2 or 4), and the waves that share a tile's keys
    const int row_waves = here <= kRowTile ? 1 : here <= 2 * kRowTile ? 2 : 4, key_waves = Waves / row_waves;
    const int row_wave = wave % row_waves, key_wave = wave / row_waves;
    const int64_t capacity = static_cast<int64_t>(c.columns) << c.page_shift;
    // keys 0 .. limit - 1 are visible to the row of token `token` of the sequence
    const auto limit_of = [&](int token) {
        const int64_t limit = rows.position + token + 1;
        return static_cast<int>(limit < 0 ? 0 : limit > capacity ? capacity : limit);
    };
    const auto token_of = [&](int row) { return static_cast<int>(by_group.div(row)); };
    const int from = part * split.part;
    const int all = limit_of(token_of(row0 + here - 1));
    if (from >= all && part > 0) return;
    const int to = part + 1 == split.count ? all : min(all, from + split.part);
    // rows past the last one stand in for it with a query of 0 and are not written
    const int tile_row = row0 + row_wave * kRowTile;
    const bool real = row_wave * kRowTile + column / S < here;
    const int r = min(tile_row + column / S, row0 + here - 1);
    const int token = token_of(r);
    const int limit = limit_of(token);
    const int least = __builtin_amdgcn_readfirstlane(limit);  // limits ascend with the columns
    const int most = min(to, __builtin_amdgcn_readlane(limit, 15));
    const int step = key_waves * kKeyBlock;
    int key = from + key_wave * kKeyBlock;

    // Lane i of `window` holds the page of table column window_from + i, so that the table's loads are not waited for
    // among the codes'.
    const int size = 1 << c.page_shift;
    const int64_t* table = c.table + static_cast<int64_t>(found.s) * c.columns;
    int window = 0, window_from = -128;
    const auto pages_of_block = [&](int key) {
        if (((key + kKeyBlock - 1) >> c.page_shift) - window_from >= 64) {
            window_from = key >> c.page_shift;
            const int64_t page = table[min(window_from + lane, c.columns - 1)];
            window = window_from + lane < c.columns && page >= 0 && page < c.pages ? static_cast<int>(page) : -1;
        }
    };
    const auto page_at = [&](int key) { return __shfl(window, (key >> c.page_shift) - window_from); };

    // A lane's piece of the keys lies in chunk column / 4, its scores and its piece of the values in chunk lane / 16. Where
    // there is no page the first one is read, and masked.
    const int key_chunk = column / 4;
    v4i k[4][U], v[D / 16];
    const int8_t* values_at;
    float key_scale, value_scale;
    int page;
    const uint32_t page_bytes = static_cast<uint32_t>(c.kv_heads) * size * D;  // at most 2^27
    const int8_t* keys_base = c.keys + (kv * size + lane % 4) * D + chunk * 16 * U;
    const int8_t* values_base = c.values + (kv * D + column) * size;
    const auto load_keys = [&](int key) {
        pages_of_block(key);
        page = page_at(key + 16 * chunk);
        const uint32_t own = max(page, 0), other = max(page_at(key + 16 * key_chunk), 0);
        const int slot = (key + 16 * key_chunk) & (size - 1), own_slot = (key + 16 * chunk) & (size - 1);
        const int8_t* at = keys_base + uint64_t{other} * page_bytes + slot * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < U; ++u) k[t][u] = *reinterpret_cast<const v4i*>(at + 4 * t * D + 16 * u);
        key_scale = c.key_scales[uint64_t{own} * static_cast<uint32_t>(c.kv_heads) + kv];
        value_scale = c.value_scales[uint64_t{own} * static_cast<uint32_t>(c.kv_heads) + kv];
        values_at = values_base + uint64_t{own} * page_bytes + own_slot;
    };
    const auto load_values = [&] {
#pragma unroll
        for (int n = 0; n < D / 16; ++n) v[n] = *reinterpret_cast<const v4i*>(values_at + 16 * n * size);
    };

    // the row's digits: features chunk * 16 U .. + 16 U - 1 of its column's row
    const float* row = q.data + (rows.row + token) * q.row + (kv * group + r - token * group) * q.head + chunk * 16 * U;
    float features[16 * U];
#pragma unroll
    for (int d = 0; d < 16 * U; ++d) features[d] = row[d];
    if (key < most) {  // in flight while the digits are made
        load_keys(key);
        load_values();
    }
    v4i digits[J][U];
    float q_factor;
    if constexpr (S == 1) {
        q_factor = query_digits(features, real, scale, digits);
    } else {
        v4i all[4][U];
        q_factor = query_digits(features, real, scale, all);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    digits[j][u][t] = taken<S>(sub, all[j][u][t], all[J + j][u][t], all[(2 * J + j) % 4][u][t],
                                               all[(3 * J + j) % 4][u][t]);
    }
    // of the digits that a column holds, and of those of lane ^ 1 or lane ^ 2 (S == 4) that hold the other half
    const bool upper = sub >= S / 2 && S > 1, odd = sub % 2 != 0;
    const float half_unit = upper ? 65536.f : 1.f, other_unit = upper ? 1.f : 65536.f;
    const float sub_unit = S == 4 && odd ? 256.f * half_unit : half_unit;
    const int shift = odd ? 8 : 0;

    float m = -INFINITY, l = 0.f;
    float o[D / 4] = {};
    for (; key < most; key += step) {
        float x[4 * J];  // of the tiles J sub .. J sub + J - 1
        int half[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            v4i sum[J];
#pragma unroll
            for (int p = 0; p < J; ++p) {
                sum[p] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < U; ++u)
                    sum[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][u], digits[p][u], sum[p], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (S == 1) {
                    x[4 * t + i] = joined(sum, i);
                    asm("" : "+v"(x[4 * t + i]));  // joined here, not behind the branch below with every tile's sums held
                } else if constexpr (S == 2) {
                    half[t][i] = (sum[1][i] << 8) + sum[0][i];
                } else {
                    half[t][i] = sum[0][i] << shift;
                }
            }
        }
        if constexpr (S == 4) {  // the halves of the tiles of the lane's parity, in half[0] and half[2]
#pragma unroll
            for (int t = 0; t < 4; t += 2)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kept = odd ? half[t + 1][i] : half[t][i], sent = odd ? half[t][i] : half[t + 1][i];
                    half[t][i] = kept + in_quad<kNextLane>(sent);
                }
        }
        if constexpr (S > 1)
#pragma unroll
            for (int t = 0; t < J; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kept = upper ? half[2 + t][i] : half[t][i], sent = upper ? half[t][i] : half[2 + t][i];
                    x[4 * t + i] = static_cast<float>(kept) * half_unit +
                                   static_cast<float>(in_quad<S == 4 ? kOtherPair : kNextLane>(sent)) * other_unit;
                    asm("" : "+v"(x[4 * t + i]));
                }
        const int first = key + 16 * chunk + 4 * J * sub;  // x[i] is key first + i
        const int seen = page < 0 ? 0 : limit - first;
        const int scale_bits = seen > 0 ? __float_as_int(value_scale) & 0x7fffffff : 0;
        const float own_scale = value_scale;
        // never 0, so that a masked key's -inf stays what it is
        float factor = score_factor(q_factor, key_scale);
        factor = factor == 0.f ? 0x1p-126f : factor;
        if (key + kKeyBlock > least || __any(page < 0)) {
            factor = seen > 0 ? factor : 1.f;  // nor NaN where the row sees none of them
#pragma unroll
            for (int i = 0; i < 4 * J; ++i) x[i] = i < seen ? x[i] : -INFINITY;
        }
        load_keys(key + step < most ? key + step : key);  // the last block once more rather than a branch
        float largest = x[0];
#pragma unroll
        for (int i = 1; i < 4 * J; ++i) largest = fmaxf(largest, x[i]);
        const float next = fmaxf(m, chunks_max(over_row<S>(largest * factor, most_of)));
        const float base = next == -INFINITY ? 0.f : next;  // nothing seen yet: every weight below is 0
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = next;
        // Heads of 64 with several columns a row: always, where the branch would spill four registers (32 x 5 x 2000 keys 19.0 us, with
        // the branch 20.6; of 128, 4 x 40000 of 4 rows 48.6 / 47.0).
        if ((D == 64 && S > 1) || __any(fabsf(base) >= kFarScore)) {
#pragma unroll
            for (int i = 0; i < 4 * J; ++i) x[i] = rounded_product(x[i], factor);
            largest = rounded_product(largest, factor);
            factor = 1.f;
        }
        // the unit of the weights times their value scales: the largest of them that the row has here, as bits, so that NaN is the
        // largest of all
        const float weight = __builtin_amdgcn_exp2f(fmaf(largest, factor, -base)) * own_scale;
        const int weight_bits = seen > 0 ? __float_as_int(weight) & 0x7fffffff : 0;
        const int top = over_chunks(over_row<S>(max(weight_bits, scale_bits - kFarBelow), most_of), most_of);
        const int e = unit_exponent(max(top, 0), kLeastWhole);
        const float to_whole = top < 0x7f800000 && seen > 0 ? ldexpf(own_scale, 30 - e) : 0.f;
        // with the unit of the column's digits, so that the sums are never smaller than what they stand for
        const float from_whole = top < 0x7f800000 ? ldexpf(sub_unit, e - 30) : NAN;
        float sum = 0.f;
        v4i weights[J];
#pragma unroll
        for (int t = 0; t < J; ++t) {
            int w[4], d4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(x[4 * t + i], factor, -base));
                sum += p;
                // from 2^23 on an f32 is whole: the bias rounds the weight too, to half a unit or its own last bit
                w[i] = static_cast<int>(fmaf(p, to_whole, static_cast<float>(kDigitBias)));
            }
            digits_of(w, d4);
#pragma unroll
            for (int p = 0; p < J; ++p) {
                if constexpr (S == 1) {
                    weights[p][t] = d4[p];
                } else if constexpr (S == 2) {
                    const int own = sub == 0 ? d4[p] : d4[J + p];
                    const int other = in_quad<kNextLane>(sub == 0 ? d4[J + p] : d4[p]);
                    weights[p][t] = sub == 0 ? own : other;
                    weights[p][J + t] = sub == 0 ? other : own;
                }
            }
            if constexpr (S == 4) {
                // the quad's digits the other way round: d4[p] of tile t from lane t to lane p, as weights[0][t]
#pragma unroll
                for (int p = 0; p < 4; p += 2) {
                    const int other = in_quad<kNextLane>(odd ? d4[p] : d4[p + 1]);
                    d4[p] = odd ? other : d4[p];
                    d4[p + 1] = odd ? d4[p + 1] : other;
                }
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int other = in_quad<kOtherPair>(upper ? d4[p] : d4[p + 2]);
                    weights[0][p] = upper ? other : d4[p];
                    weights[0][p + 2] = upper ? d4[p + 2] : other;
                }
            }
        }
        l = l * alpha + sum;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            v4i acc[J];
#pragma unroll
            for (int p = 0; p < J; ++p)
                acc[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[n], weights[p], v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float part;
                if constexpr (S == 1) part = joined(acc, i);
                else if constexpr (S == 2) part = static_cast<float>((acc[1][i] << 8) + acc[0][i]);
                else part = static_cast<float>(acc[0][i]);
                o[4 * n + i] = o[4 * n + i] * alpha + part * from_whole;
            }
        }
        load_values();
    }
    l = chunks_sum(over_row<S>(l, sum_of));
    if (chunk == 0 && sub == 0) {
        ms[wave][column / S] = m;
        ls[wave][column / S] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 4; ++d) o[d] = over_row<S>(o[d], sum_of);
    if (sub == 0)
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
            *reinterpret_cast<float4*>(&os[wave][column / S][16 * n + 4 * chunk]) =
                make_float4(o[4 * n], o[4 * n + 1], o[4 * n + 2], o[4 * n + 3]);
    __syncthreads();
    // the waves that shared a row's keys joined, in their order
    for (int i = threadIdx.x; i < here * (D / 4); i += Waves * 64) {
        const int at = i / (D / 4), d = i % (D / 4) * 4;
        const int w0 = at / kRowTile, col = at % kRowTile;
        float top = -INFINITY;
        for (int w = 0; w < key_waves; ++w) top = fmaxf(top, ms[w0 + w * row_waves][col]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < key_waves; ++w) {
            const int from_wave = w0 + w * row_waves;
            const float f = __builtin_amdgcn_exp2f(ms[from_wave][col] - base);
            const float4 add = *reinterpret_cast<const float4*>(&os[from_wave][col][d]);
            sum += f * ls[from_wave][col];
            v.x += f * add.x;
            v.y += f * add.y;
            v.z += f * add.z;
            v.w += f * add.w;
        }
        const int of_token = token_of(row0 + at);
        const int64_t to_row = static_cast<int64_t>(rows.row + of_token) * heads + kv * group + (row0 + at - of_token * group);
        if (split.count == 1) {
            const float by = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<float4*>(out + to_row * D + d) = make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
        } else {
            const int64_t record = to_row * split.count + part;
            *reinterpret_cast<float4*>(split.sums + record * D + d) = v;
            if (d == 0) {
                float* own = split.sums + static_cast<int64_t>(c.tokens) * heads * split.count * D + record * 2;
                own[0] = top;
                own[1] = sum;
            }
        }
    }
}

// One row a workgroup (single tokens whose heads share nothing). Its four digits take four columns, and all sixteen columns
// share the keys out, one to a lane: a weight costs a lane one exponential where the kernel above computes four. The sums of the
// outputs stay whole over the blocks, and are turned into f32 when the largest weight or weighted scale changes or they could
// pass 2^31. 64 x 1024 keys of 64, 12 heads: 16.5 us, 76 MB at 4.6 TB/s; 1 x 1000: 6.8 us, the launch and the chain of loads.
constexpr int kMostBlocks = 1024;  // that the whole sums hold: 2^10 blocks of 2^6 keys of 2^14

template <int D, int Waves>
__global__ __launch_bounds__(Waves * 64, D == 64 ? 4 : 2) void paged_single_kernel(Paged c, float* __restrict__ out, Strided q, int heads,
                                                                  FastDiv by_group, FastDiv by_heads, double scale, Split split) {
    constexpr int U = D / 64;
    __shared__ __attribute__((aligned(16))) float os[Waves][D];
    __shared__ float ms[Waves], ls[Waves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int column = lane % 16, chunk = lane / 16, digit = lane % 4;
    const int part = blockIdx.y;
    const int token = c.tokens - 1 - static_cast<int>(by_heads.div(blockIdx.x));
    const int head = static_cast<int>(blockIdx.x) - (c.tokens - 1 - token) * heads;
    const int kv = static_cast<int>(by_group.div(head));
    const Found found = find_sequence(c, token, [&](int64_t start, int64_t) { return start; });
    if (found.s < 0) return;
    const Rows rows = found.rows;
    if (token >= rows.row + rows.count) return;
    const int64_t capacity = static_cast<int64_t>(c.columns) << c.page_shift;
    const int64_t visible = rows.position + (token - rows.row) + 1;
    const int limit = static_cast<int>(visible < 0 ? 0 : visible > capacity ? capacity : visible);
    const int from = part * split.part;
    if (from >= limit && part > 0) return;
    const int to = part + 1 == split.count ? limit : min(limit, from + split.part);
    constexpr int step = Waves * kKeyBlock;
    int key = from + wave * kKeyBlock;

    const int size = 1 << c.page_shift;
    const int64_t* table = c.table + static_cast<int64_t>(found.s) * c.columns;
    int window = 0, window_from = -128;
    const auto pages_of_block = [&](int key) {
        if (((key + kKeyBlock - 1) >> c.page_shift) - window_from >= 64) {
            window_from = key >> c.page_shift;
            const int64_t page = table[min(window_from + lane, c.columns - 1)];
            window = window_from + lane < c.columns && page >= 0 && page < c.pages ? static_cast<int>(page) : -1;
        }
    };
    const auto page_at = [&](int key) { return __shfl(window, (key >> c.page_shift) - window_from); };
    const int key_chunk = column / 4;
    v4i k[4][U], v[D / 16];
    const int8_t* values_at;
    float key_scale, value_scale;
    int page;
    const uint32_t page_bytes = static_cast<uint32_t>(c.kv_heads) * size * D;  // at most 2^27
    const int8_t* keys_base = c.keys + (kv * size + lane % 4) * D + chunk * 16 * U;
    const int8_t* values_base = c.values + (kv * D + column) * size;
    const auto load_keys = [&](int key) {
        pages_of_block(key);
        page = page_at(key + 16 * chunk);
        const uint32_t own = max(page, 0), other = max(page_at(key + 16 * key_chunk), 0);
        const int slot = (key + 16 * key_chunk) & (size - 1), own_slot = (key + 16 * chunk) & (size - 1);
        const int8_t* at = keys_base + uint64_t{other} * page_bytes + slot * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int u = 0; u < U; ++u) k[t][u] = *reinterpret_cast<const v4i*>(at + 4 * t * D + 16 * u);
        key_scale = c.key_scales[uint64_t{own} * static_cast<uint32_t>(c.kv_heads) + kv];
        value_scale = c.value_scales[uint64_t{own} * static_cast<uint32_t>(c.kv_heads) + kv];
        values_at = values_base + uint64_t{own} * page_bytes + own_slot;
    };
    const auto load_values = [&] {
#pragma unroll
        for (int n = 0; n < D / 16; ++n) v[n] = *reinterpret_cast<const v4i*>(values_at + 16 * n * size);
    };

    const float* row = q.data + token * q.row + head * q.head + chunk * 16 * U;
    float features[16 * U];
#pragma unroll
    for (int d = 0; d < 16 * U; ++d) features[d] = row[d];
    if (key < to) {
        load_keys(key);
        load_values();
    }
    // a column's digit of the query: its lane's number in the quad
    v4i digits[U];
    float q_factor;
    {
        v4i all[4][U];
        q_factor = query_digits(features, true, scale, all);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int low = digit & 1 ? all[1][u][t] : all[0][u][t], high = digit & 1 ? all[3][u][t] : all[2][u][t];
                digits[u][t] = digit & 2 ? high : low;
            }
    }
    const int shift = 8 * (digit & 1);
    const float pair_unit = digit & 2 ? 65536.f : 1.f, digit_unit = pair_unit * (digit & 1 ? 256.f : 1.f);
    const uint32_t first_bytes = digit & 1 ? 0x03070105u : 0x06020400u, second_bytes = digit & 2 ? 0x03020706u : 0x05040100u;

    float m = -INFINITY, l = 0.f;  // l is the lane's own
    float o[D / 4] = {};           // what the column's digit adds
    v4i acc[D / 16] = {};          // since the last change of the unit
    int top = 0, blocks = 0;       // the largest weight times its value scale, as bits, so that NaN is the largest of all
    int to_whole = 0;              // the exponent that a weight takes to its units
    float from_whole = 0.f;
    const auto flush = [&](float alpha) {
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[4 * n + i] = (o[4 * n + i] + static_cast<float>(acc[n][i]) * from_whole) * alpha;
            acc[n] = v4i{0, 0, 0, 0};
        }
        blocks = 0;
    };
    for (; key < to; key += step) {
        v4i sum[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            sum[t] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u) sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][u], digits[u], sum[t], 0, 0, 0);
        }
        // column / 4 is the tile that a lane keeps, column % 4 the row of it: key `lane` of the block
        int pair[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int low = column & 4 ? sum[1][r] : sum[0][r], high = column & 4 ? sum[3][r] : sum[2][r];
            pair[r] = (column & 8 ? high : low) << shift;
            pair[r] += in_quad<kNextLane>(pair[r]);
        }
        const int kept_low = digit & 1 ? pair[1] : pair[0], kept_high = digit & 1 ? pair[3] : pair[2];
        const int kept = digit & 2 ? kept_high : kept_low, sent = digit & 2 ? kept_low : kept_high;
        const float whole = static_cast<float>(kept) * pair_unit +
                            __int_as_float(in_quad<kOtherPair>(__float_as_int(static_cast<float>(sent) * pair_unit)));
        const bool seen = page >= 0 && key + lane < to;
        const float own_scale = seen ? value_scale : 0.f;
        const float x = seen ? rounded_product(whole, score_factor(q_factor, key_scale)) : -INFINITY;
        load_keys(key + step < to ? key + step : key);  // the last block once more rather than a branch
        if (__any(x > m)) {
            float next = x;
#pragma unroll
            for (int d = 32; d > 0; d /= 2) next = fmaxf(next, __shfl_xor(next, d));
            next = fmaxf(next, m);
            const float alpha = __builtin_amdgcn_exp2f(m - next);
            flush(alpha);
            l *= alpha;
            top = __float_as_int(__int_as_float(top) * alpha) & 0x7fffffff;
            m = next;
            blocks = kMostBlocks;
        }
        const float p = __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.f : m));
        const float weight = p * own_scale;
        l += p;
        const int weight_bits = __float_as_int(weight) & 0x7fffffff;
        if (blocks >= kMostBlocks || __any(weight_bits > top)) {
            flush(1.f);
            int next = weight_bits;
#pragma unroll
            for (int d = 32; d > 0; d /= 2) next = max(next, __shfl_xor(next, d));
            top = max(top, next);
            const int e = unit_exponent(top, kLeastWhole);
            to_whole = 30 - e;  // to 149: as a factor it would be infinite for weighted scales below 2^-98
            from_whole = top < 0x7f800000 ? ldexpf(digit_unit, e - 30) : NAN;
        }
        ++blocks;
        // from 2^23 on an f32 is whole: the bias rounds the weight too, to half a unit or its own last bit
        const float units = top < 0x7f800000 ? ldexpf(weight, to_whole) : 0.f;
        int bytes = static_cast<int>(units + static_cast<float>(kDigitBias)) ^ kDigitBias;
        bytes = static_cast<int>(__builtin_amdgcn_perm(in_quad<kNextLane>(bytes), bytes, first_bytes));
        bytes = static_cast<int>(__builtin_amdgcn_perm(in_quad<kOtherPair>(bytes), bytes, second_bytes));
        // the quads' digits side by side; right in the first quad's columns, which are the ones that are read
        const v4i weights{bytes, in_quad<0x12c>(bytes), in_quad<0x128>(bytes), in_quad<0x124>(bytes)};
#pragma unroll
        for (int n = 0; n < D / 16; ++n) acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[n], weights, acc[n], 0, 0, 0);
        load_values();
    }
    flush(1.f);
#pragma unroll
    for (int d = 32; d > 0; d /= 2) l += __shfl_xor(l, d);
    if (lane == 0) {
        ms[wave] = m;
        ls[wave] = l;
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
        float x = o[i];
        x += __int_as_float(in_quad<kNextLane>(__float_as_int(x)));
        x += __int_as_float(in_quad<kOtherPair>(__float_as_int(x)));
        o[i] = x;
    }
    if (column == 0)
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
            *reinterpret_cast<float4*>(&os[wave][16 * n + 4 * chunk]) = make_float4(o[4 * n], o[4 * n + 1], o[4 * n + 2], o[4 * n + 3]);
    __syncthreads();
    if (threadIdx.x >= D) return;
    const int d = threadIdx.x;
    float most = -INFINITY;
    for (int w = 0; w < Waves; ++w) most = fmaxf(most, ms[w]);
    const float base = most == -INFINITY ? 0.f : most;
    float total = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < Waves; ++w) {
        const float f = __builtin_amdgcn_exp2f(ms[w] - base);
        total += f * ls[w];
        value += f * os[w][d];
    }
    const int64_t to_row = static_cast<int64_t>(token) * heads + head;
    if (split.count == 1) {
        out[to_row * D + d] = total == 0.f ? 0.f : value / total;
    } else {
        const int64_t record = to_row * split.count + part;
        split.sums[record * D + d] = value;
        if (d == 0) {
            float* own = split.sums + static_cast<int64_t>(c.tokens) * heads * split.count * D + record * 2;
            own[0] = most;
            own[1] = total;
        }
    }
}

// Many rows a sequence (prompts): the workgroup's four waves take 16 rows each and share every block of 64 keys through LDS,
// two blocks deep, so that a wave keeps none of it in registers. Few workgroups have two such teams (G = 2) that take every
// other block: a wave alone on its SIMD takes 1.05 us for a block of 64 features, two of them 1.5 for both.
// What bounds it where workgroups are many is the vector ALU, 30 operations a score in the kernel above, seven of which join
// the digits' sums of the outputs; here the weighted sums run on the f16 matrix cores into f32, which joins nothing: a code is an f16 value as it stands,
// converted once for the four waves, and a weight times its value scale two f16 pieces (2^-23 of it), scaled so that the
// largest that the row has is 2^13 and pieces below 2^-24 are below 2^-36 of that. 2 prompts of up to 4096, 32 heads over 8 of 128:
// 428 us, 474 TFLOP/s of the formula's products, VALU busy 0.76 and matrix cores 0.42 of the cycles; 4 x 4096 of 64: 191 us, VALU
// busy 0.83. 8 of up to 1000, 12 heads of 64: 32.5 us, VALU busy 0.54: about four workgroups a CU of unlike lengths, the longest alone
// at the end.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kPromptWaves = 4;

// 16 codes as two pieces of 8 f16: 0x6400 + b is 1024 + b for a byte b, here the code + 128.
__device__ __forceinline__ void halves_of(const v4i& codes, v4i (&pieces)[2]) {
    const v2h off{static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = static_cast<uint32_t>(codes[i]) ^ 0x80808080u;
        const uint32_t low = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
        const uint32_t high = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
        pieces[i / 2][2 * i % 4] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, low) + off);
        pieces[i / 2][2 * i % 4 + 1] = __builtin_bit_cast(int, __builtin_bit_cast(v2h, high) + off);
    }
}

// Which tile workgroup `index` of a kv head's `tiles` takes. The tiles at the ends of the sequences see most keys; where they are
// few enough to be counted out (up to 64 sequences of up to 64 tiles) all sequences' last tiles go first, so that no long
// one begins late: 8 x 1000 52 -> 44 us. Otherwise a sequence's tiles go from the last to the first. `base` becomes the tile's
// distance from its sequence's first.
__device__ __forceinline__ Found find_tile(const Paged& c, int index, int tiles, int group) {
    const int lane = threadIdx.x % 64;
    if (c.sequences <= 64) {
        const Rows rows = rows_of(c, min(lane, c.sequences - 1));
        const int own = lane < c.sequences ? (rows.count * group + kTileRows - 1) / kTileRows : 0;
        int most = own;
#pragma unroll
        for (int d = 32; d > 0; d /= 2) most = max(most, __shfl_xor(most, d));
        most = __builtin_amdgcn_readfirstlane(most);
        if (most <= 64) {
            int before = 0;
            for (int j = most - 1; j >= 0; --j) {
                uint64_t have = __ballot(own > j);
                const int n = __popcll(have);
                if (index < before + n) {
                    for (int i = before; i < index; ++i) have &= have - 1;
                    const int s = __ffsll(static_cast<unsigned long long>(have)) - 1;
                    return {s, j, from_lane(rows, s)};
                }
                before += n;
            }
            return {-1, 0, {}};
        }
    }
    const int64_t tile = tiles - 1 - index;
    Found found = find_sequence(c, tile, [&](int64_t start, int64_t at) { return tile_base(start, at, group); });
    found.base = tile - found.base;
    return found;
}

// A lane's 16 features of a query row as f16 pieces, the larger parts and the rest, of 2^(15 - e) times their value, e being
// the exponent of the row's largest; the factor as query_digits gives it.
__device__ __forceinline__ float query_halves(float (&features)[16], bool real, double scale, v8h (&high)[2], v8h (&low)[2]) {
    int bits = 0;
#pragma unroll
    for (int d = 0; d < 16; ++d) {
        features[d] = real ? features[d] : 0.f;
        bits = max(bits, __float_as_int(features[d]) & 0x7fffffff);
    }
    bits = over_chunks(bits, [](int a, int b) { return max(a, b); });
    const int e = __builtin_amdgcn_frexp_expf(__int_as_float(bits));
    const float sign = scale < 0 ? -1.f : 1.f;
#pragma unroll
    for (int d = 0; d < 16; ++d) {
        const float x = ldexpf(features[d] * sign, 15 - e);
        high[d / 8][d % 8] = static_cast<_Float16>(x);
        low[d / 8][d % 8] = static_cast<_Float16>(x - static_cast<float>(high[d / 8][d % 8]));
    }
    return bits < 0x7f800000 ? static_cast<float>(ldexp(fabs(scale) * 1.4426950408889634074, e - 15)) : NAN;
}

template <int D, int G>
__global__ __launch_bounds__(G * kPromptWaves * 64, 2) void paged_prompt_kernel(Paged c, float* __restrict__ out, Strided q,
                                                                                  int heads, FastDiv by_group, double scale,
                                                                                  Split split) {
    constexpr int U = D / 64;
    constexpr int kLd = D + 4;
    // Heads of 64 take the keys as f16 too, which spares joining the scores' digits; at 128 LDS would hold a workgroup less.
    constexpr bool kHalfKeys = D == 64;
    constexpr int kKeyPieces = 8, kValuePieces = 2 * D / 16;  // of 64 lanes' 16 bytes
    union Shared {
        v4i block[G][2][kKeyPieces + kValuePieces][64];
        float os[G * kPromptWaves][kRowTile][kLd];
    };
    __shared__ __attribute__((aligned(16))) Shared shared;
    __shared__ float ms[G * kPromptWaves][kRowTile], ls[G * kPromptWaves][kRowTile];
    const int group = static_cast<int>(by_group.divisor);
    const int any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int wave = any_wave % kPromptWaves, team = any_wave / kPromptWaves;
    const int column = lane % 16, chunk = lane / 16;
    const int part = blockIdx.y, kv = static_cast<int>(blockIdx.x % c.kv_heads);
    const Found found = find_tile(c, static_cast<int>(blockIdx.x) / c.kv_heads, static_cast<int>(gridDim.x) / c.kv_heads, group);
    if (found.s < 0) return;
    const Rows rows = found.rows;
    const int64_t tile_at = found.base * kTileRows;
    const int row_end = rows.count * group;
    if (tile_at < 0 || tile_at >= row_end) return;
    const int row0 = static_cast<int>(tile_at);
    const int here = min(row_end - row0, kTileRows);
    const int64_t capacity = static_cast<int64_t>(c.columns) << c.page_shift;
    const auto limit_of = [&](int token) {
        const int64_t limit = rows.position + token + 1;
        return static_cast<int>(limit < 0 ? 0 : limit > capacity ? capacity : limit);
    };
    const auto token_of = [&](int row) { return static_cast<int>(by_group.div(row)); };
    const int from = part * split.part;
    const int all = limit_of(token_of(row0 + here - 1));
    if (from >= all && part > 0) return;
    const int to = part + 1 == split.count ? all : min(all, from + split.part);
    const bool real = wave * kRowTile + column < here;
    const int r = min(row0 + wave * kRowTile + column, row0 + here - 1);
    const int token = token_of(r);
    const int limit = limit_of(token);
    const int least = __builtin_amdgcn_readfirstlane(limit);
    // a wave without rows works on nothing
    const int most = wave * kRowTile < here ? min(to, __builtin_amdgcn_readlane(limit, 15)) : 0;

    const int size = 1 << c.page_shift;
    const int64_t* table = c.table + static_cast<int64_t>(found.s) * c.columns;
    int window = 0, window_from = -128;
    const auto page_at = [&](int key) { return __shfl(window, (key >> c.page_shift) - window_from); };
    const int key_chunk = column / 4;
    // the wave's share of a block: tile `wave` of the keys, and U tiles of 16 features of the values
    v4i k[U], v[U];
    struct Scales {
        float key, value;
        int page;
    };
    Scales next;
    const uint32_t page_bytes = static_cast<uint32_t>(c.kv_heads) * size * D;  // at most 2^27
    const int8_t* keys_base = c.keys + (kv * size + 4 * wave + lane % 4) * D + chunk * 16 * U;
    const int8_t* values_base = c.values + (kv * D + 16 * U * wave + column) * size;
    const auto load = [&](int key) {
        if (((key + kKeyBlock - 1) >> c.page_shift) - window_from >= 64) {
            window_from = key >> c.page_shift;
            const int64_t page = table[min(window_from + lane, c.columns - 1)];
            window = window_from + lane < c.columns && page >= 0 && page < c.pages ? static_cast<int>(page) : -1;
        }
        next.page = page_at(key + 16 * chunk);
        const uint32_t own = max(next.page, 0), other = max(page_at(key + 16 * key_chunk), 0);
        const int slot = (key + 16 * key_chunk) & (size - 1), own_slot = (key + 16 * chunk) & (size - 1);
        const int8_t* at = keys_base + uint64_t{other} * page_bytes + slot * D;
        const int8_t* values = values_base + uint64_t{own} * page_bytes + own_slot;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = *reinterpret_cast<const v4i*>(at + 16 * u);
            v[u] = *reinterpret_cast<const v4i*>(values + 16 * u * size);
        }
        next.key = c.key_scales[uint64_t{own} * static_cast<uint32_t>(c.kv_heads) + kv];
        next.value = c.value_scales[uint64_t{own} * static_cast<uint32_t>(c.kv_heads) + kv];
    };
    const auto store = [&](int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v4i pieces[2];
            if constexpr (kHalfKeys) {
                halves_of(k[u], pieces);
#pragma unroll
                for (int h = 0; h < 2; ++h) shared.block[team][at][2 * wave + h][lane] = pieces[h];
            } else {
                shared.block[team][at][wave * U + u][lane] = k[u];
            }
            halves_of(v[u], pieces);
#pragma unroll
            for (int h = 0; h < 2; ++h) shared.block[team][at][kKeyPieces + 2 * (wave * U + u) + h][lane] = pieces[h];
        }
    };

    const float* row = q.data + (rows.row + token) * q.row + (kv * group + r - token * group) * q.head + chunk * 16 * U;
    float features[16 * U];
#pragma unroll
    for (int d = 0; d < 16 * U; ++d) features[d] = row[d];
    const int first = from + team * kKeyBlock;
    constexpr int step = G * kKeyBlock;
    if (first < to) load(first);
    v4i digits[4][U];
    v8h q_high[2], q_low[2];
    float q_factor;
    if constexpr (kHalfKeys) q_factor = query_halves(features, real, scale, q_high, q_low);
    else q_factor = query_digits(features, real, scale, digits);

    float m = -INFINITY, l = 0.f;
    v4f o[D / 16] = {};  // in units of 2^(top_exponent - 13)
    // the largest weight times its value scale that the row has seen, in units of its maximum, as bits, so that NaN is the
    // largest of all, and its exponent
    int top = 0, top_exponent = 0, scale_limit = 0;
    const auto work = [&](int key, const Scales& own, const v4i (*block)[64]) {
        float x[16];
        // Heads of 64: pieces are read four at a time ahead of their use, where the scheduler would put them right before it.
        // At 128 the registers for that cost a wave on the SIMD (2 x 4096 530 -> 565 us; 8 x 1000 of 64 56 -> 53 us).
        constexpr bool kAhead = D == 64;
        v4i ahead[4];
        const auto read = [&](int first) {
            if constexpr (kAhead) {
#pragma unroll
                for (int i = 0; i < 4; ++i) ahead[i] = block[first + i][lane];
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        read(0);
        if constexpr (kHalfKeys) {
#pragma unroll
            for (int t = 0; t < 4; t += 2) {
                v4i held[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) held[i] = ahead[i];
                read(t == 0 ? 4 : kKeyPieces);
                v4f sum[2] = {};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tile = i % 2, h = i / 2;
                    const v8h keys = __builtin_bit_cast(v8h, held[2 * tile + h]);
                    sum[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, q_low[h], sum[tile], 0, 0, 0);
                    sum[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, q_high[h], sum[tile], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) x[4 * t + i] = sum[i / 4][i % 4];
            }
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                v4i sum[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) sum[p] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const v4i piece = block[t * U + u][lane];
#pragma unroll
                    for (int p = 0; p < 4; ++p) sum[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(piece, digits[p][u], sum[p], 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[4 * t + i] = joined(sum, i);
                    asm("" : "+v"(x[4 * t + i]));  // joined here, not behind the branch below with every tile's sums held
                }
            }
        }
        const int seen = own.page < 0 ? 0 : limit - (key + 16 * chunk);
        float factor = score_factor(q_factor, own.key);
        factor = factor == 0.f ? 0x1p-126f : factor;
        if (key + kKeyBlock > least || __any(own.page < 0)) {
            factor = seen > 0 ? factor : 1.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = i < seen ? x[i] : -INFINITY;
        }
        float largest = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) largest = fmaxf(largest, x[i]);
        largest *= factor;
        const int scale_bits = seen > 0 ? __float_as_int(own.value) & 0x7fffffff : 0;
        // A scale of up to four units' largest weight fits whatever its weight; a larger one only if its weight makes it so, and where
        // that is looked at the unit goes by the weights: one page of far larger values takes no bits from the others.
        if (__any(largest > m || scale_bits > scale_limit)) {
            const float next = fmaxf(m, chunks_max(largest)), to = next == -INFINITY ? 0.f : next;
            const float alpha = __builtin_amdgcn_exp2f(m - to);
            l *= alpha;
            m = next;
            const int weight_bits = __float_as_int(__builtin_amdgcn_exp2f(largest - to) * own.value) & 0x7fffffff;
            top = max(__float_as_int(__int_as_float(top) * alpha) & 0x7fffffff,
                      over_chunks(seen > 0 ? max(weight_bits, scale_bits - kFarBelow) : 0, [](int a, int b) { return max(a, b); }));
            const int next_exponent = unit_exponent(top, kLeastHalf);
            const float again = ldexpf(alpha, top_exponent - next_exponent);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) o[n] *= again;
            top_exponent = next_exponent;
            scale_limit = min(__float_as_int(ldexpf(4.f, top_exponent)), 0x7f7fffff);  // infinity and NaN are always looked at
        }
        const float base = m == -INFINITY ? 0.f : m;  // nothing seen yet: every weight below is 0
        if (__any(fabsf(base) >= kFarScore)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = rounded_product(x[i], factor);
            factor = 1.f;
        }
        // the scale multiplies the weight rather than going into the exponent, whose rounding would differ from chunk to chunk
        const float to_units = top < 0x7f800000 && seen > 0 ? ldexpf(own.value, 13 - top_exponent) : 0.f;
        float sum = 0.f;
        v8h high[2], low[2];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const v2f p{__builtin_amdgcn_exp2f(fmaf(x[i], factor, -base)), __builtin_amdgcn_exp2f(fmaf(x[i + 1], factor, -base))};
            sum += p[0];
            sum += p[1];
            const v2f w{p[0] * to_units, p[1] * to_units};
            const v2h a = __builtin_convertvector(w, v2h);
            const v2f rest{w[0] - static_cast<float>(a[0]), w[1] - static_cast<float>(a[1])};
            const v2h b = __builtin_convertvector(rest, v2h);
            high[i / 8][i % 8] = a[0];
            high[i / 8][i % 8 + 1] = a[1];
            low[i / 8][i % 8] = b[0];
            low[i / 8][i % 8 + 1] = b[1];
        }
        l += sum;
        // four pieces are the values of two tiles of features, each the first half of the keys and the second
#pragma unroll
        for (int n = 0; n < D / 16; n += 2) {
            v4i held[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) held[i] = ahead[i];
            if (n + 2 < D / 16) read(kKeyPieces + 2 * (n + 2));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tile = i % 2, h = i / 2;
                const v8h values = __builtin_bit_cast(v8h, kAhead ? held[2 * tile + h] : block[kKeyPieces + 2 * (n + tile) + h][lane]);
                o[n + tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values, low[h], o[n + tile], 0, 0, 0);
                o[n + tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values, high[h], o[n + tile], 0, 0, 0);
            }
        }
    };

    if (from < to) {
        Scales own = next;
        if (first < to) store(0);
        if (first + step < to) load(first + step);
        __syncthreads();
        int buffer = 0;
        for (int key = first; key - team * kKeyBlock < to; key += step) {
            const Scales following = next;
            if (key + step < to) {
                store(buffer ^ 1);
                if (key + 2 * step < to) load(key + 2 * step);
            }
            if (key < most) work(key, own, shared.block[team][buffer]);
            own = following;
            buffer ^= 1;
            // the block stored is complete, and the one worked on free
            __syncthreads();
        }
    }
    l = chunks_sum(l);
    const float unit = top < 0x7f800000 ? ldexpf(1.f, top_exponent - 13) : NAN;
    if (chunk == 0) {
        ms[any_wave][column] = m;
        ls[any_wave][column] = l;
    }
#pragma unroll
    for (int n = 0; n < D / 16; ++n) *reinterpret_cast<v4f*>(&shared.os[any_wave][column][16 * n + 4 * chunk]) = o[n] * unit;
    __syncthreads();
    for (int i = threadIdx.x; i < here * (D / 4); i += G * kPromptWaves * 64) {
        const int at = i / (D / 4), d = i % (D / 4) * 4;
        const int w = at / kRowTile, col = at % kRowTile;
        // the teams joined, in their order
        float largest = ms[w][col], sum = ls[w][col];
        v4f sums = *reinterpret_cast<const v4f*>(&shared.os[w][col][d]);
        if constexpr (G == 2) {
            const int other = w + kPromptWaves;
            const float top = fmaxf(largest, ms[other][col]), base = top == -INFINITY ? 0.f : top;
            const float f = __builtin_amdgcn_exp2f(largest - base), g = __builtin_amdgcn_exp2f(ms[other][col] - base);
            sum = f * sum + g * ls[other][col];
            sums = sums * f + *reinterpret_cast<const v4f*>(&shared.os[other][col][d]) * g;
            largest = top;
        }
        const int of_token = token_of(row0 + at);
        const int64_t to_row = static_cast<int64_t>(rows.row + of_token) * heads + kv * group + (row0 + at - of_token * group);
        if (split.count == 1) {
            *reinterpret_cast<v4f*>(out + to_row * D + d) = sums * (sum == 0.f ? 0.f : 1.f / sum);
        } else {
            const int64_t record = to_row * split.count + part;
            *reinterpret_cast<v4f*>(split.sums + record * D + d) = sums;
            if (d == 0) {
                float* own = split.sums + static_cast<int64_t>(c.tokens) * heads * split.count * D + record * 2;
                own[0] = largest;
                own[1] = sum;
            }
        }
    }
}

// The parts of a row joined, in their order: one wave a row. Bound by its launch and one chain of loads, 4 us.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(Paged c, float* __restrict__ out, int heads, Split split) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64;  // token * heads + head
    const int lane = threadIdx.x % 64;
    if (row >= static_cast<int64_t>(c.tokens) * heads) return;
    const int token = static_cast<int>(row / heads);
    const Found found = find_sequence(c, token, [&](int64_t start, int64_t) { return start; });
    if (found.s < 0) return;
    const Rows rows = found.rows;
    if (token >= rows.row + rows.count) return;
    const int64_t limit = min(rows.position + (token - rows.row) + 1, static_cast<int64_t>(c.columns) << c.page_shift);
    // the parts that begin before the row's limit were worked on, and the first one always
    const int parts = static_cast<int>(max(int64_t{1}, min(int64_t{split.count}, (limit + split.part - 1) / split.part)));
    const float* sums = split.sums + row * split.count * D;
    const float* ml = split.sums + static_cast<int64_t>(c.tokens) * heads * split.count * D + row * split.count * 2;
    // a lane holds a part's maximum and sum, 64 parts at a time
    float top = -INFINITY, sum = 0.f, v[D / 64] = {};
    for (int p0 = 0; p0 < parts; p0 += 64) {
        const bool in = p0 + lane < parts;
        const float own = in ? ml[2 * (p0 + lane)] : -INFINITY;
        const float own_sum = in ? ml[2 * (p0 + lane) + 1] : 0.f;
        float next = own;
#pragma unroll
        for (int d = 32; d > 0; d /= 2) next = fmaxf(next, __shfl_xor(next, d));
        next = fmaxf(next, top);
        const float base = next == -INFINITY ? 0.f : next;
        const float again = __builtin_amdgcn_exp2f(top - base), f = __builtin_amdgcn_exp2f(own - base);
        float add = f * own_sum;
#pragma unroll
        for (int d = 32; d > 0; d /= 2) add += __shfl_xor(add, d);
        sum = sum * again + add;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) v[u] *= again;
        const int count = min(64, parts - p0);
        // eight parts' loads at a time; past the last one it is read again, for nothing
        for (int p = 0; p < count; p += 8) {
            float x[8][D / 64];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int u = 0; u < D / 64; ++u) x[i][u] = sums[(p0 + min(p + i, count - 1)) * D + 64 * u + lane];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float by = p + i < count ? __shfl(f, p + i) : 0.f;
#pragma unroll
                for (int u = 0; u < D / 64; ++u) v[u] += by * x[i][u];
            }
        }
        top = next;
    }
#pragma unroll
    for (int u = 0; u < D / 64; ++u) out[row * D + 64 * u + lane] = sum == 0.f ? 0.f : v[u] / sum;
}

// Bytes of a part's results of `rows` rows.
int64_t part_bytes(int64_t rows, int64_t dim) { return rows * (dim + 2) * 4; }

// How a call runs: on which kernel, with how many waves that share a tile's keys, and in how many parts of the keys.
struct Plan {
    bool prompts, single;
    int waves;    // of a workgroup; prompts: two teams of four, or one
    int columns;  // of the matrix instruction for a row (paged_attention_kernel)
    int64_t tiles;
    Split split;
};

Plan plan_of(int64_t heads, int64_t kv_heads, int64_t dim, int64_t sequences, int64_t tokens, int64_t max_keys, int64_t most) {
    Plan plan;
    const int64_t group = heads / kv_heads, rows = tokens * group, cus = compute_units();
    const bool narrow = dim == 64;
    const int64_t keys = std::min<int64_t>(std::max<int64_t>(max_keys, 1), int64_t{1} << 30);
    // By the rows of a sequence's kv head on average. From 33 on the prompts' kernel; 32 sequences of 1000 keys, 12 heads of 64,
    // 16 rows a tile / prompts, us: 16 rows 13 / 28, 32 rows 21 / 34, 48 rows 39 / 35, 64 rows 43 / 36.
    plan.prompts = rows > 32 * sequences;
    // One row: 64 x 1024 keys of 64, 12 heads, 16 rows a tile / single 18.6 / 16.4 us, 16 x 4000 21.5 / 16.5; of 128, 16 heads,
    // 32 x 2000 37.8 / 36.1.
    plan.single = rows <= sequences;
    // Up to 8 and up to 4 rows, 16 / 8 / 4 rows a tile: 5 rows, 32 x 2000, 12 heads of 64 21.0 / 18.2 / 21.3 us, 4 rows, 64 x 4000,
    // 4 kv heads 31.7 / 26.2 / 23.8; of 128 4 rows, 16 x 2000, 8 kv heads 20.4 / 19.8 / 19.7, and 64 x 500, 4 kv heads
    // 10.2 / 10.3 / 14.3, whose tiles of 4 rows leave more workgroups empty than a round of the CUs has room for.
    plan.columns = narrow && rows <= 4 * sequences ? 4 : rows <= 8 * sequences ? 2 : 1;
    const int64_t tile_rows = kTileRows / plan.columns;
    plan.tiles = tile_base(tokens, sequences, static_cast<int>(group), static_cast<int>(tile_rows));
    // the workgroups with work, if the sequences are alike
    const int64_t working = std::max<int64_t>(1, plan.single ? tokens * heads
                                                             : std::max(sequences, (rows + tile_rows - 1) / tile_rows) * kv_heads);
    const int64_t grid = plan.single ? working : std::max<int64_t>(1, plan.tiles * kv_heads);  // with those that find none
    int64_t count, least = 512;  // parts, and the keys that one is worth
    if (plan.prompts) {
        // up to half of the CUs in one launch take parts, and up to all of them for long keys: one launch / parts, us: 300 new ones
        // over 8000 of 128, 152 workgroups, 152 / 123, 1000 over 16000 of 64, 188, 183 / 152, 300 over 3000, 240, 39.8 / 40.0
        const bool whole = working > cus || (2 * working > cus && keys <= 4096);
        count = whole ? 1 : ((narrow ? 4 : 2) * cus + working - 1) / working;
    } else {
        // Parts where there are few workgroups of many keys. One launch / parts, us: of 64, one row, 12 x 2000 keys 8.5 / 10.4,
        // x 4000 11.2 / 10.8, x 8000 17.2 / 10.9, 96 x 4000 13.1 / 13.3, 192 x 8000 27.7 / 30.9; four rows, 32 x 2000 8.8 / 11.4,
        // x 4000 12.9 / 11.0, 128 x 2000 9.1 / 11.7; five, 96 x 4000 16.3 / 15.0; of 128, one row, 16 x 1000 10.8 / 10.6,
        // x 2000 16.1 / 10.6, 128 x 2000 17.1 / 17.0, x 4000 27.3 / 24.6, 256 x 4000 37.1 / 41.1; four rows, 8 x 4000 26.8 / 11.4,
        // 128 x 2000 17.9 / 19.1.
        const int64_t few = narrow ? (plan.single ? 4096 : 2048) : 2 * working >= cus ? 2048 : 1024;
        const bool whole = keys <= few || 4 * working >= 3 * cus;
        // Of 64, two workgroups a CU, four for 9 rows and more (68 x 20000, 24 rows, in 4 / 8 / 16 parts 83 / 64 / 48 us; 4 rows
        // 31.4 / 31.1 / 29.0). Of 128, one or else two: a CU with one more than the others is what the call waits for (96 x 8000 in
        // 2 / 3 / 5 parts 33.7 / 41.8 / 36.0, 32 x 40000 in 4 / 8 / 16 66.6 / 46.5 / 49.4), two from 17 rows on (68 x 10000, 24
        // rows, in 3 / 7 / 8 67 / 47 / 43).
        if (narrow) count = ((plan.columns == 1 ? 4 : 2) * cus + working - 1) / working;
        else if (rows > 16 * sequences) count = 2 * cus / working;
        else count = cus / grid > 1 ? cus / grid : 2 * cus / grid;
        if (whole) count = 1;
        if (!narrow) least = 256;
    }
    // no part longer than about 8192 keys
    count = std::max<int64_t>(1, std::min({std::max(count, keys / 8192), keys / least, most, int64_t{65535}}));
    // Eight waves for the latency of a CU's only workgroup. Four / eight, us: of 64, one row, 12 x 2000 9.5 / 8.5, 192 x 4000
    // 18.0 / 16.4, 384 x 2000 16.7 / 17.3; four rows, 128 x 2000 10.0 / 9.1, 256 x 1000 9.0 / 9.6. Keys of 128 keep a CU at the
    // 50 GB/s that it takes with four: 16 x 1000 10.8 / 11.3, 256 x 500 (288 workgroups) 11.6 / 10.2, 237 x 574 of 8 rows (294) 14.1 /
    // 19.4, 220 x 500 of 12 rows 14.1 / 20.0, 384 x 1000 19.3 / 25.1.
    plan.waves = count == 1 && (narrow ? working < cus : plan.columns > 1 && 4 * working >= 3 * cus && 8 * grid <= 9 * cus) ? 8 : 4;
    // Prompts: two teams where the workgroups are few. One / two, us: 12 heads of 64, 1 x 500 13.3 / 11.4, 1 x 1000 22.2 / 18.1,
    // 1 x 3000 58.5 / 52.8, 4 x 1000 25.8 / 24.1, 8 x 1000 35.5 / 41.5; 32 heads over 8 of 128, 1 x 500 21.5 / 17.8, 1 x 600
    // 24.9 / 24.8, 1 x 1000 38.7 / 39.5, 4 x 1000 73 / 114; in parts 100 new ones over 8000 of 64 25.4 / 23.4, of 128 51 / 55.
    if (plan.prompts) plan.waves = working * count <= (narrow ? 3 : 1) * cus ? 8 : 4;
    constexpr int64_t unit = 256;
    const int64_t part = ((keys + count - 1) / count + unit - 1) / unit * unit;
    plan.split = {static_cast<int>((keys + part - 1) / part), static_cast<int>(part), nullptr};
    return plan;
}

// ---- checks ---------------------------------------------------------------------------------------

bool aligned(const void* p, uintptr_t by) { return reinterpret_cast<uintptr_t>(p) % by == 0; }

int check_paged(const char* what, int dtype, const kd_paged_cache* cache, const kd_paged_batch* batch, Paged& c) {
    const std::string name(what);
    if (dtype != KD_F32) return fail(KD_E_UNSUPPORTED, name + ": dtype must be f32");
    if (cache == nullptr || batch == nullptr) return fail(KD_E_INVALID, name + ": cache and batch must be given");
    if (cache->head_dim != 64 && cache->head_dim != 128)
        return fail(KD_E_UNSUPPORTED, name + ": head dim must be 64 or 128");
    int shift = 4;
    while (shift < 8 && (int64_t{1} << shift) != cache->page_size) ++shift;
    if ((int64_t{1} << shift) != cache->page_size)
        return fail(KD_E_UNSUPPORTED, name + ": page size must be 16, 32, 64, 128 or 256");
    if (cache->kv_heads < 1 || cache->kv_heads > 4096 || cache->pages < 0 || cache->pages >= (int64_t{1} << 31))
        return fail(KD_E_INVALID, name + ": bad number of kv heads or pages");
    if (batch->sequences < 0 || batch->table_columns < 0 || batch->tokens < 0 || batch->sequences >= (int64_t{1} << 24) ||
        batch->tokens >= (int64_t{1} << 31) || batch->table_columns >= (int64_t{1} << 30) >> shift)
        return fail(KD_E_INVALID, name + ": bad number of sequences, table columns or tokens");
    if (batch->sequences > 0 && batch->tokens > 0) {
        if (batch->starts == nullptr || batch->lengths == nullptr || (batch->table == nullptr && batch->table_columns > 0))
            return fail(KD_E_INVALID, name + ": table, starts and lengths must be given");
        if (cache->pages > 0 && (cache->keys == nullptr || cache->values == nullptr || cache->key_scales == nullptr ||
                                 cache->value_scales == nullptr || !aligned(cache->keys, 16) || !aligned(cache->values, 16)))
            return fail(KD_E_INVALID, name + ": the cache's arrays must be given, keys and values 16-byte aligned");
    }
    c.keys = cache->keys;
    c.values = cache->values;
    c.key_scales = cache->key_scales;
    c.value_scales = cache->value_scales;
    c.table = batch->table;
    c.starts = batch->starts;
    c.lengths = batch->lengths;
    c.pages = cache->pages;
    c.kv_heads = static_cast<int>(cache->kv_heads);
    c.head_dim = static_cast<int>(cache->head_dim);
    c.page_shift = shift;
    c.sequences = static_cast<int>(batch->sequences);
    c.columns = static_cast<int>(batch->table_columns);
    c.tokens = static_cast<int>(batch->tokens);
    return KD_OK;
}

int check_strided(const char* what, const char* operand, const void* data, const int64_t* strides, int64_t tokens,
                  int64_t heads, Strided& out) {
    const std::string name = std::string(what) + ": " + operand;
    if (data == nullptr || strides == nullptr) return fail(KD_E_INVALID, name + " and its strides must be given");
    if (!aligned(data, 4)) return fail(KD_E_INVALID, name + " must be 4-byte aligned");
    for (int d = 0; d < 2; ++d) {
        if (strides[d] < 0) return fail(KD_E_INVALID, name + " has a negative stride");
        if (strides[d] >= int64_t{1} << 40 || strides[d] * 1.0 * std::max<int64_t>(d == 0 ? tokens : heads, 1) >= 1.1e12)
            return fail(KD_E_INVALID, name + " is too large");
    }
    out = {static_cast<const float*>(data), strides[0], strides[1]};
    return KD_OK;
}

int check_heads(const char* what, int64_t heads, const Paged& c) {
    if (heads < 1 || heads > 4096 || heads % c.kv_heads != 0)
        return fail(KD_E_INVALID, std::string(what) + ": heads must be a multiple of the kv heads, at most 4096");
    if (heads * c.tokens >= (int64_t{1} << 31)) return fail(KD_E_INVALID, std::string(what) + ": too many rows");
    return KD_OK;
}

int check_grid(const char* what, int64_t groups, int64_t threads) {
    return fits_grid(groups, threads) ? KD_OK : fail(KD_E_INVALID, std::string(what) + ": shape too large");
}

} // namespace

} // namespace kd

using namespace kd;

extern "C" int kd_paged_append(int dtype, const kd_paged_cache* cache, const kd_paged_batch* batch,
                               const kd_rotation* rotation, void* q_out, const void* q, const int64_t* q_strides,
                               int64_t heads, const void* k, const int64_t* k_strides, const void* v,
                               const int64_t* v_strides) {
    const char* what = "kd_paged_append";
    Paged c;
    if (int rc = check_paged(what, dtype, cache, batch, c)) return rc;
    Rotation r{};
    if (rotation != nullptr && rotation->features != 0) {
        if (rotation->features < 0 || rotation->features % 2 != 0 || rotation->features > c.head_dim ||
            rotation->positions < 0 || (rotation->interleaved != 0 && rotation->interleaved != 1))
            return fail(KD_E_INVALID, "kd_paged_append: bad rotation");
        if (rotation->positions > 0 && (rotation->cosines == nullptr || rotation->sines == nullptr))
            return fail(KD_E_INVALID, "kd_paged_append: the rotation's tables must be given");
        r = {rotation->cosines, rotation->sines, rotation->positions, static_cast<int>(rotation->features / 2),
             rotation->interleaved != 0};
    }
    if ((q == nullptr) != (q_out == nullptr)) return fail(KD_E_INVALID, "kd_paged_append: q and q_out go together");
    if (q != nullptr && q == q_out) return fail(KD_E_INVALID, "kd_paged_append: q_out must not be q");
    if (c.sequences == 0 || c.tokens == 0) return KD_OK;
    Strided qs{}, ks, vs;
    if (q != nullptr) {
        if (int rc = check_heads(what, heads, c)) return rc;
        if (int rc = check_strided(what, "q", q, q_strides, c.tokens, heads, qs)) return rc;
        if (!aligned(q_out, 16)) return fail(KD_E_INVALID, "kd_paged_append: q_out must be 16-byte aligned");
    }
    if (int rc = check_strided(what, "k", k, k_strides, c.tokens, c.kv_heads, ks)) return rc;
    if (int rc = check_strided(what, "v", v, v_strides, c.tokens, c.kv_heads, vs)) return rc;
    // four units a thread and pass at most, one wave where few tokens a sequence leave most of a page alone
    int threads = static_cast<int>(std::clamp<int64_t>((int64_t{c.head_dim} << c.page_shift) / (4 * kUnit), 64, kAppendThreads));
    if (c.tokens <= 4 * static_cast<int64_t>(c.sequences)) threads = 64;
    const int64_t cache_groups = page_base(c.tokens, c.sequences, c.page_shift) * c.kv_heads * 2;
    const int64_t per_token = heads * (c.head_dim / kUnit);
    const int q_tokens = q == nullptr ? 1 : static_cast<int>(std::max<int64_t>(1, threads / per_token));
    const int64_t q_groups = q == nullptr ? 0 : (c.tokens + q_tokens - 1) / q_tokens;
    if (int rc = check_grid(what, cache_groups + q_groups, threads)) return rc;
    if (int rc = ensure_device()) return rc;
    // 16-byte pieces need rows and tables that keep them aligned and pairs that come in fours
    const auto whole = [](const Strided& x) { return aligned(x.data, 16) && x.row % 4 == 0 && x.head % 4 == 0; };
    const bool vector = r.half % 4 == 0 && aligned(r.cosines, 16) && aligned(r.sines, 16) && whole(ks) && (q == nullptr || whole(qs));
    // Large queries are loaded past the caches, and the keys the second time: what they leave there is the second reading of the keys
    // and values. They are stored through them, for the attention reads them next. Append and attention, us, all through the caches /
    // loads past them / stores too, by the bytes of q: 40 MB 227.3 / 226.8 / 228.1, 67 MB 321.7 / 321.8 / 322.5, 104 MB 187.8 / 186.5 / 191.0
    // and 270.2 / 267.2 / 273.9, 113 MB 483.1 / 482.6 / 486.5, 203 MB 361.5 / 358.1 / 358.6; the append and a reading of its pages alone
    // take 85 / 82 / 72 at 104 MB.
    const bool past = q != nullptr && vector && int64_t{c.tokens} * heads * c.head_dim * 4 > kPastBytes;
    const auto launch = [&](auto dim, auto aligned_pieces, auto past_caches) {
        constexpr int D = decltype(dim)::value;
        hipLaunchKernelGGL((paged_append_kernel<D, decltype(aligned_pieces)::value, decltype(past_caches)::value>),
                           dim3(static_cast<uint32_t>(cache_groups + q_groups)), dim3(threads), 0, stream(), c, r, ks, vs, qs,
                           static_cast<float*>(q_out), static_cast<int>(heads), cache_groups, q_tokens);
    };
    const auto with_dim = [&](auto aligned_pieces, auto past_caches) {
        if (c.head_dim == 64) launch(std::integral_constant<int, 64>{}, aligned_pieces, past_caches);
        else launch(std::integral_constant<int, 128>{}, aligned_pieces, past_caches);
    };
    if (past) with_dim(std::true_type{}, std::true_type{});
    else if (vector) with_dim(std::true_type{}, std::false_type{});
    else with_dim(std::false_type{}, std::false_type{});
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_paged_read(int dtype, void* k, void* v, const kd_paged_cache* cache, const kd_paged_batch* batch) {
    Paged c;
    if (int rc = check_paged("kd_paged_read", dtype, cache, batch, c)) return rc;
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(KD_E_INVALID, "kd_paged_read: k and v must be 16-byte aligned");
    if (c.sequences == 0 || c.tokens == 0 || (k == nullptr && v == nullptr)) return KD_OK;
    const int64_t groups = page_base(c.tokens, c.sequences, c.page_shift) * c.kv_heads * 2;
    const int threads = c.page_shift <= 5 ? 64 : 256;
    if (int rc = check_grid("kd_paged_read", groups, threads)) return rc;
    if (int rc = ensure_device()) return rc;
    hipLaunchKernelGGL(paged_read_kernel, dim3(static_cast<uint32_t>(groups)), dim3(threads), 0, stream(), c, static_cast<float*>(k),
                       static_cast<float*>(v));
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_paged_attention_workspace(int64_t* bytes, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                            int64_t sequences, int64_t tokens, int64_t max_keys) {
    if (bytes == nullptr || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 4096 ||
        (head_dim != 64 && head_dim != 128) || sequences < 0 || sequences >= int64_t{1} << 24 || tokens < 0 ||
        tokens >= int64_t{1} << 31 || heads * tokens >= int64_t{1} << 31 || max_keys < 0)
        return fail(KD_E_INVALID, "kd_paged_attention_workspace: bad arguments");
    const Split split = plan_of(heads, kv_heads, head_dim, sequences, tokens, max_keys, INT32_MAX).split;
    *bytes = split.count > 1 ? split.count * part_bytes(tokens * heads, head_dim) : 0;
    return KD_OK;
}

extern "C" int kd_paged_attention(int dtype, void* out, const void* q, const int64_t* q_strides, int64_t heads,
                                  const kd_paged_cache* cache, const kd_paged_batch* batch, double scale, int64_t max_keys,
                                  void* workspace, int64_t workspace_bytes) {
    const char* what = "kd_paged_attention";
    Paged c;
    if (int rc = check_paged(what, dtype, cache, batch, c)) return rc;
    if (int rc = check_heads(what, heads, c)) return rc;
    if (!std::isfinite(scale)) return fail(KD_E_INVALID, "kd_paged_attention: scale must be finite");
    if (max_keys < 0 || workspace_bytes < 0 || (workspace == nullptr && workspace_bytes > 0) || !aligned(workspace, 16))
        return fail(KD_E_INVALID, "kd_paged_attention: bad max_keys or workspace");
    if (c.sequences == 0 || c.tokens == 0) return KD_OK;
    Strided qs;
    if (int rc = check_strided(what, "q", q, q_strides, c.tokens, heads, qs)) return rc;
    if (out == nullptr || !aligned(out, 16)) return fail(KD_E_INVALID, "kd_paged_attention: out must be given, 16-byte aligned");
    // the most workgroups that a plan has, of at most 512 threads
    if (int rc = check_grid(what, tile_base(c.tokens, c.sequences, static_cast<int>(heads / c.kv_heads), kTileRows / 4) * c.kv_heads, 512))
        return rc;
    if (int rc = ensure_device()) return rc;
    if (c.pages == 0) c.columns = 0;  // no position has a page
    const int64_t rows = heads * c.tokens;
    const int64_t join_groups = (rows + 3) / 4;
    const int64_t most = fits_grid(join_groups, 256) ? workspace_bytes / part_bytes(rows, c.head_dim) : 1;
    const Plan plan = plan_of(heads, c.kv_heads, c.head_dim, c.sequences, c.tokens, max_keys, most);
    const Split split{plan.split.count, plan.split.part, static_cast<float*>(workspace)};
    const auto launch = [&](auto dim, auto waves, auto columns) {
        constexpr int D = decltype(dim)::value, Waves = decltype(waves)::value, S = decltype(columns)::value;
        hipLaunchKernelGGL((paged_attention_kernel<D, Waves, S>), dim3(static_cast<uint32_t>(plan.tiles * c.kv_heads), split.count),
                           dim3(Waves * 64), 0, stream(), c, static_cast<float*>(out), qs, static_cast<int>(heads),
                           FastDiv(static_cast<uint32_t>(heads / c.kv_heads)), scale, split);
    };
    const auto with_waves = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (plan.prompts) {
            const auto launch_prompts = [&](auto teams) {
                constexpr int G = decltype(teams)::value;
                hipLaunchKernelGGL((paged_prompt_kernel<D, G>), dim3(static_cast<uint32_t>(plan.tiles * c.kv_heads), split.count),
                               dim3(G * kPromptWaves * 64), 0, stream(), c, static_cast<float*>(out), qs, static_cast<int>(heads),
                               FastDiv(static_cast<uint32_t>(heads / c.kv_heads)), scale, split);
            };
            if (plan.waves == 8) launch_prompts(std::integral_constant<int, 2>{});
            else launch_prompts(std::integral_constant<int, 1>{});
        } else if (plan.single) {
            const auto launch_single = [&](auto waves) {
                constexpr int Waves = decltype(waves)::value;
                hipLaunchKernelGGL((paged_single_kernel<D, Waves>), dim3(static_cast<uint32_t>(rows), split.count), dim3(Waves * 64), 0,
                                   stream(), c, static_cast<float*>(out), qs, static_cast<int>(heads),
                                   FastDiv(static_cast<uint32_t>(heads / c.kv_heads)), FastDiv(static_cast<uint32_t>(heads)), scale, split);
            };
            if (plan.waves == 8) launch_single(std::integral_constant<int, 8>{});
            else launch_single(std::integral_constant<int, 4>{});
        } else {
            const auto with_columns = [&](auto columns) {
                if constexpr (D == 64 || decltype(columns)::value > 1)
                    if (plan.waves == 8) launch(dim, std::integral_constant<int, 8>{}, columns);
                if (plan.waves == 4) launch(dim, std::integral_constant<int, 4>{}, columns);
            };
            if constexpr (D == 64)
                if (plan.columns == 4) with_columns(std::integral_constant<int, 4>{});
            if (plan.columns == 2) with_columns(std::integral_constant<int, 2>{});
            if (plan.columns == 1) with_columns(std::integral_constant<int, 1>{});
        }
        if (split.count > 1)
            hipLaunchKernelGGL((paged_join_kernel<D>), dim3(static_cast<uint32_t>(join_groups)), dim3(256), 0, stream(), c,
                               static_cast<float*>(out), static_cast<int>(heads), split);
    };
    if (c.head_dim == 64) with_waves(std::integral_constant<int, 64>{});
    else with_waves(std::integral_constant<int, 128>{});
    KD_LAUNCH_CHECK();
    return KD_OK;
}
