// kd_paged.hip - the paged 8-bit key / value cache: appending rotated keys and values, reading them back, and the
// attention of ragged new queries over them.
//
// A cached value is one signed byte times the f32 scale of its page and kv head. Keys lie token by token, values feature by
// feature with a page's tokens side by side, so that both are read in 16-byte pieces along the axis that the
// attention's products sum over. Everything that a caller's arrays can say wrongly (a table entry that is no page, a
// start or a length out of range) is checked here against the sizes that the host passed.
#include <algorithm>

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

// Work is handed out by slots: sequence s owns the slots base(s) .. base(s + 1) - 1, base ascending. The sequence that slot
// `slot` belongs to, or -1 for none, found by a whole wave (every lane of it has to call this) in one load for up to
// 64 sequences, two for up to 4096.
template <class Base> __device__ __forceinline__ int find_sequence(int64_t slot, int sequences, const Base& base) {
    const int lane = threadIdx.x % 64;
    int low = 0, count = sequences;
    bool any = false;
    while (count > 1 || !any) {
        const int step = (count + 63) / 64;
        const int at = lane * step;
        const bool below = at < count && base(low + at) <= slot;
        const int n = __popcll(__ballot(below));
        if (n == 0) return -1;
        any = true;
        low += (n - 1) * step;
        count = min(step, count - (n - 1) * step);
    }
    return low;
}

// ---- append ---------------------------------------------------------------------------------------

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

// Feature d of the row x, rotated by `position`'s angle, in f64: the products of two f32 are exact there.
__device__ __forceinline__ double rotated(const float* x, int d, int64_t position, const Rotation& r) {
    if (d >= 2 * r.half) return x[d];
    const int pair = r.interleaved ? d / 2 : d % r.half;
    const bool second = r.interleaved ? d % 2 != 0 : d >= r.half;
    const double a = x[r.interleaved ? 2 * pair : pair], b = x[r.interleaved ? 2 * pair + 1 : pair + r.half];
    double c = NAN, s = NAN;
    if (position < r.positions) {
        c = r.cosines[position * r.half + pair];
        s = r.sines[position * r.half + pair];
    }
    return second ? b * c + a * s : a * c - b * s;
}

constexpr int kAppendThreads = 256;

// A sequence's new tokens touch at most (count + 2 size - 2) / size pages; base(s + 1) - base(s) is at least that.
__host__ __device__ inline int64_t append_base(int64_t start, int64_t s, int shift) {
    return (start + s * ((int64_t{2} << shift) - 2)) >> shift;
}

__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(Paged c, Rotation rotation, Strided k, Strided v,
                                                                      Strided q, float* __restrict__ q_out, int heads,
                                                                      int64_t cache_groups) {
    const int group = c.kv_heads * 2;
    if (static_cast<int64_t>(blockIdx.x) >= cache_groups) {
        // the queries, one element a thread
        const int64_t i = (static_cast<int64_t>(blockIdx.x) - cache_groups) * kAppendThreads + threadIdx.x;
        const int64_t per_row = static_cast<int64_t>(heads) * c.head_dim;
        const int first = static_cast<int>((static_cast<int64_t>(blockIdx.x) - cache_groups) * kAppendThreads / per_row);
        const int64_t row = i / per_row;
        // a wave's elements may belong to two rows: each lane looks from the first one's sequence on
        int s = find_sequence(first, c.sequences, [&](int at) { return int64_t{start_of(c, at)}; });
        s = max(s, 0);
        while (s < c.sequences && start_of(c, s + 1) <= row) ++s;
        if (row >= c.tokens || s >= c.sequences) return;
        const Rows rows = rows_of(c, s);
        if (row < rows.row) return;
        const int h = static_cast<int>(i % per_row) / c.head_dim, d = static_cast<int>(i % c.head_dim);
        const int64_t position = rows.position + (row - rows.row);
        const float* x = q.data + row * q.row + h * q.head;
        q_out[i] = position < 0 ? NAN : static_cast<float>(rotated(x, d, position, rotation));
        return;
    }
    const int64_t slot = blockIdx.x / group;
    const int h = static_cast<int>(blockIdx.x % group) / 2;
    const bool keys = blockIdx.x % 2 == 0;
    const int size = 1 << c.page_shift;
    const int s = find_sequence(slot, c.sequences, [&](int at) { return append_base(start_of(c, at), at, c.page_shift); });
    if (s < 0) return;
    const Rows rows = rows_of(c, s);
    const int64_t begin = max(rows.position, int64_t{0}), end = rows.position + rows.count;
    const int64_t column = (begin >> c.page_shift) + (slot - append_base(start_of(c, s), s, c.page_shift));
    const int64_t from = max(begin, column << c.page_shift), to = min(end, (column + 1) << c.page_shift);
    if (from >= to) return;
    const int64_t page = page_of(c, s, column);
    if (page < 0) return;
    const int held = static_cast<int>(from - (column << c.page_shift));  // slots that the page holds already
    const int count = static_cast<int>(to - from);
    const int dim = c.head_dim;
    const int64_t at = page * c.kv_heads + h;
    int8_t* codes = (keys ? c.keys : c.values) + at * size * dim;
    float* scales = keys ? c.key_scales : c.value_scales;
    const Strided in = keys ? k : v;
    const float* x = in.data + (rows.row + (from - rows.position)) * in.row + h * in.head;
    const auto value = [&](int token, int d) -> double {
        const float* row = x + token * in.row;
        return keys ? rotated(row, d, from + token, rotation) : static_cast<double>(row[d]);
    };
    double most = 0;
    for (int i = threadIdx.x; i < count * dim; i += kAppendThreads) most = max_na(most, fabs(value(i / dim, i % dim)));
    for (int m = 32; m > 0; m /= 2) most = max_na(most, __shfl_xor(most, m));
    __shared__ double wave_most[kAppendThreads / 64];
    if (threadIdx.x % 64 == 0) wave_most[threadIdx.x / 64] = most;
    const float old = held > 0 ? scales[at] : 0.f;
    __syncthreads();
    for (int w = 0; w < kAppendThreads / 64; ++w) most = max_na(most, wave_most[w]);
    const float scale = most < INFINITY ? max_na(old, static_cast<float>(most / 127)) : NAN;
    if (threadIdx.x == 0) scales[at] = scale;
    const double inverse = scale > 0 ? 1.0 / scale : 0.0;  // 0 for NaN too
    for (int i = threadIdx.x; i < count * dim; i += kAppendThreads) {
        const int token = i / dim, d = i % dim;
        const double r = rint(value(token, d) * inverse);
        const int code = r != r ? 0 : static_cast<int>(fmin(fmax(r, -127.0), 127.0));
        codes[keys ? (held + token) * dim + d : d * size + held + token] = static_cast<int8_t>(code);
    }
    if (scale > old) {
        const double ratio = static_cast<double>(old) / scale;
        for (int i = threadIdx.x; i < held * dim; i += kAppendThreads) {
            int8_t* p = codes + (keys ? i : i / held * size + i % held);
            *p = static_cast<int8_t>(rint(*p * ratio));
        }
    }
}

// ---- read -----------------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void paged_read_kernel(Paged c, float* __restrict__ k, float* __restrict__ v) {
    const int64_t row = blockIdx.x;
    const int s = find_sequence(row, c.sequences, [&](int at) { return int64_t{start_of(c, at)}; });
    if (s < 0) return;
    const Rows rows = rows_of(c, s);
    if (row >= rows.row + rows.count) return;
    const int64_t position = rows.position + (row - rows.row);
    const int64_t page = position < 0 ? -1 : page_of(c, s, position >> c.page_shift);
    const int size = 1 << c.page_shift, slot = static_cast<int>(position & (size - 1));
    for (int i = threadIdx.x; i < c.kv_heads * c.head_dim; i += 256) {
        const int h = i / c.head_dim, d = i % c.head_dim;
        const int64_t at = page * c.kv_heads + h, base = at * size * c.head_dim;
        const int64_t to = row * c.kv_heads * c.head_dim + i;
        if (k != nullptr) k[to] = page < 0 ? 0.f : static_cast<float>(c.keys[base + slot * c.head_dim + d]) * c.key_scales[at];
        if (v != nullptr) v[to] = page < 0 ? 0.f : static_cast<float>(c.values[base + d * size + slot]) * c.value_scales[at];
    }
}

// ---- attention ------------------------------------------------------------------------------------

// One workgroup a (row, head), a key a thread at a time: the scores of 256 keys, then each thread a feature's sum.
__global__ __launch_bounds__(256) void paged_attention_kernel(Paged c, float* __restrict__ out, Strided q, int heads,
                                                              float scale) {
    __shared__ float qs[128], weights[256], parts[8];
    const int64_t row = blockIdx.x / heads;
    const int h = blockIdx.x % heads, kv = h / (heads / c.kv_heads);
    const int s = find_sequence(row, c.sequences, [&](int at) { return int64_t{start_of(c, at)}; });
    if (s < 0) return;
    const Rows rows = rows_of(c, s);
    if (row >= rows.row + rows.count) return;
    const int64_t limit = min(rows.position + (row - rows.row) + 1, static_cast<int64_t>(c.columns) << c.page_shift);
    const int size = 1 << c.page_shift, dim = c.head_dim, t = threadIdx.x;
    if (t < dim) qs[t] = q.data[row * q.row + h * q.head + t];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int64_t j0 = 0; j0 < limit; j0 += 256) {
        const int64_t j = j0 + t;
        const int64_t page = j < limit ? page_of(c, s, j >> c.page_shift) : -1;
        float score = -INFINITY;
        if (page >= 0) {
            const int8_t* key = c.keys + ((page * c.kv_heads + kv) * size + (j & (size - 1))) * dim;
            float sum = 0.f;
            for (int d = 0; d < dim; ++d) sum += qs[d] * key[d];
            score = sum * c.key_scales[page * c.kv_heads + kv] * scale;
        }
        float most = score;
        for (int x = 32; x > 0; x /= 2) most = max_na(most, __shfl_xor(most, x));
        if (t % 64 == 0) parts[t / 64] = most;
        __syncthreads();
        for (int w = 0; w < 4; ++w) most = max_na(most, parts[w]);
        most = max_na(m, most);
        const float p = page < 0 ? 0.f : expf(score - most);
        weights[t] = p;
        float sum = p;
        for (int x = 32; x > 0; x /= 2) sum += __shfl_xor(sum, x);
        if (t % 64 == 0) parts[4 + t / 64] = sum;
        __syncthreads();
        const float alpha = m == -INFINITY ? 0.f : expf(m - most);
        l = l * alpha + (parts[4] + parts[5] + parts[6] + parts[7]);
        m = most;
        if (t < dim) {
            o *= alpha;
            for (int i = 0; i < 256 && j0 + i < limit; ++i) {
                const int64_t value_page = page_of(c, s, (j0 + i) >> c.page_shift);
                if (value_page < 0) continue;
                const int64_t at = value_page * c.kv_heads + kv;
                o += weights[i] * (c.value_scales[at] * c.values[(at * dim + t) * size + ((j0 + i) & (size - 1))]);
            }
        }
        __syncthreads();
    }
    if (t < dim) out[(row * heads + h) * dim + t] = l == 0.f ? 0.f : o / l;
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

// A launch of `groups` workgroups in x has to stay within the grid's 2^31 - 1.
int check_grid(const char* what, int64_t groups) {
    return groups < (int64_t{1} << 31) ? KD_OK : fail(KD_E_INVALID, std::string(what) + ": shape too large");
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
    if (int rc = ensure_device()) return rc;
    const int64_t cache_groups = append_base(c.tokens, c.sequences, c.page_shift) * c.kv_heads * 2;
    const int64_t q_groups =
        q == nullptr ? 0 : (heads * c.tokens * c.head_dim + kAppendThreads - 1) / kAppendThreads;
    if (int rc = check_grid(what, cache_groups + q_groups)) return rc;
    hipLaunchKernelGGL(paged_append_kernel, dim3(static_cast<uint32_t>(cache_groups + q_groups)), dim3(kAppendThreads), 0,
                       stream(), c, r, ks, vs, qs, static_cast<float*>(q_out), static_cast<int>(heads), cache_groups);
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_paged_read(int dtype, void* k, void* v, const kd_paged_cache* cache, const kd_paged_batch* batch) {
    Paged c;
    if (int rc = check_paged("kd_paged_read", dtype, cache, batch, c)) return rc;
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(KD_E_INVALID, "kd_paged_read: k and v must be 16-byte aligned");
    if (c.sequences == 0 || c.tokens == 0 || (k == nullptr && v == nullptr)) return KD_OK;
    if (int rc = ensure_device()) return rc;
    hipLaunchKernelGGL(paged_read_kernel, dim3(static_cast<uint32_t>(c.tokens)), dim3(256), 0, stream(), c,
                       static_cast<float*>(k), static_cast<float*>(v));
    KD_LAUNCH_CHECK();
    return KD_OK;
}

extern "C" int kd_paged_attention_workspace(int64_t* bytes, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                            int64_t sequences, int64_t tokens, int64_t max_keys) {
    if (bytes == nullptr || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || head_dim < 1 || sequences < 0 ||
        tokens < 0 || max_keys < 0)
        return fail(KD_E_INVALID, "kd_paged_attention_workspace: bad arguments");
    *bytes = 0;
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
    if (int rc = ensure_device()) return rc;
    hipLaunchKernelGGL(paged_attention_kernel, dim3(static_cast<uint32_t>(heads * c.tokens)), dim3(256), 0, stream(), c,
                       static_cast<float*>(out), qs, static_cast<int>(heads), static_cast<float>(scale));
    KD_LAUNCH_CHECK();
    return KD_OK;
}
