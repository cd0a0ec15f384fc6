// attention_paged.hip -- a cache of keys and values in pages: the write of new tokens into it, and
// the attention of one new token per sequence over it,
//
//   s_p = scale (q . k_p), lse = log sum_p exp(s_p), out = sum_p exp(s_p - lse) v_p
//
// over the positions p below the sequence's length, each on the page that the table names.

#include "common.hpp"

#include <cmath>

namespace ehip {
namespace {

constexpr int kMaxDim = 128;

struct Cache {
    void *k, *v;
    int64_t pages, page_size, kv_heads, dim;
    const int32_t* table;
    int64_t ld_table, width, sequences;
};

// The row of position p of sequence s in the pools, or -1 where the table does not hold it or
// names a page outside the pool. 0 <= s < sequences.
__device__ __forceinline__ int64_t pool_row(const Cache& c, int64_t s, int64_t p) {
    if (p < 0 || p >= c.width * c.page_size) return -1;
    const int64_t at = p / c.page_size;
    const int64_t page = c.table[s * c.ld_table + at];
    if (page < 0 || page >= c.pages) return -1;
    return page * c.page_size + (p - at * c.page_size);
}

struct Bf16 {
    uint16_t bits;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(Bf16 x) {
    return __builtin_bit_cast(float, uint32_t(x.bits) << 16);
}
// The nearest value of the pool's type, ties to even.
__device__ __forceinline__ void narrow(float x, float& out) { out = x; }
__device__ __forceinline__ void narrow(float x, Bf16& out) {
    out.bits = __builtin_bit_cast(uint16_t, __bf16(x));
}

// -------------------------------------------------------------------- append

constexpr int kAppendThreads = 256;

// One token a block.
template <class T>
__global__ __launch_bounds__(kAppendThreads) void cache_append(
    Cache c, const float* __restrict__ k, int64_t ld_k, const float* __restrict__ v, int64_t ld_v,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ cu, int64_t tokens) {
    const int64_t t = blockIdx.x;
    int64_t s = t, first = t;
    if (cu != nullptr) {
        // The last sequence whose first token is not past t.
        int64_t lo = 0, hi = c.sequences;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (cu[mid] <= t) lo = mid;
            else hi = mid;
        }
        s = lo;
        first = cu[s];
        if (t < first || t >= cu[s + 1]) return;
    }
    const int64_t row = pool_row(c, s, int64_t(starts[s]) + (t - first));
    if (row < 0) return;
    const int64_t n = c.kv_heads * c.dim;
    T* dk = static_cast<T*>(c.k) + row * n;
    T* dv = static_cast<T*>(c.v) + row * n;
    for (int64_t e = threadIdx.x; e < n; e += kAppendThreads) {
        narrow(k[t * ld_k + e], dk[e]);
        narrow(v[t * ld_v + e], dv[e]);
    }
}

// ----------------------------------------------------------------- attention

// One wave for a sequence and a head: a lane for a position at a time, then a lane for a column.
template <class T>
__global__ __launch_bounds__(64) void paged_row(Cache c, const float* __restrict__ q, int64_t ld_q,
                                                int heads, const int32_t* __restrict__ lengths,
                                                int64_t longest, float scale, float* out,
                                                int64_t ld_out, float* lse) {
    const int lane = int(threadIdx.x);
    const int64_t s = blockIdx.x / heads;
    const int h = int(blockIdx.x % heads), kv = h / (heads / int(c.kv_heads)), dim = int(c.dim);
    const int64_t n = lengths[s], pitch = c.kv_heads * c.dim;
    const float* x = q + s * ld_q + int64_t(h) * dim;
    const T* k = static_cast<const T*>(c.k) + kv * dim;
    const T* v = static_cast<const T*>(c.v) + kv * dim;
    bool bad = n < 0 || n > longest || n > c.width * c.page_size;
    float m = -INFINITY;
    for (int64_t p = lane; !bad && p < n; p += 64) {
        const int64_t row = pool_row(c, s, p);
        if (row < 0) {
            bad = true;
            break;
        }
        float dot = 0.0f;
        for (int e = 0; e < dim; ++e) dot = __builtin_fmaf(x[e], widen(k[row * pitch + e]), dot);
        dot *= scale;
        if (dot != dot) bad = true;
        m = fmaxf(m, dot);
    }
    float sum = 0.0f, acc[2] = {0.0f, 0.0f};
    bad = __any(bad);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    for (int64_t p0 = 0; !bad && p0 < n; p0 += 64) {
        const int64_t p = p0 + lane;
        float w = 0.0f;
        int64_t row = 0;
        if (p < n) {
            row = pool_row(c, s, p);
            float dot = 0.0f;
            for (int e = 0; e < dim; ++e)
                dot = __builtin_fmaf(x[e], widen(k[row * pitch + e]), dot);
            w = expf(dot * scale - m) * 0x1p-24f;  // the sums stay in range with v's values
        }
        sum += w;
        const int count = n - p0 < 64 ? int(n - p0) : 64;
        for (int u = 0; u < count; ++u) {
            const float wu = __shfl(w, u);
            const int64_t at = __shfl(row, u) * pitch;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (lane + 64 * e < dim)
                    acc[e] = __builtin_fmaf(wu, widen(v[at + lane + 64 * e]), acc[e]);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < dim)
            out[s * ld_out + int64_t(h) * dim + lane + 64 * e] =
                bad ? NAN : (n == 0 ? 0.0f : acc[e] / sum);
    if (lane == 0 && lse != nullptr)
        lse[s * heads + h] = bad ? NAN : (n == 0 ? -INFINITY : m + logf(sum * 0x1p24f));
}

// ---------------------------------------------------------------- host checks

constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

int check(const char* name, const ehip_cache_t* c, Cache& out) {
    if (c == nullptr) return fail(EHIP_EINVAL, "%s: null cache", name);
    if ((c->type != EHIP_CACHE_F32 && c->type != EHIP_CACHE_BF16) || c->pages < 0 ||
        c->page_size < 1 || c->kv_heads < 1 || c->head_dim < 1 || c->sequences < 0 ||
        c->table_width < 0 || c->ld_table < c->table_width)
        return fail(EHIP_EINVAL,
                    "%s: type %d, %lld pages of %lld positions of %lld heads of %lld values, table "
                    "of %lld x %lld",
                    name, c->type, (long long)c->pages, (long long)c->page_size,
                    (long long)c->kv_heads, (long long)c->head_dim, (long long)c->sequences,
                    (long long)c->table_width);
    if (c->sequences > kMaxBlocks || c->pages > INT32_MAX || c->page_size > INT32_MAX ||
        c->table_width > INT32_MAX || c->kv_heads > kMaxBlocks || c->head_dim > kMaxBlocks)
        return fail(EHIP_EINVAL, "%s: extents past the index range", name);
    if ((c->sequences > 0 && c->table_width > 0 && c->table == nullptr) ||
        (c->pages > 0 && (c->k_pages == nullptr || c->v_pages == nullptr)))
        return fail(EHIP_EINVAL, "%s: null pool or table", name);
    out = Cache{c->k_pages, c->v_pages, c->pages, c->page_size, c->kv_heads, c->head_dim,
                c->table,   c->ld_table, c->table_width, c->sequences};
    return EHIP_OK;
}

int check_heads(const char* name, const Cache& c, int64_t heads, int64_t longest) {
    if (c.dim > kMaxDim || heads < 1 || heads % c.kv_heads != 0 || longest < 0)
        return fail(EHIP_EINVAL, "%s: %lld heads over %lld of %lld values, length %lld", name,
                    (long long)heads, (long long)c.kv_heads, (long long)c.dim, (long long)longest);
    if (heads > kMaxBlocks || c.sequences * heads > kMaxBlocks || longest > INT32_MAX)
        return fail(EHIP_EINVAL, "%s: %lld sequences of %lld heads of length %lld are too many",
                    name, (long long)c.sequences, (long long)heads, (long long)longest);
    return EHIP_OK;
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int ehip_cache_append_f32(const ehip_cache_t* cache, const float* k, int64_t ld_k, const float* v,
                          int64_t ld_v, const int32_t* starts, const int32_t* cu, int64_t tokens,
                          void* stream) {
    EHIP_READY();
    Cache c;
    if (int rc = check("cache_append", cache, c)) return rc;
    const int64_t n = c.kv_heads * c.dim;
    if (tokens < 0 || tokens > kMaxBlocks || ld_k < n || ld_v < n ||
        (cu == nullptr && tokens != c.sequences))
        return fail(EHIP_EINVAL, "cache_append: %lld tokens for %lld sequences, rows %lld and %lld "
                                 "apart",
                    (long long)tokens, (long long)c.sequences, (long long)ld_k, (long long)ld_v);
    if (tokens == 0 || c.sequences == 0) return EHIP_OK;
    if (k == nullptr || v == nullptr || starts == nullptr)
        return fail(EHIP_EINVAL, "cache_append: null tensor");
    hipStream_t s = as_stream(stream);
    if (cache->type == EHIP_CACHE_F32)
        EHIP_LAUNCH("cache_append", cache_append<float>, dim3(unsigned(tokens)),
                    dim3(kAppendThreads), 0, s, c, k, ld_k, v, ld_v, starts, cu, tokens);
    else
        EHIP_LAUNCH("cache_append", cache_append<Bf16>, dim3(unsigned(tokens)),
                    dim3(kAppendThreads), 0, s, c, k, ld_k, v, ld_v, starts, cu, tokens);
    return EHIP_OK;
}

int64_t ehip_attention_paged_workspace(const ehip_cache_t* cache, int64_t heads,
                                       int64_t longest) {
    Cache c;
    if (check("attention_paged", cache, c) || check_heads("attention_paged", c, heads, longest))
        return -1;
    return 0;
}

int ehip_attention_paged_f32(const ehip_cache_t* cache, const float* q, int64_t ld_q,
                             int64_t heads, const int32_t* lengths, int64_t longest, float scale,
                             float* out, int64_t ld_out, float* lse, void* workspace,
                             size_t workspace_bytes, void* stream) {
    EHIP_READY();
    Cache c;
    if (int rc = check("attention_paged", cache, c)) return rc;
    if (int rc = check_heads("attention_paged", c, heads, longest)) return rc;
    if (ld_q < heads * c.dim || ld_out < heads * c.dim)
        return fail(EHIP_EINVAL, "attention_paged: leading dimension below the row's length");
    if (c.sequences == 0) return EHIP_OK;
    if (q == nullptr || lengths == nullptr || out == nullptr)
        return fail(EHIP_EINVAL, "attention_paged: null tensor");
    const dim3 grid(unsigned(c.sequences * heads));
    hipStream_t s = as_stream(stream);
    if (cache->type == EHIP_CACHE_F32)
        EHIP_LAUNCH("attention_paged", paged_row<float>, grid, dim3(64), 0, s, c, q, ld_q,
                    int(heads), lengths, longest, scale, out, ld_out, lse);
    else
        EHIP_LAUNCH("attention_paged", paged_row<Bf16>, grid, dim3(64), 0, s, c, q, ld_q,
                    int(heads), lengths, longest, scale, out, ld_out, lse);
    return EHIP_OK;
}

}  // extern "C"
