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
    if (p < 0 || p > INT32_MAX || p >= c.width * c.page_size) return -1;
    const uint32_t at = uint32_t(p) / uint32_t(c.page_size);  // in 32 bits: a tenth of the steps
    const int64_t page = c.table[s * c.ld_table + at];
    if (page < 0 || page >= c.pages) return -1;
    return page * c.page_size + (p - int64_t(at) * c.page_size);
}

// log of a sum whose terms are 2^-24 of their value relative to 2^top; ln 2 in two parts.
__device__ __forceinline__ float lse_of(float top, float sum) {
    return __builtin_fmaf(top, 0.693147182464599609375f,
                          __builtin_fmaf(top, -1.904654323148236017e-9f, logf(sum * 0x1p24f)));
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

// The cache is read once and bounds the time, so the kernel's shape is that of its reads: a position's
// row of `dim` values takes LPP lanes, 16 bytes each, and a wave reads kUnroll x 64 / LPP
// positions of keys and values at a time. A lane holds its values of up to G query heads that share
// the keys. The lanes of a position add up its scores; each position's lanes keep their own running
// maximum, sum and weighted values over the positions they meet, joined at the end: of the wave, the
// block's four waves, and, where the length is split, the blocks of a sequence by a second launch.
constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / 64;
constexpr int kUnroll = 4;
constexpr int kMaxGroup = 8;  // query heads of one block

struct Paged {
    Cache c;
    const float* q;
    int64_t ld_q;
    int heads;
    const int32_t* lengths;
    int longest;
    float scale;
    float* out;
    int64_t ld_out;
    float* lse;
    int splits, chunk;   // a sequence's positions by blocks
    float2* part_stats;  // (sequences, heads, splits): maximum (as 2^x), sum
    float* part_out;     // (sequences, heads, splits, dim)
};

// x + the values of the other lanes of its group of N (the low bits of the lane number).
template <int N>
__device__ __forceinline__ float group_sum(float x) {
    if (N > 1)  // quad_perm 1 0 3 2
        x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xb1, 15, 15, true));
    if (N > 2)  // quad_perm 2 3 0 1
        x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4e, 15, 15, true));
    if (N > 4)  // row_half_mirror
        x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x141, 15, 15, true));
    if (N > 8)  // row_mirror
        x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x140, 15, 15, true));
    if (N > 16) x += __shfl_xor(x, 16);
    return x;
}

// One lane's values of a row as they are stored: 16 bytes, and its own first ones again in lanes past
// the row's end.
template <class T, bool VEC>
struct Values {
    static constexpr int N = 16 / int(sizeof(T));
    struct alignas(16) Pack {
        T v[N];
    } x;

    __device__ __forceinline__ void load(const T* row, int d0, int dim) {
        if (VEC) {
            x = *reinterpret_cast<const Pack*>(row + (d0 < dim ? d0 : 0));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) x.v[e] = row[d0 + e < dim ? d0 + e : 0];
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return widen(x.v[e]); }
};

template <class T, int LPP, int G, bool VEC>
__global__ __launch_bounds__(kPagedThreads) void paged_part(Paged a) {
    constexpr int N = 16 / int(sizeof(T)), SUBS = 64 / LPP, TILE = SUBS * kUnroll;
    __shared__ float sh_m[kPagedWaves][G], sh_l[kPagedWaves][G], sh_o[kPagedWaves][G][LPP * N];
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) / 64;
    const int kv_heads = int(a.c.kv_heads), dim = int(a.c.dim);
    const int group = a.heads / kv_heads, pieces = (group + G - 1) / G;
    uint32_t x = blockIdx.x;
    const int kv = int(x % uint32_t(kv_heads));
    x /= uint32_t(kv_heads);
    const int h0 = kv * group + int(x % uint32_t(pieces)) * G;
    const int count = min(G, (kv + 1) * group - h0);  // the block's heads
    x /= uint32_t(pieces);
    const int split = int(x % uint32_t(a.splits));
    const int64_t s = x / uint32_t(a.splits);
    const int n = a.lengths[s];
    const int64_t held = a.c.width * a.c.page_size;
    // A length that is none leaves NaN, by its first block.
    bool bad = n < 0 || n > a.longest || n > held || (n > 0 && a.c.pages == 0);
    const int begin = split * a.chunk;
    const int end = bad ? begin : min(n, begin + a.chunk);
    if (split > 0 && (bad || begin >= n)) return;

    const int sub = lane / LPP, d0 = (lane % LPP) * N, left = dim - d0;
    const float c2 = fabsf(a.scale) * 1.44269504088896340736f;
    float q[G][N], o[G][N], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
        const float* row = a.q + s * a.ld_q + int64_t(h0 + (g < count ? g : 0)) * dim + d0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            q[g][e] = e < left ? row[e] * (a.scale < 0.0f ? -c2 : c2) : 0.0f;
            o[g][e] = 0.0f;
        }
    }
    const T* const k = static_cast<const T*>(a.c.k) + int64_t(kv) * dim;
    const T* const v = static_cast<const T*>(a.c.v) + int64_t(kv) * dim;
    const int64_t pitch = int64_t(kv_heads) * dim;
    // The pool row of the tile's position `lane`.
    const auto row_of = [&](int p0) {
        const int p = p0 + lane;
        if (lane >= TILE || p >= end) return int64_t(0);
        const int64_t row = pool_row(a.c, s, p);
        if (row < 0) {
            bad = true;
            return int64_t(0);
        }
        return row;
    };
    int row = int(row_of(begin + wave * TILE));
    for (int p0 = begin + wave * TILE; p0 < end; p0 += kPagedWaves * TILE) {
        Values<T, VEC> ks[kUnroll], vs[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t at = int64_t(__shfl(row, u * SUBS + sub)) * pitch;
            ks[u].load(k + at, d0, dim);
            vs[u].load(v + at, d0, dim);
        }
        row = int(row_of(p0 + kPagedWaves * TILE));
        float kx[kUnroll][N], vx[kUnroll][N];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                kx[u][e] = ks[u][e];
                vx[u][e] = vs[u][e];
            }
        // What a lane does not have counts as 0, whatever was read in its place.
        if (dim < LPP * N) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) kx[u][e] = e < left ? kx[u][e] : 0.0f;
        }
        if (p0 + TILE > end) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) vx[u][e] = p0 + u * SUBS + sub < end ? vx[u][e] : 0.0f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float w[kUnroll], top = m[g];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float dot = 0.0f;
#pragma unroll
                for (int e = 0; e < N; ++e) dot = __builtin_fmaf(q[g][e], kx[u][e], dot);
                dot = group_sum<LPP>(dot);
                w[u] = p0 + u * SUBS + sub < end ? dot : -INFINITY;
                top = fmaxf(top, w[u]);
            }
            // Weights of 2^-24 of their value: sums over the values stay in their range.
            const float shift = top == -INFINITY ? 24.0f : top + 24.0f;
            const float keep =
                m[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[g] + 24.0f - shift);
            m[g] = top;
            l[g] *= keep;
#pragma unroll
            for (int e = 0; e < N; ++e) o[g][e] *= keep;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                w[u] = __builtin_amdgcn_exp2f(w[u] - shift);
                l[g] += w[u];
#pragma unroll
                for (int e = 0; e < N; ++e) o[g][e] = __builtin_fmaf(w[u], vx[u][e], o[g][e]);
            }
        }
    }
    bad = __syncthreads_or(bad);

    // The wave's positions, then the block's waves.
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float top = m[g];
#pragma unroll
        for (int w = LPP; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
        const float keep = m[g] == -INFINITY ? (l[g] != l[g] ? NAN : 0.0f)
                                             : __builtin_amdgcn_exp2f(m[g] - top);
        l[g] *= keep;
#pragma unroll
        for (int w = LPP; w < 64; w *= 2) l[g] += __shfl_xor(l[g], w);
        if (lane == 0) {
            sh_m[wave][g] = top;
            sh_l[wave][g] = l[g];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float y = o[g][e] * keep;
#pragma unroll
            for (int w = LPP; w < 64; w *= 2) y += __shfl_xor(y, w);
            if (sub == 0) sh_o[wave][g][d0 + e] = y;
        }
    }
    __syncthreads();
    for (int g = 0; g < count; ++g) {
        float top = sh_m[0][g], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kPagedWaves; ++w) top = fmaxf(top, sh_m[w][g]);
        float keep[kPagedWaves];
#pragma unroll
        for (int w = 0; w < kPagedWaves; ++w) {
            keep[w] = sh_m[w][g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sh_m[w][g] - top);
            sum += sh_l[w][g] * (sh_l[w][g] != sh_l[w][g] ? 1.0f : keep[w]);
        }
        const int64_t at = s * a.heads + h0 + g;
        if (bad) sum = NAN;
        if (a.splits > 1) {
            if (threadIdx.x == 0) a.part_stats[at * a.splits + split] = float2{top, sum};
        } else if (threadIdx.x == 0 && a.lse != nullptr) {
            a.lse[at] = n == 0 ? -INFINITY : lse_of(top, sum);
        }
        for (int d = int(threadIdx.x); d < dim; d += kPagedThreads) {
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < kPagedWaves; ++w) y += sh_o[w][g][d] * keep[w];
            if (a.splits > 1) a.part_out[(at * a.splits + split) * dim + d] = y;
            else a.out[s * a.ld_out + int64_t(h0 + g) * dim + d] = n == 0 ? 0.0f : y / sum;
        }
    }
}

// The blocks of a sequence and a head. Thread d % 128 has a value, two threads for alternate blocks.
__global__ __launch_bounds__(256) void paged_join(Paged a) {
    __shared__ float sh[2][kMaxDim], sh_l[2];
    const int64_t at = blockIdx.x, s = at / a.heads;
    const int h = int(at % a.heads), dim = int(a.c.dim);
    const int n = a.lengths[s];
    const bool bad = n < 0 || n > a.longest || n > a.c.width * a.c.page_size ||
                     (n > 0 && a.c.pages == 0);
    const int parts = bad ? 0 : (n + a.chunk - 1) / a.chunk;
    const int d = int(threadIdx.x) % kMaxDim, half = int(threadIdx.x) / kMaxDim;
    const float2* stats = a.part_stats + at * a.splits;
    float top = -INFINITY;
    for (int i = int(threadIdx.x) & 63; i < parts; i += 64) top = fmaxf(top, stats[i].x);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    float sum = 0.0f, y = 0.0f;
    const float* from = a.part_out + at * a.splits * dim + (d < dim ? d : 0);
#pragma unroll 4
    for (int i = half; i < parts; i += 2) {
        const float2 z = stats[i];
        const float keep = z.x == -INFINITY ? (z.y != z.y ? NAN : 0.0f)
                                            : __builtin_amdgcn_exp2f(z.x - top);
        sum += z.y * keep;
        y = __builtin_fmaf(from[int64_t(i) * dim], keep, y);
    }
    sh[half][d] = y;
    if (d == 0) sh_l[half] = sum;
    __syncthreads();
    if (half != 0) return;
    sum = sh_l[0] + sh_l[1];
    y += sh[1][d];
    if (d < dim)
        a.out[s * a.ld_out + int64_t(h) * dim + d] = bad ? NAN : (n == 0 ? 0.0f : y / sum);
    if (d == 0 && a.lse != nullptr)
        a.lse[at] = bad ? NAN : (n == 0 ? -INFINITY : lse_of(top, sum));
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
        c->table_width > INT32_MAX || c->kv_heads > kMaxBlocks || c->head_dim > kMaxBlocks ||
        c->pages * c->page_size > INT32_MAX)
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

struct Split {
    int splits, chunk;
};

// How many blocks a sequence's length is cut into, and the positions of each: enough for some
// sixteen blocks a CU over all, of 256 positions at least (below that the join costs more than the
// blocks gain).
Split split_of(const Cache& c, int64_t heads, int64_t longest) {
    const int64_t group = heads / c.kv_heads;
    const int64_t units = c.sequences * c.kv_heads * ceil_div(group, kMaxGroup);
    const int64_t most = ceil_div(longest > 0 ? longest : 1, 256);
    int64_t splits = ceil_div(4096, units > 0 ? units : 1);
    splits = splits < most ? splits : most;
    const int64_t chunk = ceil_div(ceil_div(longest > 0 ? longest : 1, splits), 64) * 64;
    return {int(ceil_div(longest > 0 ? longest : 1, chunk)), int(chunk)};
}

size_t part_bytes(const Cache& c, int64_t heads, int splits) {
    return splits > 1 ? size_t(c.sequences) * size_t(heads) * size_t(splits) *
                            (sizeof(float2) + size_t(c.dim) * sizeof(float))
                      : 0;
}

template <class T, int LPP, int G, bool VEC>
int launch_part(const Paged& a, hipStream_t s) {
    const int64_t group = a.heads / a.c.kv_heads;
    const int64_t blocks = a.c.sequences * a.splits * ceil_div(group, G) * a.c.kv_heads;
    EHIP_LAUNCH("attention_paged", (paged_part<T, LPP, G, VEC>), dim3(unsigned(blocks)),
                dim3(kPagedThreads), 0, s, a);
    return EHIP_OK;
}

template <class T, int LPP, bool VEC>
int launch_group(const Paged& a, hipStream_t s) {
    const int64_t group = a.heads / a.c.kv_heads;
    if (group == 1) return launch_part<T, LPP, 1, VEC>(a, s);
    if (group == 2) return launch_part<T, LPP, 2, VEC>(a, s);
    if (group <= 4) return launch_part<T, LPP, 4, VEC>(a, s);
    return launch_part<T, LPP, 8, VEC>(a, s);
}

template <class T, bool VEC>
int launch_lanes(const Paged& a, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    if (a.c.dim <= 32) return launch_group<T, 32 / N, VEC>(a, s);
    if (a.c.dim <= 64) return launch_group<T, 64 / N, VEC>(a, s);
    return launch_group<T, 128 / N, VEC>(a, s);
}

// 16-byte reads where every head's row begins at 16 bytes.
template <class T>
int launch_parts(const Paged& a, bool aligned, hipStream_t s) {
    return aligned && a.c.dim % int64_t(16 / sizeof(T)) == 0 ? launch_lanes<T, true>(a, s)
                                                             : launch_lanes<T, false>(a, s);
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
    return int64_t(part_bytes(c, heads, split_of(c, heads, longest).splits));
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
    const Split p = split_of(c, heads, longest);
    const size_t need = part_bytes(c, heads, p.splits);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(EHIP_EINVAL, "attention_paged: needs %zu bytes of 16-byte aligned workspace",
                    need);
    Paged a{};
    a.c = c;
    a.q = q;
    a.ld_q = ld_q;
    a.heads = int(heads);
    a.lengths = lengths;
    a.longest = int(longest);
    a.scale = scale;
    a.out = out;
    a.ld_out = ld_out;
    a.lse = lse;
    a.splits = p.splits;
    a.chunk = p.chunk;
    if (need > 0) {
        a.part_stats = static_cast<float2*>(workspace);
        a.part_out = reinterpret_cast<float*>(a.part_stats + c.sequences * heads * p.splits);
    }
    hipStream_t s = as_stream(stream);
    const bool aligned = aligned16(c.k) && aligned16(c.v);
    const int rc = cache->type == EHIP_CACHE_F32 ? launch_parts<float>(a, aligned, s)
                                                 : launch_parts<Bf16>(a, aligned, s);
    if (rc != EHIP_OK || p.splits == 1) return rc;
    EHIP_LAUNCH("attention_paged_join", paged_join, dim3(unsigned(c.sequences * heads)), dim3(256),
                0, s, a);
    return EHIP_OK;
}

}  // extern "C"
