// attention_paged.hip -- a cache of keys and values in pages: the write of new tokens into it, and
// the attention of one new token per sequence over it,
//
//   s_p = scale (q . k_p), lse = log sum_p exp(s_p), out = sum_p exp(s_p - lse) v_p
//
// over the positions p below the sequence's length, each on the page that the table names.

#include "attention_tile.hpp"
#include "common.hpp"

#include <algorithm>
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

// log of a sum whose terms are 2^-24 of their value relative to 2^top; ln 2 in two parts, whose
// products with an infinity would cancel to NaN.
__device__ __forceinline__ float lse_of(float top, float sum) {
    if (top == -INFINITY && sum == 0.0f) return -INFINITY;
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
constexpr int kAppendUnroll = 2;

// Four floats at any float's address.
using attention::floatx4u;

__device__ __forceinline__ void store4(float* to, const floatx4u& x) {
    *reinterpret_cast<floatx4u*>(to) = x;
}
__device__ __forceinline__ void store4(Bf16* to, const floatx4u& x) {
    struct alignas(8) {
        Bf16 v[4];
    } y;
#pragma unroll
    for (int e = 0; e < 4; ++e) narrow(x[e], y.v[e]);
    __builtin_memcpy(__builtin_assume_aligned(to, 8), &y, 8);
}

// The last sequence whose first token is not past t: 64 candidates at a time, a lane each.
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ cu, int sequences, int t) {
    const int lane = int(threadIdx.x) & 63;
    int lo = 0, n = sequences;  // the answer, if any, is in [lo, lo + n)
    while (true) {
        const int step = (n + 63) / 64;
        const int at = lane * step;
        const int c = __popcll(__ballot(at < n && cu[at < n ? lo + at : lo] <= t));
        if (c == 0) return lo;
        lo += (c - 1) * step;
        n = min(n - (c - 1) * step, step);
        if (step == 1) return lo;
    }
}

// WAVES waves a token. Its first values are asked for before its place is known, which takes four
// reads one after the other: the offsets (two, past 64 sequences), the start and the page. HBM
// bounds it (5061 tokens, 1024 values of k and of v, fp32: 13.9 us, 6.0 TB/s).
template <class T, int WAVES, bool VEC>
__global__ __launch_bounds__(kAppendThreads) void cache_append(
    Cache c, const float* __restrict__ k, int64_t ld_k, const float* __restrict__ v, int64_t ld_v,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ cu, int tokens) {
    constexpr int kThreads = 64 * WAVES, kStep = kThreads * (VEC ? 4 : 1);
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int t = int(blockIdx.x) * (kAppendThreads / kThreads) + wave / WAVES;
    if (t >= tokens) return;
    const int n = int(c.kv_heads * c.dim);
    const int e0 = int(threadIdx.x) % kThreads * (VEC ? 4 : 1);
    const float* const from_k = k + t * ld_k;
    const float* const from_v = v + t * ld_v;
    floatx4u x[kAppendUnroll], y[kAppendUnroll];
    const auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kAppendUnroll; ++u) {
            const int e = base + u * kStep < n ? base + u * kStep : 0;
            if (VEC) {
                x[u] = *reinterpret_cast<const floatx4u*>(from_k + e);
                y[u] = *reinterpret_cast<const floatx4u*>(from_v + e);
            } else {
                x[u][0] = from_k[e];
                y[u][0] = from_v[e];
            }
        }
    };
    load(e0);
    int s = t, first = t;
    if (cu != nullptr) {
        s = sequence_of(cu, int(c.sequences), t);
        first = cu[s];
        if (t < first || t >= cu[s + 1]) return;
    }
    const int64_t row = pool_row(c, s, int64_t(starts[s]) + (t - first));
    if (row < 0) return;
    T* const dk = static_cast<T*>(c.k) + row * n;
    T* const dv = static_cast<T*>(c.v) + row * n;
    for (int base = e0; base < n; base += kAppendUnroll * kStep) {
        if (base != e0) load(base);
#pragma unroll
        for (int u = 0; u < kAppendUnroll; ++u) {
            const int e = base + u * kStep;
            if (e >= n) continue;
            if (VEC) {
                store4(dk + e, x[u]);
                store4(dv + e, y[u]);
            } else {
                narrow(x[u][0], dk[e]);
                narrow(y[u][0], dv[e]);
            }
        }
    }
}

// ----------------------------------------------------------------- attention

// The cache is read once and bounds the time, so the kernel's shape is that of its reads: a
// position's row of `dim` values takes LPP lanes, 16 bytes each, and a wave reads kUnroll x 64 /
// LPP positions of keys and values at a time. A lane holds its values of up to G query heads that
// share the keys. The lanes of a position add up its scores; each position's lanes keep their own
// running maximum, sum and weighted values over the positions they meet, joined at the end: of the
// wave, the block's four waves, and, where the length is split, the blocks of a sequence by a
// second launch. Two sequences of 131072 in fp32, 32 heads over 8 of 128 values: 356 us at best,
// 6.0 TB/s.
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
    int workers;         // blocks of a key head (and piece of its query heads)
    float2* part_stats;  // (heads, workers + sequences): maximum (as 2^x), sum
    float* part_out;     // (heads, workers + sequences, dim)
    int* first;          // (sequences + 1): the sequences' first tiles
};

// The work is cut evenly, whatever the lengths: the positions of all sequences in tiles of kTile,
// one after the other, and a worker's blocks (one for each key head) take its share of them, which
// may be part of a long sequence or several short ones. What a worker adds to a sequence is a
// segment. Segment (worker w, sequence s) has place w + s of a head's parts, no other's: from one
// to the next at least one of them grows.
constexpr int kTile = 128;

// Positions of a sequence, -1 for a length that is none.
__device__ __forceinline__ int length_of(const Paged& a, int64_t s) {
    const int n = a.lengths[s];
    return n < 0 || n > a.longest || n > a.c.width * a.c.page_size || (n > 0 && a.c.pages == 0)
               ? -1
               : n;
}
__device__ __forceinline__ int tiles_of(int n) { return n > 0 ? (n - 1) / kTile + 1 : 0; }

// The first tile of worker w of so many tiles, and the worker of tile t. With fewer tiles than
// workers the last ones have none; every other one has one at least.
__device__ __forceinline__ int first_tile(const Paged& a, int w, int tiles) {
    const int workers = min(a.workers, tiles);
    return w < workers ? int(int64_t(w) * tiles / workers) : tiles;
}
__device__ __forceinline__ int worker_of(const Paged& a, int t, int tiles) {
    return int(((int64_t(t) + 1) * min(a.workers, tiles) - 1) / tiles);
}

struct Segment {
    int64_t s;       // the sequence
    int n;           // its length
    int begin, end;  // positions
    int t, t_end;    // the worker's tiles from here on
    int t0;          // the sequence's first
    bool whole;      // the sequence is this segment
};

__device__ __forceinline__ int wave_scan(int x) {  // inclusive
    const int lane = int(threadIdx.x) & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        x += lane >= d ? y : 0;
    }
    return x;
}

// Sequence, positions and last tile of a segment from its first tile g.t, s and t0 given.
__device__ __forceinline__ void measure(const Paged& a, Segment& g) {
    const int stop = min(g.t_end, g.t0 + tiles_of(g.n));
    g.begin = (g.t - g.t0) * kTile;
    g.end = stop - g.t0 == tiles_of(g.n) ? g.n : (stop - g.t0) * kTile;
    g.whole = g.begin == 0 && g.end == g.n;
}

// The first segment of worker w (t == t_end: none). Every wave finds the same; block 0 leaves the
// sequences' first tiles for the join.
__device__ __forceinline__ Segment first_segment(const Paged& a, int w) {
    const int lane = int(threadIdx.x) & 63;
    const int sequences = int(a.c.sequences);
    int tiles = 0;
    for (int base = 0; base < sequences; base += 64) {
        const int s = base + lane;
        const int mine = s < sequences ? tiles_of(length_of(a, s)) : 0;
        const int upto = wave_scan(mine);
        if (blockIdx.x == 0 && threadIdx.x < 64 && s < sequences)
            a.first[s] = tiles + upto - mine;
        tiles += __shfl(upto, 63);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.first[sequences] = tiles;
    Segment g{};
    g.t = first_tile(a, w, tiles);
    g.t_end = first_tile(a, w + 1, tiles);
    if (g.t == g.t_end) return g;
    int before = 0;
    for (int base = 0; base < sequences; base += 64) {
        const int s = base + lane;
        const int mine = s < sequences ? tiles_of(length_of(a, s)) : 0;
        const int upto = before + wave_scan(mine);
        const uint64_t past = __ballot(upto > g.t);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            g.s = base + at;
            g.t0 = __shfl(upto - mine, at);
            break;
        }
        before = __shfl(upto, 63);
    }
    g.s = __builtin_amdgcn_readfirstlane(int(g.s));
    g.t0 = __builtin_amdgcn_readfirstlane(g.t0);
    g.n = length_of(a, g.s);
    measure(a, g);
    return g;
}

__device__ __forceinline__ void next_segment(const Paged& a, Segment& g) {
    const int stop = g.t0 + tiles_of(g.n);
    g.t = min(g.t_end, stop);
    if (g.t == g.t_end) return;
    do {
        if (++g.s >= a.c.sequences) {  // only where the lengths changed under the launch
            g.t = g.t_end;
            return;
        }
        g.n = length_of(a, g.s);
    } while (tiles_of(g.n) == 0);
    g.t0 = stop;
    measure(a, g);
}

template <int CONTROL>
__device__ __forceinline__ float moved(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CONTROL, 15, 15, true));
}
__device__ __forceinline__ float with_row_pair(float x) {  // lanes 16 apart
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x),
                                                    __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t x0 = r[0], x1 = r[1];  // a bit cast of a vector's element takes the first
    return __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1);
}
__device__ __forceinline__ float with_half(float x) {  // lanes 32 apart
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x),
                                                    __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t x0 = r[0], x1 = r[1];  // a bit cast of a vector's element takes the first
    return __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1);
}

// The sum over the N lanes of a position (the low bits of the lane number), in each of them.
template <int N>
__device__ __forceinline__ float group_sum(float x) {
    if (N > 1) x += moved<0xb1>(x);    // quad_perm 1 0 3 2
    if (N > 2) x += moved<0x4e>(x);    // quad_perm 2 3 0 1
    if (N > 4) x += moved<0x141>(x);   // row_half_mirror
    if (N > 8) x += moved<0x140>(x);   // row_mirror
    if (N > 16) x = with_row_pair(x);
    return x;
}

// The sum over the lanes that hold the same values of the wave's 64 / N positions, in each of them.
template <int N>
__device__ __forceinline__ float across(float x) {
    if (N < 16) x += moved<0x128>(x);  // row_ror 8
    if (N < 8) x += moved<0x124>(x);   // row_ror 4
    if (N < 32) x = with_row_pair(x);
    return with_half(x);
}

// One lane's values of a row as they are stored: 16 bytes, and its own first ones again in lanes
// past the row's end.
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
__global__ __launch_bounds__(kPagedThreads, G * sizeof(T) >= 16 ? 2 : 3) void paged_part(Paged a) {
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
    const int worker = int(x);
    for (Segment seg = first_segment(a, worker); seg.t < seg.t_end; next_segment(a, seg)) {
        const int64_t s = seg.s;
        const int begin = seg.begin, end = seg.end;
        bool bad = false;  // a page outside the pool

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
            float w[G][kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float x[N];
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = ks[u][e];
                if (dim < LPP * N) {  // a lane past the row's end read something else
#pragma unroll
                    for (int e = 0; e < N; ++e) x[e] = e < left ? x[e] : 0.0f;
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float dot = q[g][0] * x[0];
#pragma unroll
                    for (int e = 1; e < N; ++e) dot = __builtin_fmaf(q[g][e], x[e], dot);
                    w[g][u] = group_sum<LPP>(dot);
                }
            }
            const bool tail = p0 + TILE > end;
            if (tail) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                    for (int g = 0; g < G; ++g)
                        w[g][u] = p0 + u * SUBS + sub < end ? w[g][u] : -INFINITY;
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float top = m[g];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) top = fmaxf(top, w[g][u]);
                const float shift = top == -INFINITY ? 0.0f : top;
                const float keep = m[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[g] - shift);
                m[g] = top;
                l[g] *= keep;
#pragma unroll
                for (int e = 0; e < N; ++e) o[g][e] *= keep;
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    // 2^-24 of the weight: sums over the values stay in their range.
                    w[g][u] = __builtin_amdgcn_exp2f(w[g][u] - shift) * 0x1p-24f;
                    l[g] += w[g][u];
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float x[N];
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = vs[u][e];
                if (tail) {  // nor does a position past the length
#pragma unroll
                    for (int e = 0; e < N; ++e) x[e] = p0 + u * SUBS + sub < end ? x[e] : 0.0f;
                }
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int e = 0; e < N; ++e) o[g][e] = __builtin_fmaf(w[g][u], x[e], o[g][e]);
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
            l[g] = across<LPP>(l[g]);
            if (lane == 0) {
                sh_m[wave][g] = top;
                sh_l[wave][g] = l[g];
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float y = o[g][e] * keep;
                y = across<LPP>(y);
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
            const int64_t at = int64_t(h0 + g) * (a.workers + a.c.sequences) + worker + s;
            if (bad) sum = NAN;
            if (threadIdx.x == 0) {
                if (!seg.whole) a.part_stats[at] = float2{top, sum};
                else if (a.lse != nullptr) a.lse[s * a.heads + h0 + g] = lse_of(top, sum);
            }
            for (int d = int(threadIdx.x); d < dim; d += kPagedThreads) {
                float y = 0.0f;
#pragma unroll
                for (int w = 0; w < kPagedWaves; ++w) y += sh_o[w][g][d] * keep[w];
                if (!seg.whole) a.part_out[at * dim + d] = y;
                else a.out[s * a.ld_out + int64_t(h0 + g) * dim + d] = y / sum;
            }
        }
        __syncthreads();
    }
}

// One head's share of a block by the formula, for those whose sums by parts are not finite: a part
// of an infinity, or an infinity times the parts of a finite value, is NaN where the product is an
// infinity or, its weight 0, nothing at all. One wave, a lane for each of 64 positions at a time,
// of rows of 16-byte units; a score of NaN or +inf settles the head as NaN (64 sequences of 1024,
// 32 heads over 8 of 128 values, us: finite 56, the first key NaN 59, the first value infinite 560;
// value by value and to the end 1870 either way).
__device__ void part_by_formula(const Paged& a, int64_t s, int h, int kv, int begin, int end,
                                float& top, float& sum, float (&o)[2]) {
    using attention::uintx4;
    int lane = int(threadIdx.x) & 63;
    asm volatile("" : "+v"(lane));  // else what follows from it is held all through the tiles
    const int dim = int(a.c.dim);
    const int64_t pitch = a.c.kv_heads * dim;
    const float* q = a.q + s * a.ld_q + int64_t(h) * dim;
    const Bf16* k = static_cast<const Bf16*>(a.c.k) + int64_t(kv) * dim;
    const Bf16* v = static_cast<const Bf16*>(a.c.v) + int64_t(kv) * dim;
    const float c2 = a.scale * 1.44269504088896340736f;
    // The pool row of position p0 + lane, the last again past the end.
    const auto row_of = [&](int p0) { return int(pool_row(a.c, s, min(p0 + lane, end - 1))); };
    const auto score = [&](int row) {
        const Bf16* at = k + int64_t(row) * pitch;
        float dot = 0.0f;
        for (int e = 0; e < dim; e += 8) {
            const uintx4 x = *reinterpret_cast<const uintx4*>(at + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t pair = x[j];
                dot = __builtin_fmaf(q[e + 2 * j] * c2, __builtin_bit_cast(float, pair << 16), dot);
                dot = __builtin_fmaf(q[e + 2 * j + 1] * c2,
                                     __builtin_bit_cast(float, pair & 0xffff0000u), dot);
            }
        }
        return dot;
    };
    top = -INFINITY;
    for (int p0 = begin; p0 < end; p0 += 64) {
        const float x = score(row_of(p0));
        if (__any(!(x < INFINITY))) {
            top = 0.0f;
            sum = o[0] = o[1] = NAN;
            return;
        }
        top = fmaxf(top, x);
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    const float shift = top == -INFINITY ? 0.0f : top;  // scores of -inf alone weigh nothing
    sum = o[0] = o[1] = 0.0f;
    const int d0 = lane < dim ? lane : 0, d1 = lane + 64 < dim ? lane + 64 : 0;
    for (int p0 = begin; p0 < end; p0 += 64) {
        const int row = row_of(p0), count = min(64, end - p0);
        const float weight = lane < count ? exp2f(score(row) - shift) * 0x1p-24f : 0.0f;
        sum += weight;
#pragma unroll 8
        for (int u = 0; u < count; ++u) {
            const Bf16* at = v + int64_t(__shfl(row, u)) * pitch;
            const float w = __shfl(weight, u);
            o[0] = __builtin_fmaf(w, widen(at[d0]), o[0]);
            o[1] = __builtin_fmaf(w, widen(at[d1]), o[1]);
        }
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
}

// A cache in bf16, up to 16 query heads of a key head at a time, on v_mfma_f32_16x16x32_bf16: the
// cached values are operands as they are, q and the weights in three parts, so a score and a
// weighted value take three products each, for any number of heads at one cost; by vector
// instructions four heads ran at 4.3 TB/s of 5.4 and eight at 2.7. Lane l holds A(l % 16, 8 (l /
// 16) + 0..7), B(8 (l / 16) + 0..7, l % 16) and D(4 (l / 16) + r, l % 16).
//   scores:  A = 16 positions by 32 values of K, as 16-byte reads leave them; B = q; D's columns
//            are heads
//   weights: the D's of positions 0..15 and 16..31 are the B of 32 positions, in the order
//            4 h + 0..3, 16 + 4 h + 0..3 for the lanes h = l / 16
//   values:  A = 16 values by those 32 positions of V: rows in LDS, read transposed
// A wave takes 32 positions at a time; the next ones' reads are out while it forms weights and
// sums. 64 sequences of 4096, 32 heads over 8 of 128 values: 213 us, 5.0 TB/s; of 64 to 4096, 66
// us, 4.0: a block passes parts of several there, and its loads run dry at each change.
constexpr int kTilePositions = 32;

template <int DP>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_part_bf16(Paged a) {
    using attention::bf16x8;
    using attention::floatx4u;
    using attention::uintx4;
    typedef float floatx4 __attribute__((ext_vector_type(4)));
    typedef short shortx4 __attribute__((ext_vector_type(4)));
    constexpr int KS = DP / 32, NV = DP / 16, LANES = DP / 8;  // lanes of a row's reads
    constexpr int kRows = 64 / LANES, kReads = (kTilePositions + kRows - 1) / kRows;
    // Rows 32 bytes apart in banks: a transposed read's sixteen rows take all banks twice.
    constexpr int kPitch = 2 * DP + 32;
    constexpr int kWaveLds = kTilePositions * kPitch;
    constexpr int kLds = kWaveLds > 16 * DP * 4 ? kWaveLds : 16 * DP * 4;
    __shared__ __attribute__((aligned(16))) char lds[kPagedWaves][kLds];
    __shared__ float sh_m[kPagedWaves][16], sh_l[kPagedWaves][16];
    const int lane = int(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int kv_heads = int(a.c.kv_heads), dim = int(a.c.dim);
    const int group = a.heads / kv_heads, pieces = (group + 15) / 16;
    uint32_t x = blockIdx.x;
    const int kv = int(x % uint32_t(kv_heads));
    x /= uint32_t(kv_heads);
    const int h0 = kv * group + int(x % uint32_t(pieces)) * 16;
    const int count = min(16, (kv + 1) * group - h0);  // the block's heads
    x /= uint32_t(pieces);
    const int worker = int(x);
    for (Segment seg = first_segment(a, worker); seg.t < seg.t_end; next_segment(a, seg)) {
        const int64_t s = seg.s;
        const int begin = seg.begin, end = seg.end;
        bool bad = false;  // a page outside the pool

        const int col = lane & 15, quarter = lane / 16;
        const float c2 = a.scale * 1.44269504088896340736f;
        bf16x8 q[KS][3];
        {
            const float* row = a.q + s * a.ld_q + int64_t(h0 + (col < count ? col : 0)) * dim;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d0 = 32 * ks + 8 * quarter;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    y[e] = d0 < dim && col < count ? row[d0 < dim ? d0 + e : 0] * c2 : 0.0f;
                attention::split8(y, q[ks]);
            }
        }
        floatx4 o[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;

        const Bf16* const k = static_cast<const Bf16*>(a.c.k) + int64_t(kv) * dim;
        const Bf16* const v = static_cast<const Bf16*>(a.c.v) + int64_t(kv) * dim;
        const int64_t pitch = int64_t(kv_heads) * dim;
        bf16x8 kx[2][KS];
        uintx4 vx[kReads];
        const int v_lane = lane / LANES, v_d0 = lane % LANES * 8;
        const auto load = [&](int p0) {
            const int p = p0 + (lane & 31);
            int64_t row = 0;
            if (p < end) {
                row = pool_row(a.c, s, p);
                if (row < 0) {
                    bad = true;
                    row = 0;
                }
            }
            const int r = int(row);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const Bf16* at = k + int64_t(__shfl(r, 16 * t + col)) * pitch;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int d0 = 32 * ks + 8 * quarter;
                    kx[t][ks] = *reinterpret_cast<const bf16x8*>(at + (d0 < dim ? d0 : 0));
                }
            }
#pragma unroll
            for (int i = 0; i < kReads; ++i) {
                const int j = i * kRows + v_lane;
                const Bf16* at = v + int64_t(__shfl(r, j < kTilePositions ? j : 0)) * pitch;
                vx[i] = *reinterpret_cast<const uintx4*>(at + (v_d0 < dim ? v_d0 : 0));
            }
        };
        char* const mine = lds[wave];
        const int first = begin + wave * kTilePositions;
        if (first < end) load(first);
        for (int p0 = first; p0 < end; p0 += kPagedWaves * kTilePositions) {
            const bool tail = p0 + kTilePositions > end;
#pragma unroll
            for (int i = 0; i < kReads; ++i) {
                const int j = i * kRows + v_lane;
                uintx4 y = vx[i];
                if (tail && p0 + j >= end) y = uintx4{0, 0, 0, 0};  // nothing, whatever is there
                if (v_lane < kRows && j < kTilePositions)
                    *reinterpret_cast<uintx4*>(mine + j * kPitch + 2 * v_d0) = y;
            }
            floatx4 sc[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int part = 2; part >= 0; --part)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        // Past the row's end q is 0 and K something else, which has to be finite.
                        bf16x8 f = kx[t][ks];
                        if (DP != dim && 32 * ks + 8 * quarter >= dim)
                            f = __builtin_bit_cast(bf16x8, uintx4{0, 0, 0, 0});
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, q[ks][part], sc[t], 0,
                                                                        0, 0);
                    }
            }
            if (p0 + kPagedWaves * kTilePositions < end) load(p0 + kPagedWaves * kTilePositions);
            if (tail) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (p0 + 16 * t + 4 * quarter + r >= end) sc[t][r] = -INFINITY;
            }
            float top = m;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, sc[t][r]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float shift = top == -INFINITY ? 0.0f : top;
            const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - shift);
            m = top;
            float w[8], part_sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] = __builtin_amdgcn_exp2f(sc[j / 4][j % 4] - shift) * 0x1p-24f;
                part_sum += w[j];
            }
            l = __builtin_fmaf(l, keep, part_sum);
            bf16x8 p[3];
            attention::split8(w, p);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                typedef __attribute__((address_space(3))) shortx4* Rows;
                // Lane: row 4 quarter + col / 4 (and 16 rows on), values 16 i + 4 (col % 4) + 0..3.
                const char* at = mine + (4 * quarter + col / 4) * kPitch + 32 * i + 8 * (col % 4);
                struct {
                    shortx4 x, y;
                } f = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((Rows)at),
                       __builtin_amdgcn_ds_read_tr16_b64_v4i16((Rows)(at + 16 * kPitch))};
                const bf16x8 vt = __builtin_bit_cast(bf16x8, f);
                floatx4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int part = 2; part >= 0; --part)
                    y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt, p[part], y, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[i][r] = __builtin_fmaf(o[i][r], keep, y[r]);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        bad = __syncthreads_or(bad);

        // The waves of the block: sums of head `col`, value 16 i + 4 quarter + r.
        l = with_half(with_row_pair(l));
        if (quarter == 0) {
            sh_m[wave][col] = m;
            sh_l[wave][col] = l;
        }
        float* const sums = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            *reinterpret_cast<floatx4*>(sums + col * DP + 16 * i + 4 * quarter) = o[i];
        __syncthreads();
        for (int g = wave; g < count; g += kPagedWaves) {
            float top = sh_m[0][g], sum = 0.0f, keep[kPagedWaves], y[2] = {0.0f, 0.0f};
#pragma unroll
            for (int u = 1; u < kPagedWaves; ++u) top = fmaxf(top, sh_m[u][g]);
            bool fine = true;
#pragma unroll
            for (int u = 0; u < kPagedWaves; ++u) {
                keep[u] = sh_m[u][g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sh_m[u][g] - top);
                sum += sh_l[u][g] * keep[u];
                fine = fine && fabsf(sh_l[u][g]) < INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = lane + 64 * e;
                if (d >= dim) continue;
#pragma unroll
                for (int u = 0; u < kPagedWaves; ++u)
                    y[e] += reinterpret_cast<const float*>(lds[u])[g * DP + d] * keep[u];
                fine = fine && fabsf(y[e]) < INFINITY;
            }
            if (!bad && !(__all(fine) && sum > 0.0f))
                part_by_formula(a, s, h0 + g, kv, begin, end, top, sum, y);
            const int64_t at = int64_t(h0 + g) * (a.workers + a.c.sequences) + worker + s;
            if (bad) sum = NAN;
            if (lane == 0) {
                if (!seg.whole) a.part_stats[at] = float2{top, sum};
                else if (a.lse != nullptr) a.lse[s * a.heads + h0 + g] = lse_of(top, sum);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = lane + 64 * e;
                if (d >= dim) continue;
                if (!seg.whole) a.part_out[at * dim + d] = y[e];
                else a.out[s * a.ld_out + int64_t(h0 + g) * dim + d] = y[e] / sum;
            }
        }
        __syncthreads();
    }
}

// The segments of a sequence and a head, where there are several, and the rows of sequences that
// have no segment. Thread d % 128 has a value, two threads for alternate segments. Latency: 3 to 6
// us.
__global__ __launch_bounds__(256) void paged_join(Paged a) {
    __shared__ float sh[2][kMaxDim], sh_l[2];
    const int64_t at = blockIdx.x, s = at / a.heads;
    const int h = int(at % a.heads), dim = int(a.c.dim);
    const int d = int(threadIdx.x) % kMaxDim, half = int(threadIdx.x) / kMaxDim;
    const int n = length_of(a, s);
    if (n <= 0) {
        if (half == 0 && d < dim)
            a.out[s * a.ld_out + int64_t(h) * dim + d] = n < 0 ? NAN : 0.0f;
        if (threadIdx.x == 0 && a.lse != nullptr) a.lse[at] = n < 0 ? NAN : -INFINITY;
        return;
    }
    const int tiles = a.first[a.c.sequences];
    const int w0 = worker_of(a, a.first[s], tiles);
    const int parts = worker_of(a, a.first[s + 1] - 1, tiles) - w0 + 1;
    if (parts == 1) return;  // the sequence was one segment
    const int64_t from = int64_t(h) * (a.workers + a.c.sequences) + w0 + s;
    const float2* stats = a.part_stats + from;
    float top = -INFINITY;
    for (int i = int(threadIdx.x) & 63; i < parts; i += 64) top = fmaxf(top, stats[i].x);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    float sum = 0.0f, y = 0.0f;
    const float* values = a.part_out + from * dim + (d < dim ? d : 0);
#pragma unroll 8
    for (int i = half; i < parts; i += 2) {
        const float2 z = stats[i];
        const float keep = z.x == -INFINITY ? (z.y != z.y ? NAN : 0.0f)
                                            : __builtin_amdgcn_exp2f(z.x - top);
        sum += z.y * keep;
        y = __builtin_fmaf(values[int64_t(i) * dim], keep, y);
    }
    sh[half][d] = y;
    if (d == 0) sh_l[half] = sum;
    __syncthreads();
    if (half != 0) return;
    sum = sh_l[0] + sh_l[1];
    y += sh[1][d];
    if (d < dim) a.out[s * a.ld_out + int64_t(h) * dim + d] = y / sum;
    if (d == 0 && a.lse != nullptr) a.lse[at] = lse_of(top, sum);
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

// Positions count on past a length by less than that again in 32 bits; pages may repeat in a table,
// so the pool's extent does not bound a length.
constexpr int64_t kMaxLength = int64_t(1) << 30;

int check_heads(const char* name, const Cache& c, int64_t heads, int64_t longest) {
    if (c.dim > kMaxDim || heads < 1 || heads % c.kv_heads != 0 || longest < 0)
        return fail(EHIP_EINVAL, "%s: %lld heads over %lld of %lld values, length %lld", name,
                    (long long)heads, (long long)c.kv_heads, (long long)c.dim, (long long)longest);
    if (heads > kMaxBlocks || c.sequences * heads > kMaxBlocks || longest > kMaxLength ||
        c.sequences * ceil_div(longest, kTile) > INT32_MAX)
        return fail(EHIP_EINVAL, "%s: %lld sequences of %lld heads of length %lld are too many",
                    name, (long long)c.sequences, (long long)heads, (long long)longest);
    return EHIP_OK;
}

// Workers for 512 blocks in all, two a CU (64 sequences of 64 to 4096 positions in bf16: 75 us
// against 85 with 1024 blocks and 101 with 2048; two of 131072 in fp32: 383, 388, 389), and no more
// than there can be tiles.
int workers_of(const Cache& c, int64_t heads, int64_t longest, int type) {
    const int64_t group = heads / c.kv_heads;
    const int64_t units = c.kv_heads * ceil_div(group, type == EHIP_CACHE_F32 ? kMaxGroup : 16);
    constexpr int64_t resident = 512;
    const int64_t most = std::max<int64_t>(1, c.sequences * ceil_div(longest, kTile));
    return int(std::min(most, std::max<int64_t>(1, resident / units)));
}

// Parts of a head, and the bytes of all heads' and of the sequences' first tiles.
size_t part_bytes(const Cache& c, int64_t heads, int workers) {
    return size_t(heads) * size_t(workers + c.sequences) *
               (sizeof(float2) + size_t(c.dim) * sizeof(float)) +
           size_t(c.sequences + 1) * sizeof(int);
}

struct Append {
    Cache c;
    const float* k;
    int64_t ld_k;
    const float* v;
    int64_t ld_v;
    const int32_t *starts, *cu;
    int tokens;
};

template <class T, int WAVES, bool VEC>
int launch_append(const Append& x, hipStream_t s) {
    EHIP_LAUNCH("cache_append", (cache_append<T, WAVES, VEC>),
                dim3(unsigned(ceil_div(x.tokens, kAppendThreads / (64 * WAVES)))),
                dim3(kAppendThreads), 0, s, x.c, x.k, x.ld_k, x.v, x.ld_v, x.starts, x.cu,
                x.tokens);
    return EHIP_OK;
}

template <class T>
int append(const Append& x, hipStream_t s) {
    const int64_t n = x.c.kv_heads * x.c.dim;
    // A wave a token (us, fp32, 16.8 M values in rows of 128: 56 against 153 with four; of 1024 46
    // : 45, in bf16 32 : 34), four for wider rows (of 4096 52 : 45).
    const bool wide = n > 1024;
    if (n % 4 == 0 && aligned16(x.c.k) && aligned16(x.c.v))
        return wide ? launch_append<T, 4, true>(x, s) : launch_append<T, 1, true>(x, s);
    return wide ? launch_append<T, 4, false>(x, s) : launch_append<T, 1, false>(x, s);
}

template <class T, int LPP, int G, bool VEC>
int launch_part(const Paged& a, hipStream_t s) {
    const int64_t group = a.heads / a.c.kv_heads;
    const int64_t blocks = a.workers * ceil_div(group, G) * a.c.kv_heads;
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
int launch_parts_f32(const Paged& a, bool aligned, hipStream_t s) {
    return aligned && a.c.dim % 4 == 0 ? launch_lanes<float, true>(a, s)
                                       : launch_lanes<float, false>(a, s);
}

template <int DP>
int launch_part_bf16(const Paged& a, hipStream_t s) {
    const int64_t group = a.heads / a.c.kv_heads;
    const int64_t blocks = a.workers * ceil_div(group, 16) * a.c.kv_heads;
    EHIP_LAUNCH("attention_paged", paged_part_bf16<DP>, dim3(unsigned(blocks)),
                dim3(kPagedThreads), 0, s, a);
    return EHIP_OK;
}

int launch_parts_bf16(const Paged& a, bool aligned, hipStream_t s) {
    if (!aligned || a.c.dim % 8 != 0) return launch_lanes<Bf16, false>(a, s);
    if (a.c.dim <= 32) return launch_part_bf16<32>(a, s);
    if (a.c.dim <= 64) return launch_part_bf16<64>(a, s);
    return launch_part_bf16<128>(a, s);
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
    if (n > kMaxLength) return fail(EHIP_EINVAL, "cache_append: rows of %lld values", (long long)n);
    if (tokens < 0 || tokens > kMaxBlocks || ld_k < n || ld_v < n ||
        (cu == nullptr && tokens != c.sequences))
        return fail(EHIP_EINVAL, "cache_append: %lld tokens for %lld sequences, rows %lld and %lld "
                                 "apart",
                    (long long)tokens, (long long)c.sequences, (long long)ld_k, (long long)ld_v);
    if (tokens == 0 || c.sequences == 0) return EHIP_OK;
    if (k == nullptr || v == nullptr || starts == nullptr)
        return fail(EHIP_EINVAL, "cache_append: null tensor");
    hipStream_t s = as_stream(stream);
    const Append x{c, k, ld_k, v, ld_v, starts, cu, int(tokens)};
    return cache->type == EHIP_CACHE_F32 ? append<float>(x, s) : append<Bf16>(x, s);
}

int64_t ehip_attention_paged_workspace(const ehip_cache_t* cache, int64_t heads,
                                       int64_t longest) {
    Cache c;
    if (check("attention_paged", cache, c) || check_heads("attention_paged", c, heads, longest))
        return -1;
    return c.sequences == 0
               ? 0
               : int64_t(part_bytes(c, heads, workers_of(c, heads, longest, cache->type)));
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
    const int workers = workers_of(c, heads, longest, cache->type);
    const size_t need = part_bytes(c, heads, workers);
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
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
    a.workers = workers;
    const int64_t parts = heads * (workers + c.sequences);
    a.part_stats = static_cast<float2*>(workspace);
    a.part_out = reinterpret_cast<float*>(a.part_stats + parts);
    a.first = reinterpret_cast<int*>(a.part_out + parts * c.dim);
    hipStream_t s = as_stream(stream);
    const bool aligned = aligned16(c.k) && aligned16(c.v);
    const int rc = cache->type == EHIP_CACHE_F32 ? launch_parts_f32(a, aligned, s)
                                                 : launch_parts_bf16(a, aligned, s);
    if (rc != EHIP_OK) return rc;
    EHIP_LAUNCH("attention_paged_join", paged_join, dim3(unsigned(c.sequences * heads)), dim3(256),
                0, s, a);
    return EHIP_OK;
}

}  // extern "C"
