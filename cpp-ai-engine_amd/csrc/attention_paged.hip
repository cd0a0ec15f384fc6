// attention_paged.hip -- a cache of keys and values in pages: the write of new tokens into it, and
// the attention of one new token per sequence over it,
//
//   s_p = scale (q . k_p), lse = log sum_p exp(s_p), out = sum_p exp(s_p - lse) v_p
//
// over the positions p below the sequence's length, each on the page that the table names.

#include "attention_paged.hpp"

namespace ehip {

using namespace paged;

namespace {

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

// The nearest whole number of scales, ties to even. The quotient in fp32 may be one off next to a
// half; what is left, exact in 64 bits, says so.
__device__ __forceinline__ int quantised(float x, float scale, float lift, float inverse) {
    float n = rintf(fminf(fmaxf(x * lift * inverse, -127.0f), 127.0f));
    const double s = double(scale), left = 2.0 * __builtin_fma(-double(n), s, double(x));
    const bool odd = int(n) & 1;
    if (left > s || (left == s && odd)) n += 1.0f;
    if (left < -s || (left == -s && odd)) n -= 1.0f;
    return int(fminf(fmaxf(n, -127.0f), 127.0f));
}

template <int N>
__device__ __forceinline__ float largest_of(float x) {
#pragma unroll
    for (int w = 1; w < N; w *= 2) x = fmaxf(x, __shfl_xor(x, w));
    return x;
}

// The scale of a head's values (those of N lanes) and a lane's four as whole numbers. A NaN or an
// infinity makes the scale NaN and so the whole head; where the scale rounds to 0 all are 0.
template <int N>
__device__ __forceinline__ float quantise(const float (&x)[4], uint32_t& codes) {
    float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) fine = fine && fabsf(x[e]) < INFINITY;
    top = largest_of<N>(fine ? top : INFINITY);
    codes = 0;
    if (!(top < INFINITY)) return NAN;
    float scale = top / 127.0f;
    if (scale == 0.0f) return 0.0f;
    if (scale * 127.0f == INFINITY)  // the next lower one: what is read back is finite
        scale = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, scale) - 1);
    const float lift = scale < 0x1p-100f ? 0x1p64f : 1.0f;  // the reciprocal is finite
    const float inverse = 1.0f / (scale * lift);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        codes |= uint32_t(quantised(x[e], scale, lift, inverse) & 0xff) << (8 * e);
    return scale;
}

// One of the four values that a lane has of a head, and where it has fewer.
__device__ __forceinline__ void load_head(const float* row, int d0, int dim, float (&x)[4]) {
    if (d0 + 4 <= dim) {
        const floatx4u y = *reinterpret_cast<const floatx4u*>(row + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = y[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = d0 + e < dim ? row[d0 + e] : 0.0f;
    }
}
__device__ __forceinline__ void store_codes(Int8* row, int d0, int dim, uint32_t codes) {
    if (d0 + 4 <= dim) {
        __builtin_memcpy(row + d0, &codes, 4);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (d0 + e < dim) row[d0 + e].n = int8_t(codes >> (8 * e));
    }
}

// In 8 bits: a wave a token, N lanes a key head, four values of k and of v each (10060 tokens, 8
// heads of 128: 39 us for 104 MB, 2.7 TB/s; vector instructions take 70 % of it).
template <int N>
__global__ __launch_bounds__(kAppendThreads) void cache_append_i8(
    Cache c, const float* __restrict__ k, int64_t ld_k, const float* __restrict__ v, int64_t ld_v,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ cu, int tokens) {
    constexpr int kHeads = 64 / N;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int t = int(blockIdx.x) * (kAppendThreads / 64) + wave;
    if (t >= tokens) return;
    const int lane = int(threadIdx.x) & 63, d0 = lane % N * 4, dim = int(c.dim);
    const int heads = int(c.kv_heads);
    float x[4], y[4];
    const auto load = [&](int h) {
        load_head(k + t * ld_k + int64_t(h < heads ? h : 0) * dim, d0, dim, x);
        load_head(v + t * ld_v + int64_t(h < heads ? h : 0) * dim, d0, dim, y);
    };
    load(lane / N);
    int s = t, first = t;
    if (cu != nullptr) {
        s = sequence_of(cu, int(c.sequences), t);
        first = cu[s];
        if (t < first || t >= cu[s + 1]) return;
    }
    uint32_t off;
    const int64_t row = pool_row(c, s, int64_t(starts[s]) + (t - first), off);
    if (row < 0) return;
    for (int h0 = 0; h0 < heads; h0 += kHeads) {
        const int h = h0 + lane / N;
        if (h0 > 0) load(h);
        uint32_t kx, vx;
        const float ks = quantise<N>(x, kx), vs = quantise<N>(y, vx);
        if (h >= heads) continue;
        const int64_t at = row * heads + h;
        store_codes(static_cast<Int8*>(c.k) + at * dim, d0, dim, kx);
        store_codes(static_cast<Int8*>(c.v) + at * dim, d0, dim, vx);
        if (d0 == 0) {
            const int64_t place = scale_of(c, row, off, h);
            c.k_scales[place] = ks;
            c.v_scales[place] = vs;
        }
    }
}

// ---------------------------------------------------------------------- read

__device__ __forceinline__ void load4(const float* from, float (&x)[4]) {
    const floatx4u y = *reinterpret_cast<const floatx4u*>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = y[e];
}
__device__ __forceinline__ void load4(const Bf16* from, float (&x)[4]) {
    Bf16 y[4];
    __builtin_memcpy(y, __builtin_assume_aligned(from, 8), 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = widen(y[e]);
}
__device__ __forceinline__ void load4(const Int8* from, float (&x)[4]) {
    Int8 y[4];
    __builtin_memcpy(y, __builtin_assume_aligned(from, 4), 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = widen(y[e]);
}

// Positions of the pools as rows: a wave a token. VEC: dim and the pools allow four values at a
// time (58430 positions, 8 heads of 128 in 8 bits: 122 us, 5.0 TB/s).
template <class T, bool VEC>
__global__ __launch_bounds__(kAppendThreads) void cache_read(
    Cache c, const int32_t* __restrict__ starts, const int32_t* __restrict__ cu, int tokens,
    float* __restrict__ k, int64_t ld_k, float* __restrict__ v, int64_t ld_v) {
    constexpr bool kScaled = sizeof(T) == 1;
    constexpr int N = VEC ? 4 : 1;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int t = int(blockIdx.x) * (kAppendThreads / 64) + wave;
    if (t >= tokens) return;
    int s = t, first = t;
    if (cu != nullptr) {
        s = sequence_of(cu, int(c.sequences), t);
        first = cu[s];
        if (t < first || t >= cu[s + 1]) return;
    }
    uint32_t off = 0;
    const int64_t row = pool_row(c, s, int64_t(starts[s]) + (t - first), off);
    const int n = int(c.kv_heads * c.dim);
    const T* const from_k = static_cast<const T*>(c.k) + row * n;
    const T* const from_v = static_cast<const T*>(c.v) + row * n;
#pragma unroll 2
    for (int e = (int(threadIdx.x) & 63) * N; e < n; e += 64 * N) {
        float x[4], y[4];
        if (row < 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = y[j] = NAN;
        } else {
            if constexpr (VEC) {
                load4(from_k + e, x);
                load4(from_v + e, y);
            } else {
                x[0] = widen(from_k[e]);
                y[0] = widen(from_v[e]);
            }
            if constexpr (kScaled) {
                const int64_t place = scale_of(c, row, off, int(uint32_t(e) / uint32_t(c.dim)));
                const float ks = c.k_scales[place], vs = c.v_scales[place];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    x[j] *= ks;
                    y[j] *= vs;
                }
            }
        }
        if (VEC) {
            *reinterpret_cast<floatx4u*>(k + t * ld_k + e) = floatx4u{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<floatx4u*>(v + t * ld_v + e) = floatx4u{y[0], y[1], y[2], y[3]};
        } else {
            k[t * ld_k + e] = x[0];
            v[t * ld_v + e] = y[0];
        }
    }
}

// The segments of a sequence and a head, where there are several, and the rows of sequences that
// have no segment.
template <int WAVES>
__global__ __launch_bounds__(join_threads(WAVES)) void paged_join(Paged a) {
    __shared__ float sh[WAVES][kMaxDim + 1];
    const int64_t at = int64_t(blockIdx.x) * (join_threads(WAVES) / (64 * WAVES)) +
                       int(threadIdx.x) / (64 * WAVES);
    if (at >= a.c.sequences * a.heads) return;
    const int64_t s = at / a.heads;
    const Own own = own_of(a, s);
    const int h = int(at % a.heads), n = length_from(a, own.length);
    if (n <= 0) {
        empty_row<WAVES>(a, s, h, n);
        return;
    }
    const Parts p[2] = {own_parts(a, own, s, h), Parts{nullptr, nullptr, 0, 1}};
    if (p[0].count == 1) return;  // the sequence was one segment
    join_parts<WAVES>(a, s, h, p, sh);
}

}  // namespace

// Workers for 512 blocks in all, two a CU (two sequences of 131072 in fp32: 383 us against 388 with
// 1024 blocks and 389 with 2048), or as many of four waves, and no more than there can be tiles. Few
// sequences and key heads leave a wave few tiles, and a row as many parts as there are waves: a tile
// takes some 0.9 us, a part of the join some 0.015, and their sum is least with 8 sqrt(tiles
// sequences) waves, of as many tiles each (bf16, 8 heads of 128 over one, one sequence of 65536: 2048
// waves 50 us, 1024 33, 512 27.6, 256 28.4; so 342, 27.4; four of up to 16384: 2048 24.9, 512 22.4,
// 256 23.4; one of 4096, 16 heads of 64: 128 13.3, 90 14.0, 64 12.5).
Cut paged::cut_of(const Cache& c, int64_t heads, int64_t longest, bool waves) {
    const int64_t group = heads / c.kv_heads;
    const int64_t units =
        c.kv_heads * ceil_div(group, waves ? 16 : kMaxGroup);
    const int64_t resident = waves ? 2048 : 512;
    const int tile = tile_of(waves, c.sequences, longest);
    const int64_t most = std::max<int64_t>(1, c.sequences * ceil_div(longest, tile));
    int64_t workers = std::min(most, std::max<int64_t>(1, resident / units));
    if (waves) {
        const double even = 8.0 * std::sqrt(double(most) * double(c.sequences));
        workers = std::min(workers, ceil_div(most, int64_t(std::ceil(double(most) / even))));
    }
    return Cut{waves, tile, int(workers)};
}

namespace {

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

template <int N>
int launch_append_i8(const Append& x, hipStream_t s) {
    EHIP_LAUNCH("cache_append", cache_append_i8<N>,
                dim3(unsigned(ceil_div(x.tokens, kAppendThreads / 64))), dim3(kAppendThreads), 0, s,
                x.c, x.k, x.ld_k, x.v, x.ld_v, x.starts, x.cu, x.tokens);
    return EHIP_OK;
}

int append_i8(const Append& x, hipStream_t s) {
    if (x.c.dim <= 16) return launch_append_i8<4>(x, s);
    if (x.c.dim <= 32) return launch_append_i8<8>(x, s);
    if (x.c.dim <= 64) return launch_append_i8<16>(x, s);
    return launch_append_i8<32>(x, s);
}

struct Read {
    Cache c;
    const int32_t *starts, *cu;
    int tokens;
    float* k;
    int64_t ld_k;
    float* v;
    int64_t ld_v;
};

template <class T>
int read(const Read& x, hipStream_t s) {
    const dim3 grid{unsigned(ceil_div(x.tokens, kAppendThreads / 64))}, block{kAppendThreads};
    if (x.c.dim % 4 == 0 && aligned16(x.c.k) && aligned16(x.c.v))
        EHIP_LAUNCH("cache_read", (cache_read<T, true>), grid, block, 0, s, x.c, x.starts, x.cu,
                    x.tokens, x.k, x.ld_k, x.v, x.ld_v);
    else
        EHIP_LAUNCH("cache_read", (cache_read<T, false>), grid, block, 0, s, x.c, x.starts, x.cu,
                    x.tokens, x.k, x.ld_k, x.v, x.ld_v);
    return EHIP_OK;
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
    if constexpr (sizeof(T) == 4)  // bf16 comes with up to four
        if (group > 4) return launch_part<T, LPP, kMaxGroup, VEC>(a, s);
    return launch_part<T, LPP, 4, VEC>(a, s);
}

template <class T, bool VEC>
int launch_lanes(const Paged& a, hipStream_t s) {
    constexpr int N = 16 / int(sizeof(T));
    if (a.c.dim <= 32) return launch_group<T, 32 / N, VEC>(a, s);
    if (a.c.dim <= 64) return launch_group<T, 64 / N, VEC>(a, s);
    return launch_group<T, 128 / N, VEC>(a, s);
}

template <class T, int DP, bool WIDE>
int launch_part_mfma(const Paged& a, hipStream_t s) {
    const int64_t group = a.heads / a.c.kv_heads;
    const int64_t blocks = ceil_div(a.workers * ceil_div(group, 16) * a.c.kv_heads, kPagedWaves);
    EHIP_LAUNCH("attention_paged", (paged_part_mfma<T, DP, WIDE>), dim3(unsigned(blocks)),
                dim3(kPagedThreads), 0, s, a);
    return EHIP_OK;
}

template <class T, bool WIDE>
int launch_mfma(const Paged& a, hipStream_t s) {
    if (a.c.dim <= 32) return launch_part_mfma<T, 32, WIDE>(a, s);
    if (a.c.dim <= 64) return launch_part_mfma<T, 64, WIDE>(a, s);
    return launch_part_mfma<T, 128, WIDE>(a, s);
}

// Whether the positions go by waves and the matrix instructions. Three kinds of bf16 heads do not, whose
// work is too little for what those kernels take before their first tile and for a join (us, vector :
// matrix). Few whole rows, a head a key head: their products have one column of 16 (16 sequences of up
// to 100, 8 heads of 64, 8.4 : 11.4; one of 4096, 16 heads 10.9 : 12.6; 64 of up to 64 12.5 : 11.5; two
// heads over one, one sequence of 8192, 12.6 : 13.0, of 8 values 12.5 : 11.0). Few rows that are not
// whole units: the last values are put in place there, and registers spilled (one sequence of 64, 16
// heads of 77 10.3 : 19.7, of 4096 22.9 : 29.7; of 2048, 32 heads over 8 of 77 21.5 : 22.9, of 100 23.7
// : 21.6; of 8192, 8 over one of 77 31.5 : 26.9; 4 of up to 4096, 32 over 8 of 77 50.8 : 38.2). And
// single ones of below eight values, which both read one by one (256 of up to 300, 16 of 7, 75 : 95;
// of 33 101 : 67).
bool waves_of(const Cache& c, int64_t heads, int64_t longest, int type) {
    if (type != EHIP_CACHE_BF16) return by_waves(type);
    const int64_t group = heads / c.kv_heads;
    const bool few = c.sequences * heads * longest <= int64_t(1) << 16;
    if (whole_rows(c, 8)) return !(few && group == 1 && c.sequences <= 16);
    return !(few && group <= 4) && !(group == 1 && c.dim < 8);
}

template <int WAVES>
int launch_join(const Paged& a, int64_t rows, hipStream_t s) {
    EHIP_LAUNCH("attention_paged_join", paged_join<WAVES>,
                dim3(unsigned(ceil_div(rows, join_threads(WAVES) / (64 * WAVES)))),
                dim3(join_threads(WAVES)), 0, s, a);
    return EHIP_OK;
}

}  // namespace

int paged::launch_parts(const Paged& a, int type, bool waves, hipStream_t s) {
    if (type == EHIP_CACHE_F32)
        return whole_rows(a.c, 4) ? launch_lanes<float, true>(a, s)
                                  : launch_lanes<float, false>(a, s);
    if (!waves && !whole_rows(a.c, 8)) return launch_lanes<Bf16, false>(a, s);
    if (!waves) {
        if (a.c.dim <= 32) return launch_part<Bf16, 4, 1, true>(a, s);
        if (a.c.dim <= 64) return launch_part<Bf16, 8, 1, true>(a, s);
        return launch_part<Bf16, 16, 1, true>(a, s);
    }
    if (type == EHIP_CACHE_BF16)
        return whole_rows(a.c, 8) ? launch_mfma<Bf16, true>(a, s) : launch_mfma<Bf16, false>(a, s);
    // Reads of whole pieces in 8 bits: of 16 values, or of 8 in heads of up to 32.
    return whole_rows(a.c, a.c.dim <= 32 ? 8 : 16) ? launch_mfma<Int8, true>(a, s)
                                                   : launch_mfma<Int8, false>(a, s);
}

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
    if (cache->type == EHIP_CACHE_I8) return append_i8(x, s);
    return cache->type == EHIP_CACHE_F32 ? append<float>(x, s) : append<Bf16>(x, s);
}

int ehip_cache_read_f32(const ehip_cache_t* cache, const int32_t* starts, const int32_t* cu,
                        int64_t tokens, float* k, int64_t ld_k, float* v, int64_t ld_v,
                        void* stream) {
    EHIP_READY();
    Cache c;
    if (int rc = check("cache_read", cache, c)) return rc;
    const int64_t n = c.kv_heads * c.dim;
    if (n > kMaxLength) return fail(EHIP_EINVAL, "cache_read: rows of %lld values", (long long)n);
    if (tokens < 0 || tokens > kMaxBlocks || ld_k < n || ld_v < n ||
        (cu == nullptr && tokens != c.sequences))
        return fail(EHIP_EINVAL, "cache_read: %lld tokens of %lld sequences, rows %lld and %lld "
                                 "apart",
                    (long long)tokens, (long long)c.sequences, (long long)ld_k, (long long)ld_v);
    if (tokens == 0 || c.sequences == 0) return EHIP_OK;
    if (k == nullptr || v == nullptr || starts == nullptr)
        return fail(EHIP_EINVAL, "cache_read: null tensor");
    hipStream_t s = as_stream(stream);
    const Read x{c, starts, cu, int(tokens), k, ld_k, v, ld_v};
    if (cache->type == EHIP_CACHE_I8) return read<Int8>(x, s);
    return cache->type == EHIP_CACHE_F32 ? read<float>(x, s) : read<Bf16>(x, s);
}

int64_t ehip_attention_paged_workspace(const ehip_cache_t* cache, int64_t heads,
                                       int64_t longest) {
    Cache c;
    if (check("attention_paged", cache, c) || check_heads("attention_paged", c, heads, longest))
        return -1;
    return c.sequences == 0
               ? 0
               : int64_t(part_bytes(c, heads, cut_of(c, heads, longest, waves_of(c, heads, longest, cache->type))
                                        .workers));
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
    const Cut cut = cut_of(c, heads, longest, waves_of(c, heads, longest, cache->type));
    const size_t need = part_bytes(c, heads, cut.workers);
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
    a.tile = cut.tile;
    a.workers = cut.workers;
    const int64_t parts = heads * (cut.workers + c.sequences);
    a.part_stats = static_cast<float2*>(workspace);
    a.part_out = reinterpret_cast<float*>(a.part_stats + parts);
    a.first = reinterpret_cast<int*>(a.part_out + parts * c.dim);
    hipStream_t s = as_stream(stream);
    if (int rc = launch_parts(a, cache->type, cut.waves, s)) return rc;
    const int64_t rows = c.sequences * heads;
    switch (join_waves(rows, cut.workers / c.sequences)) {
        case 1: return launch_join<1>(a, rows, s);
        case kPagedWaves: return launch_join<kPagedWaves>(a, rows, s);
        default: return launch_join<kManyJoinWaves>(a, rows, s);
    }
}

}  // extern "C"
