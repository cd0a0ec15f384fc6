// attention_packed.hip -- attention over packed sequences of different lengths with grouped heads,
// forward and backward, with no scores in HBM.
//
//   s_ij = scale (q_i . k_j), lse_i = log sum_j exp(s_ij), out_i = sum_j exp(s_ij - lse_i) v_j
//   p_ij = exp(s_ij - lse_i), delta_i = g_i . out_i, ds_ij = p_ij (g_i . v_j - delta_i)
//   dv_j = sum_i p_ij g_i, dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i
//
// over the pairs (i, j) that the lengths and the causal mask let see each other. The offsets of the
// sequences stay on the device: a launch has a block for every slot that a tile of rows could take
// (find_tile), and a block without a tile ends at once.

#include "attention_tile.hpp"
#include "common.hpp"

#include <cmath>

namespace ehip {
namespace {

constexpr int kMaxDim = 128;
constexpr int kThreads = 256;
constexpr int kRows = 128;  // rows (queries or keys) of one block, 32 a wave

struct Packed {
    const float *q, *k, *v;
    int64_t ld_q, ld_k, ld_v;
    const int32_t *cu_q, *cu_k;
    int sequences;
    int total_q, total_k;
    int heads, kv_heads, dim;
    float scale;
    int causal;
    float* out;
    int64_t ld_out;
    float* lse;
    const float* grad;
    int64_t ld_grad;
    float *dq, *dk, *dv;
    int64_t ld_dq, ld_dk, ld_dv;
    float* delta;  // (total_q, heads)
};

// A sequence's rows and the block's tile of them; rows == 0 where the block has none.
struct Tile {
    int q0, nq, k0, nk;  // first rows and lengths of the sequence
    int first, rows;     // the tile, counted from the sequence's first row
};

__device__ __forceinline__ int offset_at(const int32_t* cu, int s, int total) {
    const int x = cu[s];
    return x < 0 ? 0 : (x > total ? total : x);
}

// The tile of slot `slot` when every sequence's rows (offsets cu) are cut into tiles of `size`.
// Sequence s takes the slots from cu[s] / size + s on: that is at least one more for every
// sequence before it than its tiles need, as ceil((b - a) / size) <= b / size - a / size + 1 in
// whole numbers, so no sum over the sequences is needed to find a tile. The last s whose first
// slot is not past `slot` is searched 64 candidates at a time, a lane each; every wave of the block
// finds the same. Later queries and earlier keys come first within a sequence: under a causal mask
// they meet the most.
__device__ __forceinline__ Tile find_tile(const Packed& a, bool keys, int slot, int size) {
    const int32_t* cu = keys ? a.cu_k : a.cu_q;
    const int total = keys ? a.total_k : a.total_q;
    const int lane = int(threadIdx.x) & 63;
    int lo = 0, n = a.sequences;  // the answer, if any, is in [lo, lo + n)
    while (n > 0) {
        const int step = (n + 63) / 64;
        const int s = lo + lane * step;
        const bool at = lane * step < n && offset_at(cu, s, total) / size + s <= slot;
        const int c = __popcll(__ballot(at));
        if (c == 0) break;
        n = n - (c - 1) * step;
        lo += (c - 1) * step;
        n = n < step ? n : step;
        if (step == 1) break;
    }
    Tile t{};
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int begin = offset_at(cu, lo, total);
    int end = offset_at(cu, lo + 1, total);
    end = end < begin ? begin : end;
    const int tiles = (end - begin + size - 1) / size;
    const int at = slot - (begin / size + lo);
    if (at < 0 || at >= tiles) return t;
    t.q0 = offset_at(a.cu_q, lo, a.total_q);
    t.nq = offset_at(a.cu_q, lo + 1, a.total_q) - t.q0;
    t.k0 = offset_at(a.cu_k, lo, a.total_k);
    t.nk = offset_at(a.cu_k, lo + 1, a.total_k) - t.k0;
    t.nq = t.nq < 0 ? 0 : t.nq;
    t.nk = t.nk < 0 ? 0 : t.nk;
    t.first = (keys ? at : tiles - 1 - at) * size;
    t.rows = end - begin - t.first;
    t.rows = t.rows < size ? t.rows : size;
    return t;
}

// Keys that query i of the sequence sees: 0 .. count - 1.
__device__ __forceinline__ int visible(const Packed& a, const Tile& t, int i) {
    if (!a.causal) return t.nk;
    const int64_t n = int64_t(i) + t.nk - t.nq + 1;
    return n < 0 ? 0 : (n > t.nk ? t.nk : int(n));
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

__device__ __forceinline__ float dot(const float* __restrict__ x, const float* __restrict__ y,
                                     int n) {
    float s = 0.0f;
    for (int c = 0; c < n; ++c) s = __builtin_fmaf(x[c], y[c], s);
    return s;
}

// ------------------------------------------------------- one row by one wave
// The formulas as they stand, a lane for a key (or query) at a time and then a lane for a column;
// only what the row sees is read.

__device__ void forward_row(const Packed& a, const Tile& t, int h, int i) {
    const int lane = int(threadIdx.x) & 63;
    const int n = visible(a, t, i), c = h / (a.heads / a.kv_heads);
    const float* q = a.q + int64_t(t.q0 + i) * a.ld_q + int64_t(h) * a.dim;
    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    float m = -INFINITY;
    bool bad = false;  // a score that is NaN: fmaxf passes over it
    for (int j = lane; j < n; j += 64) {
        const float s = dot(q, k + j * a.ld_k, a.dim) * a.scale;
        m = fmaxf(m, s);
        bad |= s != s;
    }
    m = wave_max(m);
    if (__any(bad)) m = NAN;
    float sum = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int j = lane; j < n; j += 64) sum += expf(dot(q, k + j * a.ld_k, a.dim) * a.scale - m);
    sum = wave_sum(sum);
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane;
        float p = 0.0f;  // divided here: the sums stay in range with v's values
        if (j < n) p = expf(dot(q, k + j * a.ld_k, a.dim) * a.scale - m) / sum;
        const int count = n - j0 < 64 ? n - j0 : 64;
        for (int u = 0; u < count; ++u) {
            const float w = __shfl(p, u);
            const float* row = v + (j0 + u) * a.ld_v;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (lane + 64 * e < a.dim) acc[e] = __builtin_fmaf(w, row[lane + 64 * e], acc[e]);
        }
    }
    float* out = a.out + int64_t(t.q0 + i) * a.ld_out + int64_t(h) * a.dim;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < a.dim) out[lane + 64 * e] = acc[e];
    if (lane == 0)
        a.lse[int64_t(t.q0 + i) * a.heads + h] = n == 0 ? -INFINITY : m + logf(sum);
}

// ds_ij, and p_ij through p.
__device__ __forceinline__ float pair_gradient(const Packed& a, const float* q, const float* g,
                                               const float* k, const float* v, float lse,
                                               float delta, float& p) {
    p = expf(dot(q, k, a.dim) * a.scale - lse);
    return p * (dot(g, v, a.dim) - delta);
}

__device__ void dq_row(const Packed& a, const Tile& t, int h, int i, float delta) {
    const int lane = int(threadIdx.x) & 63;
    const int n = visible(a, t, i), c = h / (a.heads / a.kv_heads);
    const int64_t row = t.q0 + i;
    const float* q = a.q + row * a.ld_q + int64_t(h) * a.dim;
    const float* g = a.grad + row * a.ld_grad + int64_t(h) * a.dim;
    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const float lse = a.lse[row * a.heads + h];
    float acc[2] = {0.0f, 0.0f};
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane;
        float p, ds = 0.0f;
        if (j < n) ds = pair_gradient(a, q, g, k + j * a.ld_k, v + j * a.ld_v, lse, delta, p);
        const int count = n - j0 < 64 ? n - j0 : 64;
        for (int u = 0; u < count; ++u) {
            const float w = __shfl(ds, u);
            const float* x = k + (j0 + u) * a.ld_k;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (lane + 64 * e < a.dim) acc[e] = __builtin_fmaf(w, x[lane + 64 * e], acc[e]);
        }
    }
    float* dq = a.dq + row * a.ld_dq + int64_t(h) * a.dim;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < a.dim) dq[lane + 64 * e] = acc[e] * a.scale;
}

__device__ void dkv_row(const Packed& a, const Tile& t, int c, int j) {
    const int lane = int(threadIdx.x) & 63, group = a.heads / a.kv_heads;
    const int64_t row = t.k0 + j;
    const float* k = a.k + row * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + row * a.ld_v + int64_t(c) * a.dim;
    // The first query that sees key j.
    int64_t start = a.causal ? int64_t(j) - t.nk + t.nq : 0;
    start = start < 0 ? 0 : start;
    float ak[2] = {0.0f, 0.0f}, av[2] = {0.0f, 0.0f};
    for (int h = c * group; h < (c + 1) * group; ++h)
        for (int64_t i0 = start; i0 < t.nq; i0 += 64) {
            const int64_t i = i0 + lane;
            float p = 0.0f, ds = 0.0f;
            if (i < t.nq) {
                const int64_t at = t.q0 + i;
                ds = pair_gradient(a, a.q + at * a.ld_q + int64_t(h) * a.dim,
                                   a.grad + at * a.ld_grad + int64_t(h) * a.dim, k, v,
                                   a.lse[at * a.heads + h], a.delta[at * a.heads + h], p);
            }
            const int count = t.nq - i0 < 64 ? int(t.nq - i0) : 64;
            for (int u = 0; u < count; ++u) {
                const float wp = __shfl(p, u), wd = __shfl(ds, u);
                const float* x = a.q + (t.q0 + i0 + u) * a.ld_q + int64_t(h) * a.dim;
                const float* g = a.grad + (t.q0 + i0 + u) * a.ld_grad + int64_t(h) * a.dim;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (lane + 64 * e < a.dim) {
                        ak[e] = __builtin_fmaf(wd, x[lane + 64 * e], ak[e]);
                        av[e] = __builtin_fmaf(wp, g[lane + 64 * e], av[e]);
                    }
            }
        }
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (lane + 64 * e < a.dim) {
            if (a.dk != nullptr)
                a.dk[row * a.ld_dk + int64_t(c) * a.dim + lane + 64 * e] = ak[e] * a.scale;
            if (a.dv != nullptr) a.dv[row * a.ld_dv + int64_t(c) * a.dim + lane + 64 * e] = av[e];
        }
}

// ------------------------------------------------------------------- kernels
// Block = slot * heads + head, the heads of one key head 8 (or any multiple of the key heads) apart:
// with the dispatcher's round robin over the eight XCDs they meet their keys in one L2.

__device__ __forceinline__ int head_of(const Packed& a, int x) {
    return x % a.kv_heads * (a.heads / a.kv_heads) + x / a.kv_heads;
}

template <int DP, int BN, int WAVES, bool VEC>
__global__ __launch_bounds__(64 * WAVES, 2) void packed_forward(Packed a) {
    using namespace attention;
    using KeyTile = RowTile<BN, DP, 64 * WAVES, VEC>;
    using ValueTile = ColTile<BN, DP, 64 * WAVES>;
    constexpr int kTile = KeyTile::kBytes + ValueTile::kBytes;
    // Wide heads leave the third parts of the queries, which one product in six takes, in LDS: all
    // of them in registers spill.
    constexpr bool kPark = DP > 64;
    constexpr int kParked = kPark ? WAVES * (DP / 16) * 1024 : 0;
    __shared__ __attribute__((aligned(16))) char lds[2 * kTile + kParked];
    const int h = head_of(a, int(blockIdx.x % a.heads));
    const Tile t = find_tile(a, false, int(blockIdx.x / a.heads), 32 * WAVES);
    if (t.rows == 0) return;
    const int c = h / (a.heads / a.kv_heads);
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int lane = int(threadIdx.x) & 63;
    const int mine = 32 * wave + (lane & 31);  // the lane's query, of the tile
    const int i = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int limit = visible(a, t, i);
    const int last = 32 * wave + 31 < t.rows ? 32 * wave + 31 : t.rows - 1;
    const int end = visible(a, t, t.first + t.rows - 1);
    const int wave_end = 32 * wave < t.rows ? visible(a, t, t.first + last) : 0;
    const int wave_all = visible(a, t, t.first + 32 * wave);  // keys that all its queries see

    // exp(scale s - m) as 2^(c2 s - m2); a negative scale's sign goes into q. Weights are 2^-24 of
    // their value, so that sums over the values stay in their range.
    const float c2 = fabsf(a.scale) * 1.44269504088896340736f;
    bf16x8 q[DP / 16][3];
    own_row<DP, VEC>(a.q + int64_t(t.q0 + i) * a.ld_q + int64_t(h) * a.dim, a.dim,
                     a.scale < 0.0f ? -1.0f : 1.0f, q);
    char* const parked = lds + 2 * kTile + (wave * (DP / 16) * 64 + lane) * 16;
    if constexpr (kPark) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
            *reinterpret_cast<bf16x8*>(parked + 1024 * ks) = q[ks][2];
    }
    floatx16 o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] = zeros();
    float top = -INFINITY, shift = 24.0f, sum = 0.0f;

    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const int ld_k = int(a.ld_k), ld_v = int(a.ld_v);
    KeyTile kt(ld_k, a.dim);
    ValueTile vt(ld_v, a.dim);
    // The tile of keys from j on: into registers, and from there into its half of the LDS.
    const auto load = [&](int j) {
        if (j >= end) return;
        kt.load(k + int64_t(j) * ld_k, ld_k, t.nk - j, a.dim);
        vt.load(v + int64_t(j) * ld_v, ld_v, t.nk - j, a.dim);
    };
    const auto stage = [&](int j) {
        if (j >= end) return;
        char* const at = lds + (j / BN & 1) * kTile;
        kt.store(at, t.nk - j, a.dim);
        vt.store(at + KeyTile::kBytes, t.nk - j, a.dim);
    };
    load(0);
    stage(0);
    load(BN);
    __syncthreads();
    for (int j0 = 0; j0 < end; j0 += BN) {
        // One wave of a SIMD stages the next tile before its products, the other one after them:
        // one's conversions run beside the other's matrix instructions.
        const char* const lds_k = lds + (j0 / BN & 1) * kTile;
        const char* const lds_v = lds_k + KeyTile::kBytes;
        if (wave < WAVES / 2) {
            stage(j0 + BN);
            load(j0 + 2 * BN);
        }
        if (j0 < wave_end) {
            floatx16 s[BN / 32];
#pragma unroll
            for (int b = 0; b < BN / 32; ++b) s[b] = zeros();
            constexpr int NB = BN / 32, kScores = NB * (DP / 16);
            bf16x8 f[2][3];
            KeyTile::block(lds_k, 0, 0, f[0]);
#pragma unroll
            for (int n = 0; n < kScores; ++n) {
                const int ks = n / NB;
                if (kPark && n % NB == 0)
                    q[ks][2] = *reinterpret_cast<const bf16x8*>(parked + 1024 * ks);
                if (n + 1 < kScores)
                    KeyTile::block(lds_k, (n + 1) % NB, (n + 1) / NB, f[(n + 1) & 1]);
                keep_order();
                multiply(s[n % NB], f[n & 1], q[ks]);
                keep_order();
            }
            if (j0 + BN > wave_all) {
#pragma unroll
                for (int b = 0; b < BN / 32; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (j0 + 32 * b + row_of(r) >= limit) s[b][r] = -INFINITY;
            }
            float m = top;
#pragma unroll
            for (int b = 0; b < BN / 32; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) m = fmaxf(m, s[b][r]);
            m = fmaxf(m, __shfl_xor(m, 32));
            const float next = m == -INFINITY ? 24.0f : __builtin_fmaf(m, c2, 24.0f);
            const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(shift - next);
            top = m;
            shift = next;
            float part = 0.0f;
            bf16x8 p[BN / 16][3];
#pragma unroll
            for (int b = 0; b < BN / 32; ++b) {
                float w[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    w[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], c2, -shift));
                    part += w[r];
                }
                split8(w, p[2 * b]);
                split8(w + 8, p[2 * b + 1]);
            }
            sum = __builtin_fmaf(sum, keep, part);
            // The tile's sum apart from the running one: that is rounded to nearest once a tile,
            // where the instruction drops low bits towards minus infinity.
            constexpr int NU = BN / 16, kSums = NU * (DP / 32);
            floatx16 x = zeros();
            ValueTile::block(lds_v, 0, 0, f[0]);
#pragma unroll
            for (int n = 0; n < kSums; ++n) {
                if (n + 1 < kSums)
                    ValueTile::block(lds_v, (n + 1) / NU, (n + 1) % NU, f[(n + 1) & 1]);
                keep_order();
                multiply(x, f[n & 1], p[n % NU]);
                keep_order();
                if (n % NU == NU - 1) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        o[n / NU][r] = __builtin_fmaf(o[n / NU][r], keep, x[r]);
                    x = zeros();
                }
            }
        }
        if (wave >= WAVES / 2) {
            stage(j0 + BN);
            load(j0 + 2 * BN);
        }
        __syncthreads();
    }

    // Rows that saw something and have no finite result are formed again by the formula: a NaN or
    // an infinity where it counts, or one in a place of theirs that they do not see (0 times it).
    sum += __shfl_xor(sum, 32);
    const float inv = limit > 0 ? 1.0f / sum : 0.0f;
    bool fine = sum > 0.0f && sum < INFINITY;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[db][r] *= inv;
            fine = fine && fabsf(o[db][r]) < INFINITY;
        }
    fine = fine || limit == 0;
    const uint64_t again = __ballot(!fine && mine < t.rows);
    if (mine < t.rows) {
        store_own<DP, VEC>(a.out + int64_t(t.q0 + i) * a.ld_out + int64_t(h) * a.dim, a.dim, o);
        // shift ln 2 in two parts: ln 2 = hi + lo.
        if (lane < 32)
            a.lse[int64_t(t.q0 + i) * a.heads + h] =
                limit == 0 ? -INFINITY
                           : __builtin_fmaf(shift, 0.693147182464599609375f,
                                            __builtin_fmaf(shift, -1.904654323148236017e-9f,
                                                           logf(sum)));
    }
    for (uint32_t rows = uint32_t(again) | uint32_t(again >> 32); rows != 0; rows &= rows - 1)
        forward_row(a, t, h, t.first + 32 * wave + __builtin_ctz(rows));
}

// s, and so p_ij, for the pairs of the lane's own row and a block of 32 streamed ones is formed
// again from the inputs, dp likewise; then the block's share of the gradients. The queries' kernel
// also leaves delta for the keys' one.
template <int DP, int BN, bool VEC, int MINW>
__global__ __launch_bounds__(kThreads, MINW) void packed_backward_q(Packed a) {
    using namespace attention;
    using KeyTile = RowTile<BN, DP, kThreads, VEC>;
    using KeyColumns = ColTile<BN, DP, kThreads>;
    __shared__ __attribute__((aligned(16))) char lds[2 * KeyTile::kBytes + KeyColumns::kBytes];
    char* const lds_v = lds + KeyTile::kBytes;
    char* const lds_c = lds_v + KeyTile::kBytes;
    const int h = head_of(a, int(blockIdx.x % a.heads));
    const Tile t = find_tile(a, false, int(blockIdx.x / a.heads), kRows);
    if (t.rows == 0) return;
    const int c = h / (a.heads / a.kv_heads);
    const int wave = int(threadIdx.x) / 64, lane = int(threadIdx.x) & 63;
    const int mine = 32 * wave + (lane & 31);  // the lane's query, of the tile
    const int i = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int64_t row = t.q0 + i;
    const int limit = visible(a, t, i);
    const int last = 32 * wave + 31 < t.rows ? 32 * wave + 31 : t.rows - 1;
    const int end = visible(a, t, t.first + t.rows - 1);
    const int wave_end = 32 * wave < t.rows ? visible(a, t, t.first + last) : 0;
    const int wave_all = visible(a, t, t.first + 32 * wave);  // keys that all its queries see

    const float* gr = a.grad + row * a.ld_grad + int64_t(h) * a.dim;
    const float delta = own_dot<DP, VEC>(gr, a.out + row * a.ld_out + int64_t(h) * a.dim, a.dim);
    if (lane < 32 && mine < t.rows) a.delta[row * a.heads + h] = delta;
    if (a.dq == nullptr) return;
    const float c2 = a.scale * 1.44269504088896340736f;
    const float shift = limit > 0 ? a.lse[row * a.heads + h] * 1.44269504088896340736f : 0.0f;
    bf16x8 q[DP / 16][3], g[DP / 16][3];
    own_row<DP, VEC>(a.q + row * a.ld_q + int64_t(h) * a.dim, a.dim, 1.0f, q);
    own_row<DP, VEC>(gr, a.dim, 1.0f, g);
    floatx16 dq[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) dq[db] = zeros();

    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const int ld_k = int(a.ld_k), ld_v = int(a.ld_v);
    KeyTile kt(ld_k, a.dim), vt(ld_v, a.dim);
    KeyColumns ct(ld_k, a.dim);
    if (end > 0) {
        kt.load(k, ld_k, t.nk, a.dim);
        vt.load(v, ld_v, t.nk, a.dim);
        ct.load(k, ld_k, t.nk, a.dim);
    }
    for (int j0 = 0; j0 < end; j0 += BN) {
        __syncthreads();
        kt.store(lds, t.nk - j0, a.dim);
        vt.store(lds_v, t.nk - j0, a.dim);
        ct.store(lds_c, t.nk - j0, a.dim);
        const int j1 = j0 + BN;
        if (j1 < end) {
            kt.load(k + int64_t(j1) * ld_k, ld_k, t.nk - j1, a.dim);
            vt.load(v + int64_t(j1) * ld_v, ld_v, t.nk - j1, a.dim);
            ct.load(k + int64_t(j1) * ld_k, ld_k, t.nk - j1, a.dim);
        }
        __syncthreads();
        if (j0 >= wave_end) continue;
        const bool edge = j1 > wave_all;
        bf16x8 w[BN / 16][3];
#pragma unroll
        for (int b = 0; b < BN / 32; ++b) {
            floatx16 s = zeros(), dp = zeros();
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                bf16x8 f[3];
                KeyTile::block(lds, b, ks, f);
                multiply(s, f, q[ks]);
                KeyTile::block(lds_v, b, ks, f);
                multiply(dp, f, g[ks]);
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                ds[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -shift)) * (dp[r] - delta);
                if (edge && j0 + 32 * b + row_of(r) >= limit) ds[r] = 0.0f;
            }
            split8(ds, w[2 * b]);
            split8(ds + 8, w[2 * b + 1]);
        }
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
            floatx16 x = zeros();
#pragma unroll
            for (int u = 0; u < BN / 16; ++u) {
                bf16x8 f[3];
                KeyColumns::block(lds_c, db, u, f);
                multiply(x, f, w[u]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[db][r] += x[r];
        }
    }
    bool fine = true;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dq[db][r] = limit > 0 ? dq[db][r] * a.scale : 0.0f;
            fine = fine && fabsf(dq[db][r]) < INFINITY;
        }
    const uint64_t again = __ballot(!fine && mine < t.rows);
    if (mine < t.rows)
        store_own<DP, VEC>(a.dq + row * a.ld_dq + int64_t(h) * a.dim, a.dim, dq);
    for (uint32_t rows = uint32_t(again) | uint32_t(again >> 32); rows != 0; rows &= rows - 1) {
        const int r = __builtin_ctz(rows);
        dq_row(a, t, h, t.first + 32 * wave + r, __shfl(delta, r));
    }
}

template <int DP, bool VEC, int MINW>
__global__ __launch_bounds__(kThreads, MINW) void packed_backward_kv(Packed a) {
    using namespace attention;
    constexpr int BN = 32;
    using QueryTile = RowTile<BN, DP, kThreads, VEC>;
    using QueryColumns = ColTile<BN, DP, kThreads>;
    __shared__ __attribute__((aligned(16))) char
        lds[2 * QueryTile::kBytes + 2 * QueryColumns::kBytes + 2 * BN * sizeof(float)];
    char* const lds_g = lds + QueryTile::kBytes;
    char* const lds_qc = lds_g + QueryTile::kBytes;
    char* const lds_gc = lds_qc + QueryColumns::kBytes;
    float* const lds_shift = reinterpret_cast<float*>(lds_gc + QueryColumns::kBytes);
    float* const lds_delta = lds_shift + BN;
    const int c = int(blockIdx.x % a.kv_heads), group = a.heads / a.kv_heads;
    const Tile t = find_tile(a, true, int(blockIdx.x / a.kv_heads), kRows);
    if (t.rows == 0) return;
    const int wave = int(threadIdx.x) / 64, lane = int(threadIdx.x) & 63;
    const int mine = 32 * wave + (lane & 31);  // the lane's key, of the tile
    const int j = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int64_t row = t.k0 + j;
    // The first query that sees a key, and the first ones of the block and of the wave.
    const auto first_of = [&](int key) {
        const int64_t n = a.causal ? int64_t(key) - t.nk + t.nq : 0;
        return n < 0 ? 0 : int(n);
    };
    const int from = first_of(j), start = first_of(t.first);
    const int wave_start = first_of(t.first + 32 * wave);
    const int wave_all = first_of(t.first + 32 * wave + 31);

    const float c2 = a.scale * 1.44269504088896340736f;
    bf16x8 k[DP / 16][3], v[DP / 16][3];
    own_row<DP, VEC>(a.k + row * a.ld_k + int64_t(c) * a.dim, a.dim, 1.0f, k);
    own_row<DP, VEC>(a.v + row * a.ld_v + int64_t(c) * a.dim, a.dim, 1.0f, v);
    floatx16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
        dk[db] = zeros();
        dv[db] = zeros();
    }
    const int ld_q = int(a.ld_q), ld_g = int(a.ld_grad);
    const int steps = start < t.nq ? (t.nq - start + BN - 1) / BN : 0;
    QueryTile qt(ld_q, a.dim), gt(ld_g, a.dim);
    QueryColumns qc(ld_q, a.dim), gc(ld_g, a.dim);
    float stat = 0.0f;  // of the thread's query: lse (threads 0..31), delta (32..63)
    // Tile n: head n / steps of the group, its queries from start + n % steps * BN on.
    const auto load = [&](int n) {
        const int h = c * group + n / steps, i0 = start + n % steps * BN;
        const int64_t at = t.q0 + i0;
        const int left = t.nq - i0;
        const float* q = a.q + at * a.ld_q + int64_t(h) * a.dim;
        const float* g = a.grad + at * a.ld_grad + int64_t(h) * a.dim;
        qt.load(q, ld_q, left, a.dim);
        gt.load(g, ld_g, left, a.dim);
        qc.load(q, ld_q, left, a.dim);
        gc.load(g, ld_g, left, a.dim);
        if (wave == 0) {
            const int r = (lane & 31) < left ? lane & 31 : left - 1;
            stat = (lane < 32 ? a.lse : a.delta)[(at + r) * a.heads + h];
        }
    };
    const int count = steps * group;
    if (count > 0) load(0);
    for (int n = 0; n < count; ++n) {
        const int i0 = start + n % steps * BN, left = t.nq - i0;
        __syncthreads();
        qt.store(lds, left, a.dim);
        gt.store(lds_g, left, a.dim);
        qc.store(lds_qc, left, a.dim);
        gc.store(lds_gc, left, a.dim);
        if (wave == 0) lds_shift[lane] = lane < 32 ? stat * 1.44269504088896340736f : stat;
        if (n + 1 < count) load(n + 1);
        __syncthreads();
        if (i0 + BN <= wave_start) continue;
        const bool edge = i0 < wave_all || left < BN;
        floatx16 s = zeros(), dp = zeros();
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
            bf16x8 f[3];
            QueryTile::block(lds, 0, ks, f);
            multiply(s, f, k[ks]);
            QueryTile::block(lds_g, 0, ks, f);
            multiply(dp, f, v[ks]);
        }
        float p[16], ds[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int at = row_of(r);
            p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -lds_shift[at]));
            ds[r] = p[r] * (dp[r] - lds_delta[at]);
            if (edge && (i0 + at < from || at >= left)) p[r] = ds[r] = 0.0f;
        }
        bf16x8 wp[2][3], wd[2][3];
        split8(p, wp[0]);
        split8(p + 8, wp[1]);
        split8(ds, wd[0]);
        split8(ds + 8, wd[1]);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
            floatx16 x = zeros(), y = zeros();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                bf16x8 f[3];
                QueryColumns::block(lds_gc, db, u, f);
                multiply(x, f, wp[u]);
                QueryColumns::block(lds_qc, db, u, f);
                multiply(y, f, wd[u]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dv[db][r] += x[r];
                dk[db][r] += y[r];
            }
        }
    }
    bool fine = true;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dk[db][r] *= a.scale;
            fine = fine && fabsf(dk[db][r]) < INFINITY && fabsf(dv[db][r]) < INFINITY;
        }
    const uint64_t again = __ballot(!fine && mine < t.rows);
    if (mine < t.rows) {
        if (a.dk != nullptr)
            store_own<DP, VEC>(a.dk + row * a.ld_dk + int64_t(c) * a.dim, a.dim, dk);
        if (a.dv != nullptr)
            store_own<DP, VEC>(a.dv + row * a.ld_dv + int64_t(c) * a.dim, a.dim, dv);
    }
    for (uint32_t rows = uint32_t(again) | uint32_t(again >> 32); rows != 0; rows &= rows - 1)
        dkv_row(a, t, c, t.first + 32 * wave + __builtin_ctz(rows));
}

// ---------------------------------------------------------------- host checks

int64_t slots(int64_t total, int64_t sequences, int rows = kRows) {
    return total / rows + sequences;
}

// Tiles address their rows by 32-bit byte offsets from the first one.
constexpr int64_t kMaxLd = int64_t(1) << 22;

int fill(const char* name, const ehip_attention_packed_t* d, Packed& a) {
    if (d == nullptr) return fail(EHIP_EINVAL, "%s: null descriptor", name);
    if (d->sequences < 0 || d->total_q < 0 || d->total_k < 0 || d->heads < 1 || d->kv_heads < 1 ||
        d->heads % d->kv_heads != 0 || d->head_dim < 1 || d->head_dim > kMaxDim)
        return fail(EHIP_EINVAL,
                    "%s: %lld sequences, %lld and %lld rows, %lld heads over %lld of %lld values",
                    name, (long long)d->sequences, (long long)d->total_q, (long long)d->total_k,
                    (long long)d->heads, (long long)d->kv_heads, (long long)d->head_dim);
    constexpr int64_t kBlocks = (int64_t(1) << 24) - 1;
    if (d->heads > kBlocks || d->sequences > kBlocks || d->total_q > INT32_MAX ||
        d->total_k > INT32_MAX ||
        slots(d->total_q > d->total_k ? d->total_q : d->total_k, d->sequences) * d->heads > kBlocks)
        return fail(EHIP_EINVAL, "%s: %lld x %lld rows of %lld heads are too many", name,
                    (long long)d->total_q, (long long)d->total_k, (long long)d->heads);
    const int64_t wide = d->heads * d->head_dim, narrow = d->kv_heads * d->head_dim;
    if (d->ld_q < wide || d->ld_out < wide || d->ld_k < narrow || d->ld_v < narrow ||
        d->ld_q > kMaxLd || d->ld_k > kMaxLd || d->ld_v > kMaxLd)
        return fail(EHIP_EINVAL, "%s: leading dimension below the row's length or above 2^22",
                    name);
    if (d->sequences > 0 && (d->cu_q == nullptr || d->cu_k == nullptr))
        return fail(EHIP_EINVAL, "%s: null offsets", name);
    if ((d->total_q > 0 && (d->q == nullptr || d->out == nullptr || d->lse == nullptr)) ||
        (d->total_k > 0 && (d->k == nullptr || d->v == nullptr)))
        return fail(EHIP_EINVAL, "%s: null tensor", name);
    a = Packed{};
    a.q = d->q;
    a.k = d->k;
    a.v = d->v;
    a.ld_q = d->ld_q;
    a.ld_k = d->ld_k;
    a.ld_v = d->ld_v;
    a.cu_q = d->cu_q;
    a.cu_k = d->cu_k;
    a.sequences = int(d->sequences);
    a.total_q = int(d->total_q);
    a.total_k = int(d->total_k);
    a.heads = int(d->heads);
    a.kv_heads = int(d->kv_heads);
    a.dim = int(d->head_dim);
    a.scale = d->scale;
    a.causal = d->causal != 0;
    a.out = d->out;
    a.ld_out = d->ld_out;
    a.lse = d->lse;
    return EHIP_OK;
}

template <int DP, int BN, int WAVES, bool VEC>
int launch_forward(const Packed& a, hipStream_t s) {
    const unsigned blocks = unsigned(slots(a.total_q, a.sequences, 32 * WAVES) * a.heads);
    EHIP_LAUNCH("attention_packed", (packed_forward<DP, BN, WAVES, VEC>), dim3(blocks),
                dim3(64 * WAVES), 0, s, a);
    return EHIP_OK;
}

template <int DP, bool VEC>
int launch_backward(const Packed& a, hipStream_t s) {
    if (a.total_q > 0 && (a.dq != nullptr || a.dk != nullptr)) {
        const unsigned blocks = unsigned(slots(a.total_q, a.sequences) * a.heads);
        EHIP_LAUNCH("attention_packed_backward_q", (packed_backward_q<DP, 32, VEC, DP <= 64 ? 2 : 1>),
                    dim3(blocks), dim3(kThreads), 0, s, a);
    }
    if (a.total_k > 0 && (a.dk != nullptr || a.dv != nullptr)) {
        const unsigned blocks = unsigned(slots(a.total_k, a.sequences) * a.kv_heads);
        EHIP_LAUNCH("attention_packed_backward_kv", (packed_backward_kv<DP, VEC, DP <= 32 ? 2 : 1>),
                    dim3(blocks), dim3(kThreads), 0, s, a);
    }
    return EHIP_OK;
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int ehip_attention_packed_f32(const ehip_attention_packed_t* desc, void* stream) {
    EHIP_READY();
    Packed a;
    if (int rc = fill("attention_packed", desc, a)) return rc;
    if (a.sequences == 0 || a.total_q == 0) return EHIP_OK;
    const bool vec = a.dim % 8 == 0;
    if (a.dim <= 32) return vec ? launch_forward<32, 64, 8, true>(a, as_stream(stream))
                                : launch_forward<32, 64, 8, false>(a, as_stream(stream));
    if (a.dim <= 64) return vec ? launch_forward<64, 64, 8, true>(a, as_stream(stream))
                                : launch_forward<64, 64, 8, false>(a, as_stream(stream));
    if (a.dim <= 96) return vec ? launch_forward<96, 32, 8, true>(a, as_stream(stream))
                                : launch_forward<96, 32, 8, false>(a, as_stream(stream));
    return vec ? launch_forward<128, 32, 8, true>(a, as_stream(stream))
               : launch_forward<128, 32, 8, false>(a, as_stream(stream));
}

int64_t ehip_attention_packed_backward_workspace(const ehip_attention_packed_t* desc) {
    Packed a;
    if (fill("attention_packed_backward", desc, a)) return -1;
    return int64_t(a.total_q) * a.heads * int64_t(sizeof(float));
}

int ehip_attention_packed_backward_f32(const ehip_attention_packed_t* desc, const float* grad,
                                       int64_t ld_grad, float* dq, int64_t ld_dq, float* dk,
                                       int64_t ld_dk, float* dv, int64_t ld_dv, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    EHIP_READY();
    Packed a;
    if (int rc = fill("attention_packed_backward", desc, a)) return rc;
    if (a.sequences == 0) return EHIP_OK;
    const int64_t wide = int64_t(a.heads) * a.dim, narrow = int64_t(a.kv_heads) * a.dim;
    if (a.total_q > 0 && (grad == nullptr || ld_grad < wide || ld_grad > kMaxLd))
        return fail(EHIP_EINVAL, "attention_packed_backward: null gradient, or its leading dimension "
                                 "below the row's length or above 2^22");
    if ((dq != nullptr && ld_dq < wide) || (dk != nullptr && ld_dk < narrow) ||
        (dv != nullptr && ld_dv < narrow))
        return fail(EHIP_EINVAL,
                    "attention_packed_backward: leading dimension below the row's length");
    const size_t need = size_t(a.total_q) * size_t(a.heads) * sizeof(float);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(EHIP_EINVAL,
                    "attention_packed_backward: needs %zu bytes of 16-byte aligned workspace", need);
    a.grad = grad;
    a.ld_grad = ld_grad;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.ld_dq = ld_dq;
    a.ld_dk = ld_dk;
    a.ld_dv = ld_dv;
    a.delta = static_cast<float*>(workspace);
    hipStream_t s = as_stream(stream);
    const bool vec = a.dim % 8 == 0;
    if (a.dim <= 32) return vec ? launch_backward<32, true>(a, s) : launch_backward<32, false>(a, s);
    if (a.dim <= 64) return vec ? launch_backward<64, true>(a, s) : launch_backward<64, false>(a, s);
    if (a.dim <= 96) return vec ? launch_backward<96, true>(a, s) : launch_backward<96, false>(a, s);
    return vec ? launch_backward<128, true>(a, s) : launch_backward<128, false>(a, s);
}

}  // extern "C"
