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

#include <algorithm>
#include <cmath>

namespace ehip {
namespace {

constexpr int kMaxDim = 128;
constexpr int kThreads = 256;
constexpr int kRows = 128;  // rows (queries or keys) of one block, 32 a wave

struct Packed {
    // What the host shares out the work by: a sequence's rows, and how many such there are.
    int64_t each_q, each_k, count_q, count_k;
    const float *q, *k, *v;
    int64_t ld_q, ld_k, ld_v;
    const int32_t *cu_q, *cu_k;
    int sequences;
    int total_q, total_k;
    int heads, kv_heads, dim;
    float scale;
    int causal;
    bool by_work;  // blocks in the order of their work
    float* out;
    int64_t ld_out;
    float* lse;
    int pieces;          // of a tile's keys in the forward; 1: the kernel writes the results
    float2* piece_stats;  // (total_q, heads, pieces): maximum (as 2^x), sum
    float* piece_out;     // (total_q, heads, pieces, dim)
    const float* grad;
    int64_t ld_grad;
    float *dq, *dk, *dv;
    int64_t ld_dq, ld_dk, ld_dv;
    float* delta;             // (total_q, heads)
    // Shares of the gradients: of a piece of the keys or queries that a block passes, and for dk
    // and dv of a query head; or null.
    int pieces_q, pieces_k;
    float* part_q;            // (total_q, heads, pieces_q, dim)
    float *part_k, *part_v;  // (total_k, heads, pieces_k, dim)
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

// Tile `at` of sequence s, which has one.
__device__ __forceinline__ Tile tile_of(const Packed& a, bool keys, int s, int at, int size) {
    Tile t{};
    t.q0 = offset_at(a.cu_q, s, a.total_q);
    t.nq = offset_at(a.cu_q, s + 1, a.total_q) - t.q0;
    t.k0 = offset_at(a.cu_k, s, a.total_k);
    t.nk = offset_at(a.cu_k, s + 1, a.total_k) - t.k0;
    t.nq = t.nq < 0 ? 0 : t.nq;
    t.nk = t.nk < 0 ? 0 : t.nk;
    t.first = at * size;
    t.rows = (keys ? t.nk : t.nq) - t.first;
    t.rows = t.rows < size ? t.rows : size;
    return t;
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
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int begin = offset_at(cu, lo, total), end = offset_at(cu, lo + 1, total);
    const int tiles = end > begin ? (end - begin + size - 1) / size : 0;
    const int at = slot - (begin / size + lo);
    if (at < 0 || at >= tiles) return Tile{};
    return tile_of(a, keys, lo, keys ? at : tiles - 1 - at, size);
}

// The same, under a causal mask and for up to 64 sequences, in the order of the tiles' work, the
// most first: the last blocks to start are the shortest, whatever their sequences. A sequence of n
// tiles has one of work w for every w from 1 to n, so C(w), the sum over the sequences of n - w + 1
// where that is positive, tiles have work w or more, and slot's has the largest w with C(w) > slot.
// A lane has a sequence's n for all of them, and then a candidate w, 64 at a time.
__device__ __forceinline__ Tile find_tile_by_work(const Packed& a, bool keys, int slot, int size) {
    const int32_t* cu = keys ? a.cu_k : a.cu_q;
    const int total = keys ? a.total_k : a.total_q;
    const int lane = int(threadIdx.x) & 63;
    int tiles = 0;
    if (lane < a.sequences) {
        const int begin = offset_at(cu, lane, total), end = offset_at(cu, lane + 1, total);
        tiles = end > begin ? (end - begin + size - 1) / size : 0;
    }
    int n = tiles;  // the answer, if any, is in [w, w + n)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n = max(n, __shfl_xor(n, o));
    n = __builtin_amdgcn_readfirstlane(n);
    int w = 1, above = 0;  // above: C(w + 1)
    while (n > 0) {
        const int step = (n + 63) / 64;
        const int mine = w + min(lane * step, n) - 1;
        int c = 0;
        for (int s = 0; s < a.sequences; ++s)
            c += max(0, __builtin_amdgcn_readlane(tiles, s) - mine);
        const int last = __popcll(__ballot(lane * step < n && c > slot)) - 1;
        if (last < 0) return Tile{};
        if (last < 63) above = __builtin_amdgcn_readlane(c, last + 1);
        w += last * step;
        n = min(n - last * step, step);
        if (step == 1) break;
    }
    uint64_t with = __ballot(tiles >= w);
    for (int skip = slot - above; skip > 0; --skip) with &= with - 1;
    if (n == 0 || with == 0) return Tile{};
    const int s = __builtin_amdgcn_readfirstlane(__builtin_ctzll(with));
    return tile_of(a, keys, s, keys ? __builtin_amdgcn_readlane(tiles, s) - w : w - 1, size);
}

__device__ __forceinline__ Tile block_tile(const Packed& a, bool keys, int slot, int size) {
    return a.by_work ? find_tile_by_work(a, keys, slot, size) : find_tile(a, keys, slot, size);
}

// Keys that query i of the sequence sees: 0 .. count - 1.
__device__ __forceinline__ int visible(const Packed& a, const Tile& t, int i) {
    if (!a.causal) return t.nk;
    const int64_t n = int64_t(i) + t.nk - t.nq + 1;
    return n < 0 ? 0 : (n > t.nk ? t.nk : int(n));
}

// Rows of each of so many pieces of n: what a step takes at a time divides them.
constexpr int kLeastPiece = 128;
__device__ __forceinline__ int piece_length(int n, int pieces) {
    const int each = n / pieces / 64 * 64 + 64;
    return each > kLeastPiece ? each : kLeastPiece;
}

// Piece `piece` of rows [first, end): its first row (end if it is empty), and the row after its
// last.
__device__ __forceinline__ void take_piece(int piece, int pieces, int& first, int& end) {
    if (pieces == 1) return;
    const int64_t each = piece_length(end - first, pieces), begin = first + piece * each;
    first = int(min(begin, int64_t(end)));
    end = int(min(begin + each, int64_t(end)));
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

// ------------------------------------------------------- one row by one wave

// The formulas as they stand, for rows whose tiles gave no finite result; only what the row sees is
// read. Sixteen lanes take one streamed row, its values 16 apart, so that a wave reads four rows at
// a time and U times four ahead: a NaN or an infinity that every row sees has all rows formed here,
// and then the reads' latency bounds a call (4 sequences of 512, 8 heads of 64, the first key
// infinite: 168 us forward and 708 backward; without it 43 and 86; a lane for each key took 760 and
// 4750. One of 16384, 8 heads of 128 over 2: 104 ms and 110, without it 2.8 and 10.1). Where a
// score, lse or delta settles the row as NaN nothing else is read (first key NaN: 39 and 101 us,
// 767 and 4750 without that).

constexpr int kRowLanes = 16, kRowColumns = kMaxDim / kRowLanes;

// A lane's values of a row of `dim`, 0 past its end.
struct Columns {
    float x[kRowColumns];

    __device__ __forceinline__ void load(const float* row, int dim) {
        const int d = int(threadIdx.x) % kRowLanes;
#pragma unroll
        for (int e = 0; e < kRowColumns; ++e) {
            x[e] = 0.0f;
            if (kRowLanes * e < dim && d + kRowLanes * e < dim) x[e] = row[d + kRowLanes * e];
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < kRowColumns; ++e) x[e] = 0.0f;
    }
    __device__ __forceinline__ void add(float w, const Columns& y) {
#pragma unroll
        for (int e = 0; e < kRowColumns; ++e) x[e] = __builtin_fmaf(w, y.x[e], x[e]);
    }
    // The four groups' sums, times `factor`, into a row; or one value for all of it.
    __device__ __forceinline__ void store(float* row, int dim, float factor) {
        const int d = int(threadIdx.x) % kRowLanes, group = (int(threadIdx.x) & 63) / kRowLanes;
#pragma unroll
        for (int e = 0; e < kRowColumns; ++e) {
            if (kRowLanes * e >= dim) break;
            float y = x[e];
            y += __shfl_xor(y, 16);
            y += __shfl_xor(y, 32);
            if (group == 0 && d + kRowLanes * e < dim) row[d + kRowLanes * e] = y * factor;
        }
    }
    __device__ __forceinline__ static void fill(float* row, int dim, float value) {
        for (int d = int(threadIdx.x) & 63; d < dim; d += 64) row[d] = value;
    }
};

// The product of two rows, in each of their sixteen lanes.
__device__ __forceinline__ float dot(const Columns& x, const Columns& y) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < kRowColumns; ++e) s = __builtin_fmaf(x.x[e], y.x[e], s);
#pragma unroll
    for (int o = kRowLanes / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
    return s;
}

// Rows j0 + the lane's group, and every fourth after it, of those before n (the last again past
// it).
template <int U>
__device__ __forceinline__ void load_rows(Columns (&x)[U], const float* base, int64_t ld,
                                          int64_t j0, int64_t n, int dim) {
    const int group = (int(threadIdx.x) & 63) / kRowLanes;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(base + min(j0 + 4 * u + group, n - 1) * ld, dim);
}
__device__ __forceinline__ bool row_is_there(int64_t j0, int u, int64_t n) {
    return j0 + 4 * u + (int(threadIdx.x) & 63) / kRowLanes < n;
}

template <int U>
__device__ void forward_row(const Packed& a, const Tile& t, int h, int i) {
    const int n = visible(a, t, i), c = h / (a.heads / a.kv_heads);
    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    float* const out = a.out + int64_t(t.q0 + i) * a.ld_out + int64_t(h) * a.dim;
    Columns q;
    q.load(a.q + int64_t(t.q0 + i) * a.ld_q + int64_t(h) * a.dim, a.dim);
    // A group's running maximum and sum; a score of NaN or +inf settles the row.
    float m = -INFINITY, sum = 0.0f;
    bool settled = false;
    for (int64_t j0 = 0; j0 < n && !settled; j0 += 4 * U) {
        Columns x[U];
        load_rows(x, k, a.ld_k, j0, n, a.dim);
        float s[U], top = m;
        bool bad = false;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = dot(q, x[u]) * a.scale;
            if (!row_is_there(j0, u, n)) s[u] = -INFINITY;
            bad |= !(s[u] < INFINITY);
            top = fmaxf(top, s[u]);
        }
        settled = __any(bad);
        const float shift = top == -INFINITY ? 0.0f : top;
        sum *= expf(m - shift);  // -inf - 0 where there was nothing yet
#pragma unroll
        for (int u = 0; u < U; ++u) sum += expf(s[u] - shift);
        m = top;
    }
    float top = fmaxf(m, __shfl_xor(m, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    sum *= expf(m - (top == -INFINITY ? 0.0f : top));
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if ((threadIdx.x & 63) == 0)
        a.lse[int64_t(t.q0 + i) * a.heads + h] = settled            ? NAN
                                                 : top == -INFINITY ? -INFINITY
                                                                    : top + logf(sum);
    if (settled || top == -INFINITY) {  // of scores of -inf alone: 0 / 0
        Columns::fill(out, a.dim, n == 0 ? 0.0f : NAN);
        return;
    }
    Columns o;
    o.clear();
    for (int64_t j0 = 0; j0 < n; j0 += 4 * U) {
        Columns x[U], y[U];
        load_rows(x, k, a.ld_k, j0, n, a.dim);
        load_rows(y, v, a.ld_v, j0, n, a.dim);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // Divided here: the sums stay in range with v's values.
            const float p = expf(dot(q, x[u]) * a.scale - top) / sum;
            if (row_is_there(j0, u, n)) o.add(p, y[u]);
        }
    }
    o.store(out, a.dim, 1.0f);
}

// The share of keys [begin, end).
__device__ void dq_row(const Packed& a, const Tile& t, int h, int i, float delta, int begin,
                       int end, float* dq) {
    constexpr int U = 4;
    const int n = min(visible(a, t, i), end), c = h / (a.heads / a.kv_heads);
    const int64_t row = t.q0 + i;
    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const float lse = a.lse[row * a.heads + h];
    if (begin < n && (lse != lse || delta != delta)) {  // every ds is
        Columns::fill(dq, a.dim, NAN);
        return;
    }
    Columns q, g, sum;
    q.load(a.q + row * a.ld_q + int64_t(h) * a.dim, a.dim);
    g.load(a.grad + row * a.ld_grad + int64_t(h) * a.dim, a.dim);
    sum.clear();
    for (int64_t j0 = begin; j0 < n; j0 += 4 * U) {
        Columns x[U], y[U];
        load_rows(x, k, a.ld_k, j0, n, a.dim);
        load_rows(y, v, a.ld_v, j0, n, a.dim);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float ds = expf(dot(q, x[u]) * a.scale - lse) * (dot(g, y[u]) - delta);
            if (row_is_there(j0, u, n)) sum.add(ds, x[u]);
        }
    }
    sum.store(dq, a.dim, a.scale);
}

// Query head h's share of queries [begin, end) in dk (KEYS) or dv of key j.
template <bool KEYS>
__device__ void dkv_row(const Packed& a, const Tile& t, int h, int j, int begin, int end,
                        float* to) {
    constexpr int U = 4;
    const int c = h / (a.heads / a.kv_heads), lane = int(threadIdx.x) & 63;
    const int64_t row = t.k0 + j;
    // The first query that sees key j.
    int64_t start = a.causal ? int64_t(j) - t.nk + t.nq : 0;
    start = start < begin ? begin : start;
    const float* lse = a.lse + int64_t(t.q0) * a.heads + h;
    const float* delta = a.delta + int64_t(t.q0) * a.heads + h;
    bool settled = false;  // a query whose every p, or ds, is NaN
    for (int64_t i0 = start; i0 < end && !settled; i0 += 64) {
        const int64_t i = min(i0 + lane, int64_t(end) - 1) * a.heads;
        settled = __any(lse[i] != lse[i] || (KEYS && delta[i] != delta[i]));
    }
    if (settled) {
        Columns::fill(to, a.dim, NAN);
        return;
    }
    const float* q = a.q + int64_t(t.q0) * a.ld_q + int64_t(h) * a.dim;
    const float* g = a.grad + int64_t(t.q0) * a.ld_grad + int64_t(h) * a.dim;
    Columns k, v, sum;
    k.load(a.k + row * a.ld_k + int64_t(c) * a.dim, a.dim);
    if (KEYS) v.load(a.v + row * a.ld_v + int64_t(c) * a.dim, a.dim);
    sum.clear();
    for (int64_t i0 = start; i0 < end; i0 += 4 * U) {
        Columns x[U], y[U];
        float z[U], d[U];
        load_rows(x, q, a.ld_q, i0, end, a.dim);
        load_rows(y, g, a.ld_grad, i0, end, a.dim);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = min(i0 + 4 * u + lane / kRowLanes, int64_t(end) - 1) * a.heads;
            z[u] = lse[i];
            d[u] = KEYS ? delta[i] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float w = expf(dot(k, x[u]) * a.scale - z[u]);
            if (KEYS) w *= dot(v, y[u]) - d[u];
            if (row_is_there(i0, u, end)) sum.add(w, KEYS ? x[u] : y[u]);
        }
    }
    sum.store(to, a.dim, KEYS ? a.scale : 1.0f);
}

// ------------------------------------------------------------------- kernels
// Block = slot * heads + head, the heads of one key head 8 (or any multiple of the key heads)
// apart: with the dispatcher's round robin over the eight XCDs they meet their keys in one L2.

__device__ __forceinline__ int head_of(const Packed& a, int x) {
    return x % a.kv_heads * (a.heads / a.kv_heads) + x / a.kv_heads;
}

// log of a sum of terms relative to 2^shift; ln 2 in two parts.
__device__ __forceinline__ float lse_of(float shift, float sum) {
    return __builtin_fmaf(shift, 0.693147182464599609375f,
                          __builtin_fmaf(shift, -1.904654323148236017e-9f, logf(sum)));
}

__device__ __forceinline__ int64_t piece_of(const Packed& a, int64_t row, int h, int piece) {
    return (row * a.heads + h) * a.pieces + piece;
}

// A wave's 32 queries stay in registers; tiles of BN keys and their values pass through LDS with
// the running maximum, sum and weighted values beside them. For long sequences the products bound
// it (16384 tokens, 8 heads of 128 values, causal: 2.6 to 2.8 ms, 195 to 210 TFLOP/s of 201 that a
// sixth of a bf16 product of 8192^3 reaches, with 12 to 15 registers spilled); shorter ones spend
// as long on exponents and on splitting the weights (16 of 512, 16 heads of 64: 72 to 85 us, the
// matrix units busy 40 % of it).
template <int DP, int BN, int WAVES, int READS>
__global__ __launch_bounds__(64 * WAVES, 2) void packed_forward(Packed a) {
    constexpr int BUFFERS = WAVES / 4;
    using namespace attention;
    using KeyTile = RowTile<BN, DP, 64 * WAVES, READS>;
    constexpr int kTile = 2 * KeyTile::kBytes;
    // Wide heads leave the third parts of the queries, which one product in six takes, in LDS: all
    // of them in registers spill.
    constexpr bool kPark = DP > 64;
    constexpr int kParked = kPark ? WAVES * (DP / 16) * 1024 : 0;
    __shared__ __attribute__((aligned(16))) char lds[BUFFERS * kTile + kParked];
    const int h = head_of(a, int(blockIdx.x % a.heads));
    const int slot = int(blockIdx.x / a.heads), piece = slot % a.pieces;
    const Tile t = block_tile(a, false, slot / a.pieces, 32 * WAVES);
    if (t.rows == 0) return;
    const int c = h / (a.heads / a.kv_heads);
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int lane = int(threadIdx.x) & 63;
    const int mine = 32 * wave + (lane & 31);  // the lane's query, of the tile
    const int i = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int limit = visible(a, t, i);
    const int last = 32 * wave + 31 < t.rows ? 32 * wave + 31 : t.rows - 1;
    // The block's keys.
    int begin = 0, end = visible(a, t, t.first + t.rows - 1);
    take_piece(piece, a.pieces, begin, end);
    if (piece > 0 && begin == end) {
        if (mine < t.rows && lane < 32)
            a.piece_stats[piece_of(a, t.q0 + i, h, piece)] = float2{-INFINITY, 0.0f};
        return;
    }
    const int wave_end = 32 * wave < t.rows ? min(visible(a, t, t.first + last), end) : 0;
    const int wave_all = visible(a, t, t.first + 32 * wave);  // keys that all its queries see

    // exp(scale s - m) as 2^(c2 s - m2); a negative scale's sign goes into q, and so does a scale
    // of 0, with which a masked score's -inf would be NaN.
    const float c2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896340736f;
    bf16x8 q[DP / 16][3];
    own_row<DP, READS>(a.q + int64_t(t.q0 + i) * a.ld_q + int64_t(h) * a.dim, a.dim,
                       a.scale < 0.0f ? -1.0f : (a.scale > 0.0f ? 1.0f : a.scale), q);
    char* const parked = lds + BUFFERS * kTile + (wave * (DP / 16) * 64 + lane) * 16;
    if constexpr (kPark) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
            *reinterpret_cast<bf16x8*>(parked + 1024 * ks) = q[ks][2];
    }
    floatx16 o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] = zeros();
    float top = -INFINITY, shift = 0.0f, sum = 0.0f;

    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const int ld_k = int(a.ld_k), ld_v = int(a.ld_v);
    KeyTile kt(ld_k, a.dim), vt(ld_v, a.dim);
    // The tile of keys from j on: into registers, and from there into its half of the LDS.
    const auto load = [&](int j) {
        if (j >= end) return;
        kt.load(k + int64_t(j) * ld_k, ld_k, t.nk - j, a.dim);
        vt.load(v + int64_t(j) * ld_v, ld_v, t.nk - j, a.dim);
    };
    const auto stage = [&](int j) {
        if (j >= end) return;
        char* const at = lds + j / BN % BUFFERS * kTile;
        kt.store(at, t.nk - j, a.dim);
        vt.store(at + KeyTile::kBytes, t.nk - j, a.dim);
    };
    load(begin);
    stage(begin);
    load(begin + BN);
    __syncthreads();
    for (int j0 = begin; j0 < end; j0 += BN) {
        // One wave of a SIMD stages the next tile before its products, the other one after them:
        // one's conversions run beside the other's matrix instructions.
        const char* const lds_k = lds + j0 / BN % BUFFERS * kTile;
        const char* const lds_v = lds_k + KeyTile::kBytes;
        if (BUFFERS == 2 && wave < WAVES / 2) {
            stage(j0 + BN);
            load(j0 + 2 * BN);
        }
        if (j0 < wave_end) {
            floatx16 s[BN / 32];
            scores<KeyTile>(s, lds_k, q, [&](int ks) {
                if (kPark) q[ks][2] = *reinterpret_cast<const bf16x8*>(parked + 1024 * ks);
            });
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
            const float next = m == -INFINITY ? 0.0f : m * c2;
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
            // The tile's sum apart from the running one, which is rounded to nearest once a tile.
            weighted<KeyTile, DP / 32, BN / 16>(
                lds_v, 0, DP / 32, p, [&](int db, const floatx16& x) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[db][r] = __builtin_fmaf(o[db][r], keep, x[r]);
                });
        }
        if (BUFFERS == 1) __syncthreads();
        if (BUFFERS == 1 || wave >= WAVES / 2) {
            stage(j0 + BN);
            load(j0 + 2 * BN);
        }
        __syncthreads();
    }

    sum += __shfl_xor(sum, 32);
    if (a.pieces > 1) {
        const int64_t at = piece_of(a, t.q0 + i, h, piece);
        if (mine < t.rows) {
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
                store_own<READS>(a.piece_out + at * a.dim, a.dim, db, o[db]);
            if (lane < 32)
                a.piece_stats[at] = float2{top == -INFINITY ? -INFINITY : shift, sum};
        }
        return;
    }
    // Rows that saw something and have no finite result are formed again by the formula: a NaN or
    // an infinity where it counts, or one in a place of theirs that they do not see (0 times it).
    // A row that saw nothing is 0, whatever the keys of its wave's other rows left in its sums.
    const float inv = 1.0f / sum;
    bool fine = sum > 0.0f && sum < INFINITY;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[db][r] = limit > 0 ? o[db][r] * inv : 0.0f;
            fine = fine && fabsf(o[db][r]) < INFINITY;
        }
    fine = fine || limit == 0;
    const uint64_t votes = __ballot(!fine && mine < t.rows);
    const uint32_t again = uint32_t(votes) | uint32_t(votes >> 32);
    if (mine < t.rows && !(again >> (lane & 31) & 1)) {
        float* out = a.out + int64_t(t.q0 + i) * a.ld_out + int64_t(h) * a.dim;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) store_own<READS>(out, a.dim, db, o[db]);
        if (lane < 32)
            a.lse[int64_t(t.q0 + i) * a.heads + h] =
                limit == 0 ? -INFINITY
                           : lse_of(shift, sum);
    }
    for (uint32_t rows = again; rows != 0; rows &= rows - 1)
        forward_row<4>(a, t, h, t.first + 32 * wave + __builtin_ctz(rows));
}

// The rows' pieces. One wave a row and head, two values a lane: latency (66912 rows of 96 values in
// two pieces 27 us, 78 MB).
__global__ __launch_bounds__(kThreads) void packed_forward_join(Packed a) {
    const int lane = int(threadIdx.x) & 63;
    const int n_row = __builtin_amdgcn_readfirstlane(
        int(blockIdx.x) * (kThreads / 64) + int(threadIdx.x) / 64);
    const int row = n_row / a.heads, h = n_row - row * a.heads;
    const int64_t at = n_row;
    if (row < offset_at(a.cu_q, 0, a.total_q) ||
        row >= offset_at(a.cu_q, a.sequences, a.total_q))
        return;
    // A lane has a piece's statistics, and then two values of every piece, four pieces asked for at
    // a time; those that saw nothing left none.
    const float2 x = lane < a.pieces ? a.piece_stats[at * a.pieces + lane]
                                     : float2{-INFINITY, 0.0f};
    const float top = wave_max(x.x);
    const bool saw = x.x != -INFINITY || x.y != 0.0f;
    const float mine = saw ? __builtin_amdgcn_exp2f(x.x - top) : 0.0f;
    const float sum = wave_sum(saw ? x.y * mine : 0.0f);
    const uint64_t seen = __ballot(saw);
    const float* const values = a.piece_out + at * a.pieces * a.dim;
    float o[2] = {0.0f, 0.0f};
    for (int n0 = 0; n0 < a.pieces; n0 += 4) {
        float y[4][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int n = n0 + u < a.pieces ? n0 + u : 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = lane + 64 * e;
                y[u][e] = values[int64_t(n) * a.dim + (d < a.dim ? d : 0)];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int n = n0 + u;
            const float keep = __shfl(mine, n & 63);
            if (n >= a.pieces || !(seen >> n & 1)) continue;
#pragma unroll
            for (int e = 0; e < 2; ++e) o[e] = __builtin_fmaf(y[u][e], keep, o[e]);
        }
    }
    const float inv = 1.0f / sum;
    bool fine = sum > 0.0f && sum < INFINITY;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        o[e] *= inv;
        fine = fine && fabsf(o[e]) < INFINITY;
    }
    if (__all(fine)) {
        float* const out = a.out + row * a.ld_out + int64_t(h) * a.dim;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (lane + 64 * e < a.dim) out[lane + 64 * e] = o[e];
        if (lane == 0) a.lse[at] = lse_of(top, sum);
        return;
    }
    // A row that saw nothing, or not finite: by the formula, in its sequence, the last that begins
    // at or before it.
    int lo = 0, n = a.sequences;
    while (n > 1) {
        const int mid = lo + n / 2;
        const bool in = offset_at(a.cu_q, mid, a.total_q) <= row;
        lo = in ? mid : lo;
        n = in ? n - n / 2 : n / 2;
    }
    const Tile t = tile_of(a, false, lo, 0, kRows);
    // One row ahead: more registers would leave fewer waves for the rows that are fine.
    if (row - t.q0 < t.nq) forward_row<1>(a, t, h, row - t.q0);
}

// The backward forms s, and so p_ij, again from the inputs, and dp likewise, for the pairs of a
// wave's own rows and a block of 32 streamed ones, then the block's share of the gradients.

// Where a piece's share of dq goes.
__device__ __forceinline__ float* row_dq(const Packed& a, int64_t row, int h, int piece) {
    return a.part_q != nullptr
               ? a.part_q + ((row * a.heads + h) * a.pieces_q + piece) * a.dim
               : a.dq + row * a.ld_dq + int64_t(h) * a.dim;
}

// dq_i = scale sum_j ds_ij k_j of heads of up to 64 values, with delta on the way (left in the
// workspace for the keys' kernel): a wave has room for q and g both, and needs no partner (16 of
// 512 tokens, 16 heads of 64, causal: 98 to 115 us, bound as the forward).
template <int DP, int BN, int READS>
__global__ __launch_bounds__(kThreads, 2) void packed_backward_q(Packed a) {
    using namespace attention;
    using KeyTile = RowTile<BN, DP, kThreads, READS>;
    __shared__ __attribute__((aligned(16))) char lds[2 * KeyTile::kBytes];
    char* const lds_v = lds + KeyTile::kBytes;
    const int h = head_of(a, int(blockIdx.x % a.heads));
    const int slot = int(blockIdx.x / a.heads), piece = slot % a.pieces_q;
    const Tile t = block_tile(a, false, slot / a.pieces_q, kRows);
    if (t.rows == 0) return;
    const int c = h / (a.heads / a.kv_heads);
    const int wave = int(threadIdx.x) / 64, lane = int(threadIdx.x) & 63;
    const int mine = 32 * wave + (lane & 31);  // the lane's query, of the tile
    const int i = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int64_t row = t.q0 + i;
    const int limit = visible(a, t, i);
    const int last = 32 * wave + 31 < t.rows ? 32 * wave + 31 : t.rows - 1;
    int begin = 0, end = visible(a, t, t.first + t.rows - 1);
    take_piece(piece, a.pieces_q, begin, end);
    const int wave_end = 32 * wave < t.rows ? min(visible(a, t, t.first + last), end) : 0;
    const int wave_all = visible(a, t, t.first + 32 * wave);  // keys that all its queries see

    const float* gr = a.grad + row * a.ld_grad + int64_t(h) * a.dim;
    const float delta = own_dot<DP, READS>(gr, a.out + row * a.ld_out + int64_t(h) * a.dim, a.dim);
    if (piece == 0 && lane < 32 && mine < t.rows) a.delta[row * a.heads + h] = delta;
    if (a.dq == nullptr) return;
    const float c2 = a.scale * 1.44269504088896340736f;
    const float shift = limit > 0 ? a.lse[row * a.heads + h] * 1.44269504088896340736f : 0.0f;
    bf16x8 q[DP / 16][3], g[DP / 16][3];
    own_row<DP, READS>(a.q + row * a.ld_q + int64_t(h) * a.dim, a.dim, 1.0f, q);
    own_row<DP, READS>(gr, a.dim, 1.0f, g);
    floatx16 dq[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) dq[db] = zeros();

    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const int ld_k = int(a.ld_k), ld_v = int(a.ld_v);
    KeyTile kt(ld_k, a.dim), vt(ld_v, a.dim);
    if (begin < end) {
        kt.load(k + int64_t(begin) * ld_k, ld_k, t.nk - begin, a.dim);
        vt.load(v + int64_t(begin) * ld_v, ld_v, t.nk - begin, a.dim);
    }
    for (int j0 = begin; j0 < end; j0 += BN) {
        __syncthreads();
        kt.store(lds, t.nk - j0, a.dim);
        vt.store(lds_v, t.nk - j0, a.dim);
        const int j1 = j0 + BN;
        if (j1 < end) {
            kt.load(k + int64_t(j1) * ld_k, ld_k, t.nk - j1, a.dim);
            vt.load(v + int64_t(j1) * ld_v, ld_v, t.nk - j1, a.dim);
        }
        __syncthreads();
        if (j0 >= wave_end) continue;
        const bool edge = j1 > wave_all;
        bf16x8 w[BN / 16][3];
#pragma unroll
        for (int b = 0; b < BN / 32; ++b) {
            floatx16 s[1], dp[1];
            scores<KeyTile>(s, lds, q, [](int) {});
            scores<KeyTile>(dp, lds_v, g, [](int) {});
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                ds[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], c2, -shift)) *
                        (dp[0][r] - delta);
                if (edge && j0 + 32 * b + row_of(r) >= limit) ds[r] = 0.0f;
            }
            split8(ds, w[2 * b]);
            split8(ds + 8, w[2 * b + 1]);
        }
        weighted<KeyTile, DP / 32, BN / 16>(lds, 0, DP / 32, w, [&](int db, const floatx16& x) {
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[db][r] += x[r];
        });
    }
    bool fine = true;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dq[db][r] = limit > 0 ? dq[db][r] * a.scale : 0.0f;
            fine = fine && fabsf(dq[db][r]) < INFINITY;
        }
    const uint64_t votes = __ballot(!fine && mine < t.rows);
    const uint32_t again = uint32_t(votes) | uint32_t(votes >> 32);
    if (mine < t.rows && !(again >> (lane & 31) & 1))
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
            store_own<READS>(row_dq(a, row, h, piece), a.dim, db, dq[db]);
    for (uint32_t rows = again; rows != 0; rows &= rows - 1) {
        const int r = __builtin_ctz(rows);
        dq_row(a, t, h, t.first + 32 * wave + r, __shfl(delta, r), begin, end,
               row_dq(a, t.q0 + t.first + 32 * wave + r, h, piece));
    }
}

// Its larger kernels' blocks own 128 rows, as four groups of 32 and two waves a group: both form
// scores for the same pairs, one wave s and the other dp = g . v, exchange them through LDS, and
// each accumulates its share of the gradients. So a wave holds one own row and half of the results
// a lane, which leaves room for two waves a SIMD at every head size: a lone wave issues a vector
// instruction every eighth cycle only. A step is two phases with a barrier after each: the scores,
// from the streamed rows, then the gradients, from the same rows read transposed.
constexpr int kBackThreads = 512;

// Gives the two waves of a group the rows (a bit each) that either found without a finite result.
__device__ __forceinline__ uint32_t shared_rows(uint32_t* votes, bool bad) {
    const uint64_t b = __ballot(bad);
    const int wave = int(threadIdx.x) / 64;
    if ((threadIdx.x & 63) == 0) votes[wave] = uint32_t(b) | uint32_t(b >> 32);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(votes[wave & 3] | votes[(wave & 3) + 4]);
}

// dq and delta of wider heads. Wave role 0 forms s and p, role 1 dp - delta; both then have ds, and
// half of dq's values each (5576 tokens in 11 sequences, 12 heads of 96 over 4: 189 to 238 us,
// the matrix units busy 40 %, by turns as in the keys' kernel).
template <int DP, int BN, int READS>
__global__ __launch_bounds__(kBackThreads, 2) void packed_backward_q_pair(Packed a) {
    using namespace attention;
    using KeyTile = RowTile<BN, DP, kBackThreads, READS>;
    constexpr int NB = BN / 32, NU = BN / 16, kBlocks = DP / 32, kHalf = (kBlocks + 1) / 2;
    constexpr int kSwap = 4 * NB * 4096;  // one role's scores
    __shared__ __attribute__((aligned(16))) char
        lds[4 * KeyTile::kBytes + 2 * kSwap];  // two tiles of both, by turns
    char* const lds_x = lds + 4 * KeyTile::kBytes;
    const int h = head_of(a, int(blockIdx.x % a.heads));
    const int slot = int(blockIdx.x / a.heads), piece = slot % a.pieces_q;
    const Tile t = block_tile(a, false, slot / a.pieces_q, kRows);
    if (t.rows == 0) return;
    const int c = h / (a.heads / a.kv_heads);
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int role = wave / 4, w0 = 32 * (wave & 3), lane = int(threadIdx.x) & 63;
    const int mine = w0 + (lane & 31);  // the lane's query, of the tile
    const int i = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int64_t row = t.q0 + i;
    const int limit = visible(a, t, i);
    const int last = w0 + 31 < t.rows ? w0 + 31 : t.rows - 1;
    int begin = 0, end = visible(a, t, t.first + t.rows - 1);
    take_piece(piece, a.pieces_q, begin, end);
    const int wave_end = w0 < t.rows ? min(visible(a, t, t.first + last), end) : 0;
    const int wave_all = visible(a, t, t.first + w0);  // keys that all its queries see

    const float* qr = a.q + row * a.ld_q + int64_t(h) * a.dim;
    const float* gr = a.grad + row * a.ld_grad + int64_t(h) * a.dim;
    const float delta = own_dot<DP, READS>(gr, a.out + row * a.ld_out + int64_t(h) * a.dim, a.dim);
    if (piece == 0 && wave < 4 && lane < 32 && mine < t.rows) a.delta[row * a.heads + h] = delta;
    if (a.dq == nullptr) return;
    const float c2 = a.scale * 1.44269504088896340736f;
    const float shift = limit > 0 ? a.lse[row * a.heads + h] * 1.44269504088896340736f : 0.0f;
    bf16x8 own[DP / 16][3];
    own_row<DP, READS>(role == 0 ? qr : gr, a.dim, 1.0f, own);
    floatx16 dq[kHalf];
#pragma unroll
    for (int d = 0; d < kHalf; ++d) dq[d] = zeros();

    const float* k = a.k + int64_t(t.k0) * a.ld_k + int64_t(c) * a.dim;
    const float* v = a.v + int64_t(t.k0) * a.ld_v + int64_t(c) * a.dim;
    const int ld_k = int(a.ld_k), ld_v = int(a.ld_v);
    KeyTile kt(ld_k, a.dim), vt(ld_v, a.dim);
    const auto load_rows = [&](int j) {
        if (j >= end) return;
        kt.load(k + int64_t(j) * ld_k, ld_k, t.nk - j, a.dim);
        vt.load(v + int64_t(j) * ld_v, ld_v, t.nk - j, a.dim);
    };
    const auto stage_rows = [&](int j) {
        if (j >= end) return;
        char* const at = lds + (j / BN & 1) * 2 * KeyTile::kBytes;
        kt.store(at, t.nk - j, a.dim);
        vt.store(at + KeyTile::kBytes, t.nk - j, a.dim);
    };
    char* const give = lds_x + role * kSwap + ((wave & 3) * NB * 256 + lane) * 16;
    const char* const take = lds_x + (1 - role) * kSwap + ((wave & 3) * NB * 256 + lane) * 16;
    load_rows(begin);
    stage_rows(begin);
    load_rows(begin + BN);
    __syncthreads();
    for (int j0 = begin; j0 < end; j0 += BN) {
        const bool active = j0 < wave_end;
        const char* const tile = lds + (j0 / BN & 1) * 2 * KeyTile::kBytes;
        if (role == 1) {  // the next tile: one wave of a SIMD before its products, the other after
            stage_rows(j0 + BN);
            load_rows(j0 + 2 * BN);
        }
        floatx16 s[NB];
        if (active) {
            scores<KeyTile>(s, tile + role * KeyTile::kBytes, own, [](int) {});
            if (role == 0) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], c2, -shift));
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[b][r] -= delta;
            }
            if (j0 + BN > wave_all) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[b][r] = j0 + 32 * b + row_of(r) >= limit ? 0.0f : s[b][r];
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<floatx4u*>(give + (4 * b + r / 4) * 1024) =
                        floatx4u{s[b][r], s[b][r + 1], s[b][r + 2], s[b][r + 3]};
        }
        __syncthreads();
        if (active) {
            bf16x8 w[NU][3];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float ds[16];
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const floatx4u x =
                        *reinterpret_cast<const floatx4u*>(take + (4 * b + r / 4) * 1024);
#pragma unroll
                    for (int e = 0; e < 4; ++e) ds[r + e] = s[b][r + e] * x[e];
                }
                split8(ds, w[2 * b]);
                split8(ds + 8, w[2 * b + 1]);
            }
            const int mid = role * kHalf;  // the wave's first block of values
            weighted<KeyTile, kHalf, NU>(tile, mid, min(kHalf, kBlocks - mid), w,
                                         [&](int d, const floatx16& x) {
#pragma unroll
                                             for (int r = 0; r < 16; ++r) dq[d][r] += x[r];
                                         });
        }
        if (role == 0) {
            stage_rows(j0 + BN);
            load_rows(j0 + 2 * BN);
        }
        __syncthreads();
    }
    bool fine = true;
#pragma unroll
    for (int d = 0; d < kHalf; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dq[d][r] = limit > 0 ? dq[d][r] * a.scale : 0.0f;
            fine = fine && fabsf(dq[d][r]) < INFINITY;
        }
    const uint32_t again = shared_rows(reinterpret_cast<uint32_t*>(lds), !fine && mine < t.rows);
    if (mine < t.rows && !(again >> (lane & 31) & 1)) {
        float* out = row_dq(a, row, h, piece);
#pragma unroll
        for (int d = 0; d < kHalf; ++d)
            if (role * kHalf + d < kBlocks)
                store_own<READS>(out, a.dim, role * kHalf + d, dq[d]);
    }
    if (role == 0)
        for (uint32_t rows = again; rows != 0; rows &= rows - 1) {
            const int r = __builtin_ctz(rows);
            dq_row(a, t, h, t.first + w0 + r, __shfl(delta, r), begin, end,
                   row_dq(a, t.q0 + t.first + w0 + r, h, piece));
        }
}

// dv_j = sum_i p_ij g_i by the waves of role 0, from s and p, and dk_j = scale sum_i ds_ij q_i by
// those of role 1, from dp and the other's p: 16 of 512 tokens, 16 heads of 64, 143 to 173 us; 5576
// tokens, 12 heads of 96, 228 to 288. The matrix units are busy 37 and 51 %: both waves of a SIMD
// are in the phase of the scores, mostly vector work, or both in that of the gradients. Heads of
// 128 values spill 37 to 40 registers, of 64 6 to 9.
template <int DP, int BN, int READS>
__global__ __launch_bounds__(kBackThreads, 2) void packed_backward_kv(Packed a) {
    using namespace attention;
    using QueryTile = RowTile<BN, DP, kBackThreads, READS>;
    constexpr int NB = BN / 32, NU = BN / 16, kBlocks = DP / 32;
    constexpr int kSwap = 4 * NB * 4096;
    __shared__ __attribute__((aligned(16))) char lds[4 * QueryTile::kBytes + kSwap];
    __shared__ __attribute__((aligned(16))) float stats[2][2][BN];  // as the tiles, by turns
    char* const lds_x = lds + 4 * QueryTile::kBytes;
    const int h = head_of(a, int(blockIdx.x % a.heads)), c = h / (a.heads / a.kv_heads);
    const int slot = int(blockIdx.x / a.heads), piece = slot % a.pieces_k;
    const Tile t = block_tile(a, true, slot / a.pieces_k, kRows);
    if (t.rows == 0) return;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int role = wave / 4, w0 = 32 * (wave & 3), lane = int(threadIdx.x) & 63;
    const int mine = w0 + (lane & 31);  // the lane's key, of the tile
    const int j = t.first + (mine < t.rows ? mine : t.rows - 1);
    const int64_t row = t.k0 + j;
    // The first query that sees a key; of the block's keys, the wave's, and all of the wave's.
    const auto first_of = [&](int key) {
        const int64_t n = a.causal ? int64_t(key) - t.nk + t.nq : 0;
        return n < 0 ? 0 : int(n);
    };
    const int from = first_of(j);
    int start = first_of(t.first), end = t.nq;  // the block's queries
    take_piece(piece, a.pieces_k, start, end);
    const int wave_start = w0 < t.rows ? first_of(t.first + w0) : t.nq;
    const int wave_all = first_of(t.first + w0 + 31);

    const float c2 = a.scale * 1.44269504088896340736f;
    bf16x8 own[DP / 16][3];
    own_row<DP, READS>(role == 0 ? a.k + row * a.ld_k + int64_t(c) * a.dim
                               : a.v + row * a.ld_v + int64_t(c) * a.dim,
                     a.dim, 1.0f, own);
    floatx16 sum[kBlocks];  // dv or dk
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) sum[d] = zeros();
    const int ld_q = int(a.ld_q), ld_g = int(a.ld_grad);
    QueryTile qt(ld_q, a.dim), gt(ld_g, a.dim);
    float stat = 0.0f;  // a query's lse (threads 0 .. BN - 1) or delta (the next BN)
    // Tile n: the queries from start + n * BN on.
    const int count = (end - start + BN - 1) / BN;
    const auto load_rows = [&](int n) {
        if (n >= count) return;
        const int i0 = start + n * BN, left = end - i0;
        const int64_t at = t.q0 + i0;
        qt.load(a.q + at * a.ld_q + int64_t(h) * a.dim, ld_q, left, a.dim);
        gt.load(a.grad + at * a.ld_grad + int64_t(h) * a.dim, ld_g, left, a.dim);
        if (threadIdx.x < 2 * BN) {
            const int r = int(threadIdx.x) % BN < left ? int(threadIdx.x) % BN : left - 1;
            stat = (threadIdx.x < BN ? a.lse : a.delta)[(at + r) * a.heads + h];
        }
    };
    const auto stage_rows = [&](int n) {
        if (n >= count) return;
        const int left = end - (start + n * BN);
        char* const at = lds + (n & 1) * 2 * QueryTile::kBytes;
        qt.store(at, left, a.dim);
        gt.store(at + QueryTile::kBytes, left, a.dim);
        if (threadIdx.x < BN) stats[n & 1][0][threadIdx.x] = stat * 1.44269504088896340736f;
        else if (threadIdx.x < 2 * BN) stats[n & 1][1][threadIdx.x - BN] = stat;
    };
    char* const swap = lds_x + ((wave & 3) * NB * 256 + lane) * 16;
    const int half = lane / 32;
    load_rows(0);
    stage_rows(0);
    load_rows(1);
    __syncthreads();
    for (int n = 0; n < count; ++n) {
        const int i0 = start + n * BN, left = end - i0;
        const bool active = i0 + BN > wave_start;
        const char* const tile = lds + (n & 1) * 2 * QueryTile::kBytes;
        if (role == 1) {  // the next tile: one wave of a SIMD before its products, the other after
            stage_rows(n + 1);
            load_rows(n + 2);
        }
        floatx16 s[NB];
        if (active) {
            scores<QueryTile>(s, tile + role * QueryTile::kBytes, own, [](int) {});
            const float* const stat_of = stats[n & 1][role] + 4 * half;
            if (role == 0) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const floatx4u y =
                            *reinterpret_cast<const floatx4u*>(stat_of + 32 * b + 2 * r);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[b][r + e] = __builtin_amdgcn_exp2f(
                                __builtin_fmaf(s[b][r + e], c2, -y[e]));
                    }
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const floatx4u y =
                            *reinterpret_cast<const floatx4u*>(stat_of + 32 * b + 2 * r);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[b][r + e] -= y[e];
                    }
            }
            if (i0 < wave_all || left < BN) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int q = 32 * b + row_of(r);
                        s[b][r] = ((i0 + q < from) | (q >= left)) ? 0.0f : s[b][r];
                    }
            }
            if (role == 0) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        *reinterpret_cast<floatx4u*>(swap + (4 * b + r / 4) * 1024) =
                            floatx4u{s[b][r], s[b][r + 1], s[b][r + 2], s[b][r + 3]};
            }
        }
        __syncthreads();
        if (active) {
            if (role != 0) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const floatx4u p =
                            *reinterpret_cast<const floatx4u*>(swap + (4 * b + r / 4) * 1024);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[b][r + e] *= p[e];
                    }
            }
            bf16x8 w[NU][3];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float y[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] = s[b][r];
                split8(y, w[2 * b]);
                split8(y + 8, w[2 * b + 1]);
            }
            // dv from the gradient's rows, dk from the queries'.
            weighted<QueryTile, kBlocks, NU>(tile + (1 - role) * QueryTile::kBytes, 0, kBlocks, w,
                                             [&](int d, const floatx16& x) {
#pragma unroll
                                                 for (int r = 0; r < 16; ++r) sum[d][r] += x[r];
                                             });
        }
        if (role == 0) {
            stage_rows(n + 1);
            load_rows(n + 2);
        }
        __syncthreads();
    }
    const float factor = role == 0 ? 1.0f : a.scale;
    // Without dk there may be no delta either.
    const bool wanted = (role == 0 ? a.dv : a.dk) != nullptr;
    bool fine = true;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            sum[d][r] *= factor;
            fine = fine && fabsf(sum[d][r]) < INFINITY;
        }
    const uint64_t votes = __ballot(wanted && !fine && mine < t.rows);
    const uint32_t again = uint32_t(votes) | uint32_t(votes >> 32);
    // Where the wave's gradient of key row `at` goes.
    float* const part = role == 0 ? a.part_v : a.part_k;
    float* const whole = role == 0 ? a.dv : a.dk;
    const int64_t ld = role == 0 ? a.ld_dv : a.ld_dk;
    const auto row_to = [&](int64_t at) {
        return part != nullptr ? part + ((at * a.heads + h) * a.pieces_k + piece) * a.dim
                               : whole + at * ld + int64_t(c) * a.dim;
    };
    if (wanted && mine < t.rows && !(again >> (lane & 31) & 1)) {
        float* const out = row_to(row);
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) store_own<READS>(out, a.dim, d, sum[d]);
    }
    for (uint32_t rows = again; rows != 0; rows &= rows - 1) {
        const int key = t.first + w0 + __builtin_ctz(rows);
        float* const out = row_to(t.k0 + key);
        if (role == 0) dkv_row<false>(a, t, h, key, start, end, out);
        else dkv_row<true>(a, t, h, key, start, end, out);
    }
}

// Rows of one gradient, or of dk and dv, from `count` shares of each head's row one after the
// other, in their order: the pieces', and for dk and dv the group's query heads'. Thread = row,
// head, value. HBM (5576 rows, 12 heads of 96 over 4: 13 us for 69 MB).
template <int N>
struct Shares {
    const int32_t* cu;
    int sequences, total;
    int heads, count, dim;
    const float* from[N];
    float* to[N];  // may be null
    int64_t ld[N];
};
template <int N>
__global__ __launch_bounds__(kThreads) void packed_backward_join(Shares<N> x) {
    const int64_t width = int64_t(x.heads) * x.dim;
    const int first = offset_at(x.cu, 0, x.total);
    const int last = offset_at(x.cu, x.sequences, x.total);
    for (int64_t e = first * width + int64_t(blockIdx.x) * kThreads + threadIdx.x; e < last * width;
         e += int64_t(gridDim.x) * kThreads) {
        const int64_t row = e / width;
        const int at = int(e - row * width), c = at / x.dim, d = at - c * x.dim;
        const int64_t from = (row * x.heads + c) * x.count * x.dim + d;
        float y[N] = {};
#pragma unroll 4
        for (int n = 0; n < x.count; ++n)
#pragma unroll
            for (int g = 0; g < N; ++g) y[g] += x.from[g][from + int64_t(n) * x.dim];
#pragma unroll
        for (int g = 0; g < N; ++g)
            if (x.to[g] != nullptr) x.to[g][row * x.ld[g] + at] = y[g];
    }
}

// ---------------------------------------------------------------- host checks

int64_t slots(int64_t total, int64_t sequences, int rows = kRows) {
    return total / rows + sequences;
}

// Rows are taken to be in sequences of the mean length, or, where the longest is known, in as many
// of that length as they make: a long one among short or empty ones then counts as itself.
void share(int64_t total, int64_t sequences, int64_t longest, int64_t& each, int64_t& count) {
    each = sequences == 0 ? 0 : longest > 0 ? std::min(longest, total) : total / sequences;
    count = longest > 0 && each > 0 ? std::min(sequences, ceil_div(total, each)) : sequences;
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
    constexpr int64_t kBlocks = (int64_t(1) << 23) - 1;  // of 512 threads, 2^32 in all at most
    if (d->heads > kBlocks || d->sequences > kBlocks || d->total_q > INT32_MAX ||
        d->total_k > INT32_MAX ||
        slots(d->total_q > d->total_k ? d->total_q : d->total_k, d->sequences) * d->heads > kBlocks)
        return fail(EHIP_EINVAL, "%s: %lld x %lld rows of %lld heads are too many", name,
                    (long long)d->total_q, (long long)d->total_k, (long long)d->heads);
    if (d->longest_q < 0 || d->longest_k < 0)
        return fail(EHIP_EINVAL, "%s: longest sequences of %lld and %lld rows", name,
                    (long long)d->longest_q, (long long)d->longest_k);
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
    share(d->total_q, d->sequences, d->longest_q, a.each_q, a.count_q);
    share(d->total_k, d->sequences, d->longest_k, a.each_k, a.count_k);
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
    // Under a causal mask by work (16 sequences of 512: forward 82 -> 70 us, dq 114 -> 97), for as
    // many sequences as a wave has lanes: find_tile_by_work has one in each.
    a.by_work = a.causal && a.sequences <= 64;
    a.out = d->out;
    a.ld_out = d->ld_out;
    a.lse = d->lse;
    return EHIP_OK;
}

template <int DP, int BN, int WAVES, int READS>
int launch_forward(const Packed& a, hipStream_t s) {
    const unsigned blocks =
        unsigned(slots(a.total_q, a.sequences, 32 * WAVES) * a.heads * a.pieces);
    EHIP_LAUNCH("attention_packed", (packed_forward<DP, BN, WAVES, READS>), dim3(blocks),
                dim3(64 * WAVES), 0, s, a);
    if (a.pieces > 1)
        EHIP_LAUNCH("attention_packed_join", packed_forward_join,
                    dim3(unsigned(ceil_div(int64_t(a.total_q) * a.heads, kThreads / 64))),
                    dim3(kThreads), 0, s, a);
    return EHIP_OK;
}

// 256 queries a block convert their keys once and read them by turns of two tiles; 128 leave
// less between the last block and the others. Without the causal mask all blocks of a sequence
// are alike, and 256 it is once they fill the card (us, 128 : 256 queries, heads of 64 values:
// one of 4096, 16 heads, 341 : 326, with 8 heads 216 : 275). With it, long sequences that fill
// the card twice over (4 of 2048, 16 heads, 207 : 200; 24 of 64 to 1291 147 : 169; one of 8192,
// 8 heads, 490 : 566). Heads over 96 values spill with 128, and take them for short causal ones
// alone (64 of 128 87 : 103; one of 4096 593 : 509; without the mask 64 of 128 136 : 82).
bool narrow_blocks(const Packed& a) {
    const int64_t blocks = a.total_q / 256 * a.heads;
    return a.dim > 96 ? a.causal && a.each_q < 256
           : a.causal ? a.each_q < 2048 || blocks < 512
                      : blocks < 256;
}

// Pieces for `want` blocks in all where the tiles make `blocks` of them and pass `rows` rows, of
// kLeastPiece rows or more; and no more than make kMostBlocks of those launched, most of which have
// no tile where few of the sequences are long (8 heads of 128, 128 queries behind 16384 keys beside
// 43 of one each, us whole 2052, for 4096 209, 8192 126, 16384 125; 500 behind 4000 beside 200 of
// one 521, 369, 208, 249).
constexpr int64_t kMostBlocks = 8192;
int pieces_for(int64_t want, int64_t blocks, int64_t launched, int64_t rows) {
    if (rows < 384) return 1;
    const int64_t most = std::min({rows / kLeastPiece, int64_t(32), kMostBlocks / launched});
    return int(std::max<int64_t>(1, std::min((want + blocks / 2) / blocks, most)));
}

// Pieces of a tile's keys, where the tiles alone leave CUs without work: for 512 blocks in all, or
// 1024 of those of 128 queries where a causal mask leaves them uneven and the tiles make 256 (us,
// heads of 64: one of 2048, 8 heads, whole 107, for 512 53, for 1024 63; one of 4096 212, 145, 125;
// heads of 128: 128 queries behind 16384 keys 2049, 105; one of 4096, 8 heads, 525, 216, 271), of
// 128 keys or more (8 of 64 to 946, heads of 128, 127 whole and with 256 or more, 82 with 128).
// Sequences that are shorter do not make up for the second launch (4 of 256, 4 heads of 64, 18.6
// whole, 21.2 in two).
int pieces_of(const Packed& a) {
    const bool narrow = narrow_blocks(a);
    const int rows = narrow ? 128 : 256;
    const int64_t blocks = slots(a.total_q, a.count_k, rows) * a.heads;
    return pieces_for(narrow && a.causal && blocks >= 256 ? 1024 : 512, blocks,
                      slots(a.total_q, a.sequences, rows) * a.heads, a.each_k);
}

size_t piece_bytes(const Packed& a) {
    const int pieces = pieces_of(a);
    return pieces == 1 ? 0
                       : size_t(a.total_q) * size_t(a.heads) * size_t(pieces) *
                             (sizeof(float2) + size_t(a.dim) * sizeof(float));
}

template <int DP, int BN, int READS>
int forward_of(const Packed& a, hipStream_t s) {
    return narrow_blocks(a) ? launch_forward<DP, BN, 4, READS>(a, s)
                            : launch_forward<DP, BN, 8, READS>(a, s);
}

// The backward's pieces likewise, of the keys for dq and of the queries for dk and dv: for 512
// blocks under a causal mask, else for 256, one a CU (us, whole : for 256 : for 512, 8 heads of 64
// values: one sequence of 4096 584 : 572 : 416; 128 queries behind 4096 keys 327 : 78 : 76; without
// the mask one of 2048 311 : 193 : 201, 8 of 512 117 : 113 : 136; heads of 96, 8 of 512 143 : 139 :
// 208).
int backward_pieces(const Packed& a, int64_t rows, int64_t each, int64_t count) {
    return pieces_for(a.causal ? 512 : 256, slots(rows, count) * a.heads,
                      slots(rows, a.sequences) * a.heads, each);
}

// Shares of dq, and of each of dk and dv. dk and dv of grouped heads are formed head by head, for
// as many blocks as the queries have, and summed afterwards (12 heads over 4, 5576 rows of 96: one
// block a group took 2.8 times as long).
struct BackwardSpace {
    int pieces_q, pieces_k;
    size_t delta, part_q, part_k;  // bytes
};
BackwardSpace space_of(const Packed& a) {
    BackwardSpace x;
    x.pieces_q = backward_pieces(a, a.total_q, a.each_k, a.count_k);
    x.pieces_k = backward_pieces(a, a.total_k, a.each_q, a.count_q);
    const auto aligned = [](size_t n) { return (n + 15) & ~size_t(15); };
    const size_t row = size_t(a.heads) * sizeof(float), dim = size_t(a.dim);
    x.delta = aligned(size_t(a.total_q) * row);
    x.part_q = x.pieces_q > 1 ? aligned(size_t(a.total_q) * row * dim * size_t(x.pieces_q)) : 0;
    x.part_k = x.pieces_k > 1 || a.heads != a.kv_heads
                   ? aligned(size_t(a.total_k) * row * dim * size_t(x.pieces_k))
                   : 0;
    return x;
}
size_t bytes_of(const BackwardSpace& x) { return x.delta + x.part_q + 2 * x.part_k; }

template <int N>
int join_shares(const Shares<N>& x, hipStream_t s) {
    const int64_t n = int64_t(x.total) * x.heads * x.dim;
    EHIP_LAUNCH("attention_packed_backward_join", packed_backward_join<N>,
                dim3(unsigned(std::min<int64_t>(ceil_div(n, kThreads), 1 << 16))), dim3(kThreads),
                0, s, x);
    return EHIP_OK;
}

template <int DP, int BN, int READS>
int launch_backward(const Packed& a, hipStream_t s) {
    if (a.total_q > 0 && (a.dq != nullptr || a.dk != nullptr)) {
        const unsigned blocks = unsigned(slots(a.total_q, a.sequences) * a.heads * a.pieces_q);
        if constexpr (DP <= 64)
            EHIP_LAUNCH("attention_packed_backward_q", (packed_backward_q<DP, 32, READS>),
                        dim3(blocks), dim3(kThreads), 0, s, a);
        else
            EHIP_LAUNCH("attention_packed_backward_q", (packed_backward_q_pair<DP, BN, READS>),
                        dim3(blocks), dim3(kBackThreads), 0, s, a);
        if (a.part_q != nullptr) {
            const Shares<1> x{a.cu_q, a.sequences, a.total_q, a.heads,  a.pieces_q,
                              a.dim,  {a.part_q},  {a.dq},    {a.ld_dq}};
            if (int rc = join_shares(x, s)) return rc;
        }
    }
    if (a.total_k == 0 || (a.dk == nullptr && a.dv == nullptr)) return EHIP_OK;
    const unsigned blocks = unsigned(slots(a.total_k, a.sequences) * a.heads * a.pieces_k);
    EHIP_LAUNCH("attention_packed_backward_kv", (packed_backward_kv<DP, BN, READS>), dim3(blocks),
                dim3(kBackThreads), 0, s, a);
    if (a.part_k == nullptr) return EHIP_OK;
    const Shares<2> x{a.cu_k,
                      a.sequences,
                      a.total_k,
                      a.kv_heads,
                      a.heads / a.kv_heads * a.pieces_k,
                      a.dim,
                      {a.part_k, a.part_v},
                      {a.dk, a.dv},
                      {a.ld_dk, a.ld_dv}};
    return join_shares(x, s);
}

// A head's values in blocks of 32; wider heads take 32 rows of a tile at a time.
template <int READS>
int forward_dim(const Packed& a, hipStream_t s) {
    if (a.dim <= 32) return forward_of<32, 64, READS>(a, s);
    if (a.dim <= 64) return forward_of<64, 64, READS>(a, s);
    if (a.dim <= 96) return forward_of<96, 32, READS>(a, s);
    return forward_of<128, 32, READS>(a, s);
}
template <int READS>
int backward_dim(const Packed& a, hipStream_t s) {
    if (a.dim <= 32) return launch_backward<32, 64, READS>(a, s);
    if (a.dim <= 64) return launch_backward<64, 64, READS>(a, s);
    if (a.dim <= 96) return launch_backward<96, 32, READS>(a, s);
    return launch_backward<128, 32, READS>(a, s);
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int64_t ehip_attention_packed_workspace(const ehip_attention_packed_t* desc) {
    Packed a;
    if (fill("attention_packed", desc, a)) return -1;
    return int64_t(piece_bytes(a));
}

int ehip_attention_packed_f32(const ehip_attention_packed_t* desc, void* workspace,
                              size_t workspace_bytes, void* stream) {
    EHIP_READY();
    Packed a;
    if (int rc = fill("attention_packed", desc, a)) return rc;
    if (a.sequences == 0 || a.total_q == 0) return EHIP_OK;
    const size_t need = piece_bytes(a);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(EHIP_EINVAL, "attention_packed: needs %zu bytes of 16-byte aligned workspace",
                    need);
    a.pieces = pieces_of(a);
    a.piece_stats = static_cast<float2*>(workspace);
    a.piece_out = reinterpret_cast<float*>(
        a.piece_stats + int64_t(a.total_q) * a.heads * a.pieces);
    hipStream_t s = as_stream(stream);
    using namespace attention;
    if (a.dim < 4) return forward_of<32, 64, kSingle>(a, s);
    return a.dim % 4 == 0 ? forward_dim<kFours>(a, s) : forward_dim<kClamped>(a, s);
}

int64_t ehip_attention_packed_backward_workspace(const ehip_attention_packed_t* desc) {
    Packed a;
    if (fill("attention_packed_backward", desc, a)) return -1;
    return int64_t(bytes_of(space_of(a)));
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
        return fail(EHIP_EINVAL, "attention_packed_backward: null gradient, or its leading "
                                 "dimension below the row's length or above 2^22");
    if ((dq != nullptr && ld_dq < wide) || (dk != nullptr && ld_dk < narrow) ||
        (dv != nullptr && ld_dv < narrow))
        return fail(EHIP_EINVAL,
                    "attention_packed_backward: leading dimension below the row's length");
    const BackwardSpace space = space_of(a);
    const size_t need = bytes_of(space);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(EHIP_EINVAL,
                    "attention_packed_backward: needs %zu bytes of 16-byte aligned workspace",
                    need);
    a.grad = grad;
    a.ld_grad = ld_grad;
    a.dq = dq;
    a.dk = dk;
    a.dv = dv;
    a.ld_dq = ld_dq;
    a.ld_dk = ld_dk;
    a.ld_dv = ld_dv;
    a.delta = static_cast<float*>(workspace);
    // Without dq its kernel leaves delta alone, for which one piece is enough.
    a.pieces_q = dq != nullptr ? space.pieces_q : 1;
    a.pieces_k = space.pieces_k;
    char* at = static_cast<char*>(workspace) + space.delta;
    if (a.pieces_q > 1) a.part_q = reinterpret_cast<float*>(at);
    at += space.part_q;
    if (space.part_k != 0) {
        a.part_k = reinterpret_cast<float*>(at);
        a.part_v = reinterpret_cast<float*>(at + space.part_k);
    }
    hipStream_t s = as_stream(stream);
    using namespace attention;
    if (a.dim < 4) return launch_backward<32, 64, kSingle>(a, s);
    return a.dim % 4 == 0 ? backward_dim<kFours>(a, s) : backward_dim<kClamped>(a, s);
}

}  // extern "C"
