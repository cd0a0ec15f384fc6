// attention_paged.hpp -- the paged cache of keys and values and attention over it, of one token per
// sequence or, for positions that several sequences share, of one token of each of them:
//
//   s_p = scale (q . k_p), lse = log sum_p exp(s_p), out = sum_p exp(s_p - lse) v_p
#ifndef EHIP_ATTENTION_PAGED_HPP
#define EHIP_ATTENTION_PAGED_HPP

#include "attention_tile.hpp"
#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace ehip {
namespace paged {

constexpr int kMaxDim = 128;

struct Cache {
    void *k, *v;
    int64_t pages, page_size, kv_heads, dim;
    const int32_t* table;
    int64_t ld_table, width, sequences;
    float *k_scales, *v_scales;  // (pages, kv_heads, page_size) of a cache in 8 bits
    int page_shift;              // where the page size is 2 to it, else -1
};

// A position's table entry, and its place in the page: the read, and what is made of it.
struct Entry {
    int32_t page;
    uint32_t off;
};
// Of position p of sequence s, both in range. A position, a pool's rows and a page's are below 2^31:
// in 32 bits the division takes a tenth of the steps.
__device__ __forceinline__ Entry entry_of(const Cache& c, int64_t s, uint32_t p) {
    const uint32_t size = uint32_t(c.page_size);
    const uint32_t at = c.page_shift >= 0 ? p >> c.page_shift : p / size;
    return Entry{c.table[s * c.ld_table + at], p - at * size};
}
// The pools' row, or -1 where the entry names no page of theirs.
__device__ __forceinline__ int64_t row_of_entry(const Cache& c, const Entry& e) {
    if (e.page < 0 || e.page >= c.pages) return -1;
    return int64_t(uint64_t(uint32_t(e.page)) * uint32_t(c.page_size) + e.off);
}
// Of any position, -1 too where the table does not hold it.
__device__ __forceinline__ int64_t pool_row(const Cache& c, int64_t s, int64_t p, uint32_t& off) {
    if (p < 0 || p > INT32_MAX || p >= c.width * c.page_size) return -1;
    const Entry e = entry_of(c, s, uint32_t(p));
    off = e.off;
    return row_of_entry(c, e);
}
__device__ __forceinline__ int64_t pool_row(const Cache& c, int64_t s, int64_t p) {
    uint32_t off;
    return pool_row(c, s, p, off);
}
// Where the scale of a row's key head is: (page kv_heads + head) page_size + off.
__device__ __forceinline__ int64_t scale_of(const Cache& c, int64_t row, uint32_t off, int head) {
    const uint32_t heads = uint32_t(c.kv_heads);  // below 2^24
    return int64_t(uint64_t(uint32_t(row)) * heads - uint64_t(off) * (heads - 1)) +
           int64_t(head) * c.page_size;
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
// A whole number from -127 to 127, of a scale that its position and key head have.
struct Int8 {
    int8_t n;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(Bf16 x) {
    return __builtin_bit_cast(float, uint32_t(x.bits) << 16);
}
__device__ __forceinline__ float widen(Int8 x) { return float(x.n); }
// The nearest value of the pool's type, ties to even.
__device__ __forceinline__ void narrow(float x, float& out) { out = x; }
__device__ __forceinline__ void narrow(float x, Bf16& out) {
    out.bits = __builtin_bit_cast(uint16_t, __bf16(x));
}

// ----------------------------------------------------------------- attention

// The cache is read once and bounds the time, so the kernel's shape is that of its reads: a
// position's row of `dim` values takes LPP lanes, 16 bytes each, and a wave reads kUnroll x 64 /
// LPP positions of keys and values at a time. A lane holds its values of up to G query heads that
// share the keys. The lanes of a position add up its scores; each position's lanes keep their own
// running maximum, sum and weighted values over the positions they meet, joined at the end: of the
// wave, the block's four waves, and, where the length is split, the blocks of a sequence by a
// second launch. Two sequences of 131072 in fp32, 32 heads over 8 of 128 values: 356 us at best,
// 6.0 TB/s. It takes fp32, and bf16 where there is little (waves_of).
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
    int tile;            // positions that the work is cut by
    int workers;         // blocks, or waves, of a key head (and piece of its query heads)
    float2* part_stats;  // (heads, workers + sequences): maximum (as 2^x), sum
    float* part_out;     // (heads, workers + sequences, dim)
    int* first;          // (sequences + 1): the sequences' first tiles
    const int* starts;   // the sequences' first positions that are not shared, or null: 0
    // Positions that the sequences of a group share, read through its first sequence's table row.
    // A block has `rows` of the group's rows, its sequences' query heads of the key head.
    const int32_t *group_cu, *shared;
    int groups, rows;
    int places;          // parts of a key head, `rows` rows each
};

// The work is cut evenly, whatever the lengths: the positions of all sequences in tiles, one after
// the other, and a worker (a block of the vector kernel, a wave of the other, for each key head)
// takes its share of them, which may be part of a long sequence or several short ones. What a worker
// adds to a sequence is a segment. Segment (worker w, sequence s) has place w + s of a head's parts,
// no other's: from one to the next at least one of them grows.
constexpr int kTile = 128;      // of blocks
constexpr int kWaveTile = 32;   // of waves

// Positions of a sequence, -1 for a length that is none.
__device__ __forceinline__ int length_from(const Paged& a, int n) {
    return n < 0 || n > a.longest || n > a.c.width * a.c.page_size || (n > 0 && a.c.pages == 0)
               ? -1
               : n;
}
__device__ __forceinline__ int length_of(const Paged& a, int64_t s) {
    return length_from(a, a.lengths[s]);
}
__device__ __forceinline__ int tiles_of(const Paged& a, int n) {
    return n > 0 ? int(uint32_t(n - 1) / uint32_t(a.tile)) + 1 : 0;
}

// The first of a sequence's positions that are its own.
__device__ __forceinline__ int start_of(const Paged& a, int64_t s) {
    return a.starts != nullptr ? a.starts[s] : 0;
}

// A group's first sequence; the offsets ascend and are in range, and a group shares nothing that
// its table row could not have: shared_plan has seen to it.
__device__ __forceinline__ int group_begin(const Paged& a, int g) { return a.group_cu[g]; }
__device__ __forceinline__ int shared_of(const Paged& a, int g) { return a.shared[g]; }
// Place of the first row tile of a group: every group before it has at most as many as that.
__device__ __forceinline__ int row_tile_base(const Paged& a, int g) {
    const int group = a.heads / int(a.c.kv_heads);
    return int(int64_t(group_begin(a, g)) * group / a.rows) + g;
}

// What the tiles are counted over, 64 at a time in the lanes of a wave: the sequences, or with SHARED
// the groups, each row tile of which passes all of the group's positions.
struct Items {
    int base;        // of lane 0
    int start, end;  // positions
    int first;       // the sequence whose table row it goes by
    int rows;        // with SHARED the group's
};
// Tiles of a sequence or row tile, and row tiles, of a lane.
__device__ __forceinline__ int tiles_of(const Paged& a, const Items& x) {
    return tiles_of(a, x.end - x.start);
}
template <bool SHARED>
__device__ __forceinline__ int row_tiles_of(const Paged& a, int rows) {
    return SHARED ? (rows + a.rows - 1) / a.rows : 1;
}
template <bool SHARED>
__device__ __forceinline__ int items(const Paged& a) {
    return SHARED ? a.groups : int(a.c.sequences);
}
template <bool SHARED>
__device__ __forceinline__ Items items_from(const Paged& a, int base) {
    const int i = base + (int(threadIdx.x) & 63);
    Items x{base, 0, 0, i, 0};
    if (i < items<SHARED>(a)) {
        if (SHARED) {
            const int group = a.heads / int(a.c.kv_heads);
            x.first = group_begin(a, i);
            x.rows = (group_begin(a, i + 1) - x.first) * group;  // at most 2^24
            x.end = shared_of(a, i);
        } else {
            x.start = start_of(a, i);
            x.end = length_of(a, i);
        }
    }
    return x;
}

// The first tile of worker w of so many tiles, and the worker of tile t. With fewer tiles than
// workers the last ones have none; every other one has one at least.
__device__ __forceinline__ int first_tile(const Paged& a, int w, int tiles) {
    const int workers = min(a.workers, tiles);
    return w < workers ? int(int64_t(w) * tiles / workers) : tiles;
}
__device__ __forceinline__ int worker_of(const Paged& a, int t, int tiles) {
    // Both numbers are whole and below 2^53, so the quotient's rounding does not pass a whole one; in
    // whole numbers the division takes several times the steps.
    return int(double((int64_t(t) + 1) * min(a.workers, tiles) - 1) / double(tiles));
}

struct Segment {
    int64_t s;       // the sequence whose table row it goes by
    int item;        // the sequence, or the group
    int row_tile;    // of the group
    int rows;        // of the group
    int n;           // tiles of the sequence, or of the group's positions
    int row_tiles;   // of the group
    int from, to;    // all of the positions
    int begin, end;  // the segment's
    int t, t_end;    // the worker's tiles from here on
    int t0;          // the sequence's or the row tile's first
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

// The segment's positions from its item, row tile, t and t0.
template <bool SHARED>
__device__ __forceinline__ void measure(const Paged& a, Segment& g) {
    const int stop = min(g.t_end, g.t0 + g.n);
    g.begin = g.from + (g.t - g.t0) * a.tile;
    g.end = stop - g.t0 == g.n ? g.to : g.from + (stop - g.t0) * a.tile;
    g.whole = !SHARED && g.begin == 0 && g.end == g.to;
}

// Takes the item of a lane.
template <bool SHARED>
__device__ __forceinline__ void take(const Paged& a, const Items& x, int lane, Segment& g) {
    const auto of = [&](int y) { return __builtin_amdgcn_readlane(y, lane); };
    g.item = x.base + lane;
    g.s = SHARED ? of(x.first) : g.item;
    g.rows = SHARED ? of(x.rows) : 0;
    g.row_tiles = row_tiles_of<SHARED>(a, g.rows);
    g.from = SHARED ? 0 : of(x.start);
    g.to = of(x.end);
    g.n = tiles_of(a, g.to - g.from);
}

// The first segment of worker w (t == t_end: none), and the items that it is among. Every wave finds
// the same; block 0 leaves the items' first tiles for the join.
template <bool SHARED>
__device__ __forceinline__ Segment first_segment(const Paged& a, uint32_t block, int w, Items& x) {
    const int lane = int(threadIdx.x) & 63;
    const int count = items<SHARED>(a);
    int tiles = 0;
    for (int base = 0; base < count; base += 64) {
        x = items_from<SHARED>(a, base);
        const int mine = tiles_of(a, x) * row_tiles_of<SHARED>(a, x.rows), upto = wave_scan(mine);
        if (block == 0 && threadIdx.x < 64 && base + lane < count)
            a.first[base + lane] = tiles + upto - mine;
        tiles += __shfl(upto, 63);
    }
    if (block == 0 && threadIdx.x == 0) a.first[count] = tiles;
    Segment g{};
    g.t = __builtin_amdgcn_readfirstlane(first_tile(a, w, tiles));
    g.t_end = __builtin_amdgcn_readfirstlane(first_tile(a, w + 1, tiles));
    if (g.t == g.t_end) return g;
    int before = 0;
    for (int base = 0; base < count; base += 64) {
        if (count > 64) x = items_from<SHARED>(a, base);
        const int mine = tiles_of(a, x) * row_tiles_of<SHARED>(a, x.rows), upto = before + wave_scan(mine);
        const uint64_t past = __ballot(upto > g.t);
        if (past != 0) {
            const int at = __builtin_ctzll(past);
            take<SHARED>(a, x, at, g);
            g.t0 = __builtin_amdgcn_readlane(upto - mine, at);
            break;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    g.n = max(1, g.n);  // 0 only where lengths change under the launch
    if (SHARED) {
        g.row_tile = (g.t - g.t0) / g.n;
        g.t0 += g.row_tile * g.n;
    }
    measure<SHARED>(a, g);
    return g;
}

template <bool SHARED>
__device__ __forceinline__ void next_segment(const Paged& a, Segment& g, Items& x) {
    const int stop = g.t0 + g.n;
    g.t = min(g.t_end, stop);
    if (g.t == g.t_end) return;
    g.t0 = stop;
    if (SHARED && g.row_tile + 1 < g.row_tiles) {
        ++g.row_tile;
        measure<SHARED>(a, g);
        return;
    }
    g.row_tile = 0;
    int lane = g.item - x.base + 1;  // 64 at most
    while (true) {
        const uint64_t some = lane < 64 ? __ballot(x.end > x.start && (!SHARED || x.rows > 0)) >> lane : 0;
        if (some != 0) {
            lane += __builtin_ctzll(some);
            break;
        }
        if (x.base + 64 >= items<SHARED>(a)) {  // only where the lengths changed under the launch
            g.t = g.t_end;
            return;
        }
        x = items_from<SHARED>(a, x.base + 64);
        lane = 0;
    }
    take<SHARED>(a, x, lane, g);
    measure<SHARED>(a, g);
}

// A block's query rows of a segment: heads h0 .. of the sequence, or rows of the group, each a head
// of one of its sequences.
template <bool SHARED>
__device__ __forceinline__ int rows_of(const Paged& a, const Segment& g, int count) {
    return SHARED ? min(a.rows, g.rows - g.row_tile * a.rows) : count;
}
template <bool SHARED>
__device__ __forceinline__ const float* query_row(const Paged& a, const Segment& g, int kv, int h0,
                                                  int i) {
    if (!SHARED) return a.q + g.s * a.ld_q + int64_t(h0 + i) * a.c.dim;
    const int group = a.heads / int(a.c.kv_heads);
    const int r = g.row_tile * a.rows + i;
    return a.q + (g.s + r / group) * a.ld_q + (int64_t(kv) * group + r % group) * a.c.dim;
}
// Where the part of row i is.
template <bool SHARED>
__device__ __forceinline__ int64_t part_of(const Paged& a, const Segment& g, int worker, int kv,
                                           int h0, int i) {
    if (!SHARED) return int64_t(h0 + i) * (a.workers + a.c.sequences) + worker + g.s;
    const int place = worker + row_tile_base(a, g.item) + g.row_tile;
    return (int64_t(kv) * a.places + place) * a.rows + i;
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

// The largest of the four lanes 16 apart, in each of them.
__device__ __forceinline__ float largest_of_rows(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x),
                                                    __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t x0 = r[0], x1 = r[1];
    x = fmaxf(__builtin_bit_cast(float, x0), __builtin_bit_cast(float, x1));
    const auto h = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x),
                                                    __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t y0 = h[0], y1 = h[1];
    return fmaxf(__builtin_bit_cast(float, y0), __builtin_bit_cast(float, y1));
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
__global__ __launch_bounds__(kPagedThreads, G >= 4 ? 2 : 3) void paged_part(Paged a) {
    constexpr int N = Values<T, VEC>::N, SUBS = 64 / LPP, TILE = SUBS * kUnroll;
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
    Items among;
    for (Segment seg = first_segment<false>(a, blockIdx.x, worker, among); seg.t < seg.t_end;
         next_segment<false>(a, seg, among)) {
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
            const float* row = query_row<false>(a, seg, kv, h0, g < count ? g : 0) + d0;
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
            const int64_t at = part_of<false>(a, seg, worker, kv, h0, g);
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

// Up to AGAIN heads' share of a segment by the formula, for those whose sums by parts are not finite: a
// part of an infinity, or an infinity times the parts of a finite value, is NaN where the product is
// an infinity or, its weight 0, nothing at all. One wave, a lane for each of 64 positions at a time; a
// score of NaN or +inf settles its head as NaN. Each segment's wave forms its own, so its reads are
// several at a time and serve four heads (64 sequences of 1024, 32 heads over 8 of 128 values, us, bf16
// and 8 bits: finite 52 and 37; the first key NaN 69 and 48, a head and a read at a time 82 and 98; the
// first value infinite 274 and 130, and 623 and 555).
template <class T, int DP, int AGAIN>
__device__ void part_by_formula(const Paged& a, int64_t s, const float* const (&q)[AGAIN], int kv,
                                int begin, int end, float (&top)[AGAIN], float (&sum)[AGAIN],
                                float (&o)[AGAIN][2]) {
    using attention::uintx4;
    constexpr int kReads = DP > 64 ? 4 : 2;  // more than the tiles leave registers for hold up those
    int lane = int(threadIdx.x) & 63;
    asm volatile("" : "+v"(lane));  // else what follows from it is held all through the tiles
    const int dim = int(a.c.dim);
    const int64_t pitch = a.c.kv_heads * dim;
    const T* k = static_cast<const T*>(a.c.k) + int64_t(kv) * dim;
    const T* v = static_cast<const T*>(a.c.v) + int64_t(kv) * dim;
    const float c2 = a.scale * 1.44269504088896340736f;
    // The pool row of position p0 + lane, the last again past the end, and where its scales are.
    int64_t place = 0;
    const auto row_of = [&](int p0) {
        uint32_t off = 0;
        const int64_t row = pool_row(a.c, s, min(p0 + lane, end - 1), off);
        if constexpr (sizeof(T) == 1) place = scale_of(a.c, row, off, kv);
        return int(row);
    };
    // Rows of 16-byte units, or others four values at a time at any address.
    const bool units = sizeof(T) == 2 && dim % 8 == 0 && aligned16(a.c.k);
    const auto scores = [&](int row, float (&dot)[AGAIN]) {
        const T* at = k + int64_t(row) * pitch;
        const float by = sizeof(T) == 1 ? a.c.k_scales[place] : 1.0f;
#pragma unroll
        for (int g = 0; g < AGAIN; ++g) dot[g] = 0.0f;
        const auto add = [&](int e, float x) {
#pragma unroll
            for (int g = 0; g < AGAIN; ++g) dot[g] = __builtin_fmaf(q[g][e] * c2, x, dot[g]);
        };
        int e = 0;
        if (units) {
            for (; e < dim; e += 8 * kReads) {  // several at a time, past the end the first again
                uintx4 x[kReads];
#pragma unroll
                for (int i = 0; i < kReads; ++i)
                    x[i] = *reinterpret_cast<const uintx4*>(at + (e + 8 * i < dim ? e + 8 * i : 0));
#pragma unroll
                for (int i = 0; i < kReads; ++i) {
                    __builtin_amdgcn_sched_barrier(0);  // the next eight of q are not held as well
                    if (e + 8 * i >= dim) break;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t pair = x[i][j];
                        add(e + 8 * i + 2 * j, __builtin_bit_cast(float, pair << 16));
                        add(e + 8 * i + 2 * j + 1, __builtin_bit_cast(float, pair & 0xffff0000u));
                    }
                }
            }
            return;
        }
        for (; e + 16 <= dim; e += 16) {
            T x[16];
            __builtin_memcpy(x, at + e, sizeof(x));
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (j % 4 == 0) __builtin_amdgcn_sched_barrier(0);
                add(e + j, sizeof(T) == 1 ? widen(x[j]) * by : widen(x[j]));
            }
        }
        for (; e + 4 <= dim; e += 4) {
            T x[4];
            __builtin_memcpy(x, at + e, sizeof(x));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                add(e + j, sizeof(T) == 1 ? widen(x[j]) * by : widen(x[j]));
        }
        for (; e < dim; ++e) add(e, sizeof(T) == 1 ? widen(at[e]) * by : widen(at[e]));
    };
    float x[AGAIN], shift[AGAIN];
    bool settled[AGAIN], all = false;
#pragma unroll
    for (int g = 0; g < AGAIN; ++g) {
        top[g] = -INFINITY;
        settled[g] = false;
    }
    for (int p0 = begin; p0 < end && !all; p0 += 64) {
        scores(row_of(p0), x);
        all = true;
#pragma unroll
        for (int g = 0; g < AGAIN; ++g) {
            settled[g] = settled[g] || __any(!(x[g] < INFINITY));
            all = all && settled[g];
            top[g] = fmaxf(top[g], x[g]);
        }
    }
#pragma unroll
    for (int g = 0; g < AGAIN; ++g) {
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) top[g] = fmaxf(top[g], __shfl_xor(top[g], w));
        shift[g] = top[g] == -INFINITY ? 0.0f : top[g];  // scores of -inf alone weigh nothing
        sum[g] = o[g][0] = o[g][1] = 0.0f;
    }
    const int d0 = lane < dim ? lane : 0, d1 = lane + 64 < dim ? lane + 64 : 0;
    bool none = false;  // a scale that is not finite settles the values, whatever its weight
    for (int p0 = begin; p0 < end && !all; p0 += 64) {
        const int row = row_of(p0), count = min(64, end - p0);
        scores(row, x);
#pragma unroll
        for (int g = 0; g < AGAIN; ++g) {
            x[g] = lane < count ? exp2f(x[g] - shift[g]) * 0x1p-24f : 0.0f;
            sum[g] += x[g];
        }
        const float vs = sizeof(T) == 1 ? a.c.v_scales[place] : 1.0f;
        if (sizeof(T) == 1) none = none || __any(!(fabsf(vs) < INFINITY));
        if (none) continue;
        for (int u0 = 0; u0 < count; u0 += 2 * kReads) {  // several positions' reads at a time
            T from[2 * kReads][2];
#pragma unroll
            for (int i = 0; i < 2 * kReads; ++i) {
                const T* at = v + int64_t(__shfl(row, u0 + i)) * pitch;
                from[i][0] = at[d0];
                from[i][1] = at[d1];
            }
#pragma unroll
            for (int i = 0; i < 2 * kReads; ++i) {
                const int u = u0 + i;  // 63 at most; past the end the last again, for nothing
                const float scale = sizeof(T) == 1 ? __shfl(vs, u) : 1.0f;
                float y[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    y[e] = widen(from[i][e]);
                    if (sizeof(T) == 1) y[e] *= scale;
                    y[e] = u < count ? y[e] : 0.0f;
                }
#pragma unroll
                for (int g = 0; g < AGAIN; ++g) {
                    const float w = __shfl(x[g], u);
                    o[g][0] = __builtin_fmaf(w, y[0], o[g][0]);
                    o[g][1] = __builtin_fmaf(w, y[1], o[g][1]);
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < AGAIN; ++g) {
#pragma unroll
        for (int w = 32; w > 0; w >>= 1) sum[g] += __shfl_xor(sum[g], w);
        if (settled[g]) top[g] = 0.0f, sum[g] = NAN;
        if (settled[g] || none) o[g][0] = o[g][1] = NAN;
    }
}

// The next rows of a set, the last again past its end, which is cleared of them.
template <int AGAIN>
struct Again {
    int row[AGAIN], count;
    __device__ __forceinline__ explicit Again(uint32_t& rows) : count(0) {
#pragma unroll
        for (int g = 0; g < AGAIN; ++g) {
            row[g] = rows != 0 ? __builtin_ctz(rows) : row[g > 0 ? g - 1 : 0];
            count += rows != 0;
            rows &= rows - 1;
        }
    }
};

// A cache in bf16, up to 16 query heads of a key head at a time, on v_mfma_f32_16x16x32_bf16: the
// cached values are operands as they are, q and the weights in three parts, so a score and a
// weighted value take three products each, for any number of heads at one cost; by vector
// instructions four heads ran at 4.3 TB/s of 5.4 and eight at 2.7. HBM bounds it (64 sequences up
// to 4096, 32 heads over 8 of 128: 265 MB in 49 us, 5.4 TB/s). Lane l holds A(l % 16, 8 (l / 16) +
// 0..7), B(8 (l / 16) + 0..7, l % 16) and D(4 (l / 16) + r, l % 16).
//   scores:  A = 16 positions by 32 values of K, as 16-byte reads leave them; B = q; D's columns
//            are heads
//   weights: the D's of positions 0..15 and 16..31 are the B of 32 positions, in the order
//            4 h + 0..3, 16 + 4 h + 0..3 for the lanes h = l / 16
//   values:  A = 16 values by those 32 positions of V: rows in LDS, read transposed
// A wave takes 32 positions at a time; the next ones' reads are out while it forms weights and sums,
// and so across the end of a segment: the waves of a block have nothing in common but that they read
// the key heads of the same positions, which lie next to each other.
constexpr int kTilePositions = 32;

// A cache in 8 bits goes the same way: whole numbers up to 127 are bf16 values, made of the bytes
// in registers, a score is multiplied by its position's scale of K and a weight by that of V. The
// 1.5 instructions a value are a third of the kernel's (64 sequences up to 8192: 260 MB in 53 us, 4.9
// TB/s).
using attention::uintx4;
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

// A lane's N values of a row from d0 on, as they are read, and eight of them at a time as bf16.
// WIDE: rows of whole groups of N values at N bytes in 8 bits, or of 8 values at 16 bytes in bf16.
template <class T, int N, bool WIDE>
struct Piece;
template <int N, bool WIDE>
struct Piece<Bf16, N, WIDE> {
    static_assert(N == 8, "what is read at a time");
    uintx4 x;
    __device__ __forceinline__ void load(const Bf16* row, int d0, int dim) {
        if (WIDE) {
            x = *reinterpret_cast<const uintx4*>(row + (d0 < dim ? d0 : 0));
        } else if (dim < 8) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint32_t lo = d0 + e < dim ? row[d0 + e].bits : 0;
                const uint32_t hi = d0 + e + 1 < dim ? row[d0 + e + 1].bits : 0;
                x[e / 2] = lo | hi << 16;
            }
        } else {
            __builtin_memcpy(&x, row + min(d0, dim - 8), 16);
        }
    }
    // Past the row's end 0, or with WIDE anything.
    __device__ __forceinline__ uintx4 bf16(int, int d0, int dim) const {
        if (WIDE || dim < 8) return x;
        uint64_t z[2];
        __builtin_memcpy(z, &x, 16);
        const int by = 16 * max(0, min(d0 - (dim - 8), 8)), low = by & 63;
        const uint64_t both = z[0] >> low | z[1] << 1 << (63 - low), high = z[1] >> low;
        z[0] = by < 64 ? both : by < 128 ? high : 0;
        z[1] = by < 64 ? high : 0;
        uintx4 y;
        __builtin_memcpy(&y, z, 16);
        return y;
    }
};
// Other rows, of any length and at any address, are read eight values at a time, the last eight
// where fewer are left. Those are shifted to their places where they are used: earlier, the read
// would be waited for a tile ahead (in 8 bits, 64 sequences up to 8192, 32 heads over 8 of 128
// values, with reads like that: 202 us in place of 85).
template <int N, bool WIDE>
struct Piece<Int8, N, WIDE> {
    uint32_t x[N / 4];
    __device__ __forceinline__ void load(const Int8* row, int d0, int dim) {
        if (WIDE) {
            __builtin_memcpy(x, __builtin_assume_aligned(row + (d0 < dim ? d0 : 0), N), N);
            return;
        }
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            if (dim < 8) {
                uint64_t y = 0;
                for (int e = 0; e < dim; ++e) y |= uint64_t(uint8_t(row[e].n)) << (8 * e);
                __builtin_memcpy(x + 2 * i, &y, 8);
            } else {
                __builtin_memcpy(x + 2 * i, row + min(d0 + 8 * i, dim - 8), 8);
            }
        }
    }
    // Values 8 i .. of the piece; past the row's end 0, or with WIDE anything.
    __device__ __forceinline__ uintx4 bf16(int i, int d0, int dim) const {
        uint32_t y[2] = {x[2 * i], x[2 * i + 1]};
        if (!WIDE) {
            uint64_t z;
            __builtin_memcpy(&z, y, 8);
            const int d = d0 + 8 * i, from = max(0, min(d, dim - 8));
            z = d < dim ? z >> (8 * (d - from)) : 0;
            __builtin_memcpy(y, &z, 8);
        }
        uintx4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int32_t word = int32_t(y[j / 2]);
            const float lo = float(int8_t(word >> (16 * (j & 1))));
            const float hi = float(int8_t(word >> (16 * (j & 1) + 8)));
            r[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi),
                                         __builtin_bit_cast(uint32_t, lo), 0x07060302u);
        }
        return r;
    }
};

// Whether a query row, of this largest |scale q|, is left to the formula. Below 2^-110 the parts of its
// values lose bits. In 8 bits the products are sums of q times whole numbers of up to 127, which the
// position's scale multiplies only then: from 2^113 on they could pass fp32 where the score does not.
// (A factor for such rows, taken out of q and put to their scores, held a register more through the
// tiles: 256 sequences up to 300 in bf16, 16 heads of 128, 93 us against 90, and 88 without either.)
template <class T>
__device__ __forceinline__ bool out_of_parts(float largest) {
    return (largest > 0.0f && largest < 0x1p-100f) || (sizeof(T) == 1 && largest > 0x1p112f);
}

// Eight values of a query row of any length at any address, four at a time, which are put in place where
// they are used; one by one an address each is held, and with heads over 64 spilled (64 sequences up
// to 1024, 32 heads over 8 of 100, bf16 65 us, like this 52; 256 up to 300, 16 of 33, 8 bits 63, 65).
__device__ __forceinline__ void ask_eight(const float* row, int d0, int dim, float (&x)[8]) {
    if (dim < 4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = row[d0 + e < dim ? d0 + e : 0];
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        const auto y = *reinterpret_cast<const attention::floatx4u*>(
            row + attention::clamped<attention::kClamped>(d0 + e, dim));
#pragma unroll
        for (int j = 0; j < 4; ++j) x[e + j] = y[j];
    }
}
__device__ __forceinline__ void eight_in_place(float (&x)[8], int d0, int dim) {
    if (dim < 4) return;
    attention::in_place<attention::kClamped>(x, d0, dim);
    attention::in_place<attention::kClamped>(x + 4, d0 + 4, dim);
}

constexpr int value_pitch(int dp) { return 2 * dp + 32; }  // bytes of a row of V in LDS
template <int DP>
struct alignas(16) PartLds {
    char values[kPagedWaves][kTilePositions * value_pitch(DP)];
    float scales[kPagedWaves][2][kTilePositions];
};

template <class T, int DP, bool WIDE, bool SHARED, int AGAIN>
__device__ __forceinline__ void part_by_waves(const Paged& a, uint32_t block, PartLds<DP>& lds) {
    constexpr bool kScaled = sizeof(T) == 1;
    using attention::bf16x8;
    using attention::floatx4u;
    typedef float floatx4 __attribute__((ext_vector_type(4)));
    typedef short shortx4 __attribute__((ext_vector_type(4)));
    constexpr int N = kScaled && DP > 32 ? 16 : 8;             // values of a piece
    constexpr int KS = DP / 32, KP = DP / (4 * N), NV = DP / 16;
    constexpr int LANES = DP / N;                              // of a row's reads
    constexpr int kRows = 64 / LANES, kReads = (kTilePositions + kRows - 1) / kRows;
    // Rows 32 bytes apart in banks: a transposed read's sixteen rows take all banks twice.
    constexpr int kPitch = value_pitch(DP);
    const int lane = int(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int kv_heads = int(a.c.kv_heads), dim = int(a.c.dim);
    const int group = a.heads / kv_heads, pieces = SHARED ? 1 : (group + 15) / 16;
    uint32_t x = block * kPagedWaves + wave;
    const int kv = int(x % uint32_t(kv_heads));
    x /= uint32_t(kv_heads);
    const int h0 = kv * group + int(x % uint32_t(pieces)) * 16;
    const int heads = min(16, (kv + 1) * group - h0);  // the wave's
    x /= uint32_t(pieces);
    const int worker = int(x);
    if (worker >= a.workers) return;  // no barrier follows
    Items among;
    for (Segment seg = first_segment<SHARED>(a, block, worker, among); seg.t < seg.t_end;
         next_segment<SHARED>(a, seg, among)) {
        const int64_t s = seg.s;
        const int count = rows_of<SHARED>(a, seg, heads);
        const int begin = seg.begin, end = seg.end;
        bool bad = false;  // a page outside the pool

        const int col = lane & 15, quarter = lane / 16;
        const float c2 = a.scale * 1.44269504088896340736f;
        floatx4 o[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        uint64_t apart = 0;  // rows for the formula

        const T* const k = static_cast<const T*>(a.c.k) + int64_t(kv) * dim;
        const T* const v = static_cast<const T*>(a.c.v) + int64_t(kv) * dim;
        const uint32_t pitch = uint32_t(kv_heads * dim);  // below 2^31, as the rows
        Piece<T, N, WIDE> kx[2][KP], vx[kReads];
        float k_scale = 0.0f, v_scale = 0.0f;  // of the tile's position lane % 32
        const int v_lane = lane / LANES, v_d0 = lane % LANES * N;
        // The table's entry of position p0 + lane % 32, or the last, is asked for a tile before its
        // row is read, and last of the tile's reads: what is made of it waits for those before it
        // too. So would a choice that stands between the read and its use.
        Entry entry;
        int r = 0;
        int64_t place = 0;
        const auto ask = [&](int p0) {
            entry = entry_of(a.c, s, uint32_t(min(p0 + (lane & 31), end - 1)));
        };
        const auto find = [&] {
            int64_t row = row_of_entry(a.c, entry);
            if (row < 0) {
                bad = true;
                row = 0;
                entry.off = 0;
            }
            if constexpr (kScaled) place = scale_of(a.c, row, entry.off, kv);
            r = int(row);
        };
        const auto load = [&](int p0) {
            if constexpr (kScaled) {
                const bool in = p0 + (lane & 31) < end;
                k_scale = in ? a.c.k_scales[place] : 0.0f;
                v_scale = in ? a.c.v_scales[place] : 0.0f;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const T* at = k + uint64_t(uint32_t(__shfl(r, 16 * t + col))) * pitch;
#pragma unroll
                for (int p = 0; p < KP; ++p)
                    kx[t][p].load(at, 4 * N * p + N * quarter, dim);
            }
#pragma unroll
            for (int i = 0; i < kReads; ++i) {
                const int j = i * kRows + v_lane;
                const T* at = v + uint64_t(uint32_t(__shfl(r, j < kTilePositions ? j : 0))) * pitch;
                vx[i].load(at, v_d0, dim);
            }
        };
        char* const mine = lds.values[wave];
        // q is asked for between the table and the rows that it names, and split while those are on
        // their way; of wide heads in bf16, where that spills, before the table.
        constexpr bool kFirst = !kScaled && DP > 64, kFours = !WIDE && DP > 64;
        float qx[KS][8];
        bf16x8 q[KS][3];
        const auto ask_query = [&] {
            const float* const row = query_row<SHARED>(a, seg, kv, h0, col < count ? col : 0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d0 = 4 * N * (8 * ks / N) + N * quarter + 8 * ks % N;
                // With WIDE a head is a multiple of eight values, and one offset serves them all: those
                // of each would be kept over the segments, in scratch.
                if (kFours) {
                    ask_eight(row, d0, dim, qx[ks]);
                    continue;
                }
                const int from = WIDE && d0 < dim ? d0 : 0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    qx[ks][e] = row[WIDE ? from + e : d0 + e < dim ? d0 + e : 0];
            }
        };
        const auto split_query = [&] {
            float largest = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d0 = 4 * N * (8 * ks / N) + N * quarter + 8 * ks % N;
                if (kFours) eight_in_place(qx[ks], d0, dim);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = d0 + (WIDE ? 0 : e) < dim;
                    qx[ks][e] = in && col < count ? qx[ks][e] : 0.0f;
                    largest = fmaxf(largest, fabsf(qx[ks][e]));
                }
            }
            apart = __ballot(out_of_parts<T>(largest_of_rows(largest) * fabsf(c2)));
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 8; ++e) qx[ks][e] *= c2;
                attention::split8(qx[ks], q[ks]);
            }
        };
        if (kFirst) {
            ask_query();
            split_query();
            __builtin_amdgcn_sched_barrier(0);
        }
        ask(begin);
        if (!kFirst) ask_query();
        find();
        load(begin);
        ask(begin + kTilePositions);
        if (!kFirst) split_query();
        for (int p0 = begin; p0 < end; p0 += kTilePositions) {
            const bool tail = p0 + kTilePositions > end;
#pragma unroll
            for (int i = 0; i < kReads; ++i) {
                const int j = i * kRows + v_lane;
#pragma unroll
                for (int e = 0; e < N / 8; ++e) {
                    uintx4 y = vx[i].bf16(e, v_d0, dim);
                    // Nothing, whatever is there; in 8 bits its scale is 0.
                    if (!kScaled && tail && p0 + j >= end) y = uintx4{0, 0, 0, 0};
                    if (v_lane < kRows && j < kTilePositions)
                        *reinterpret_cast<uintx4*>(mine + j * kPitch + 2 * v_d0 + 16 * e) = y;
                }
            }
            if constexpr (kScaled) {
                if (lane < kTilePositions) {
                    lds.scales[wave][0][lane] = k_scale;
                    lds.scales[wave][1][lane] = v_scale;
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
            const auto scales = [&](int which, int t) {  // of a lane's scores
                return *reinterpret_cast<const floatx4*>(
                    &lds.scales[wave][which][16 * t + 4 * quarter]);
            };
            // The smaller parts' products and the first parts' apart, four chains of them: the
            // matrix instruction drops the low bits of its sums, least where they are small.
            floatx4 sc[2], small[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) sc[t] = small[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d0 = 4 * N * (8 * ks / N) + N * quarter;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    // Past the row's end q is 0 and K something else, which has to be finite.
                    bf16x8 f = __builtin_bit_cast(
                        bf16x8, kx[t][8 * ks / N].bf16(ks % (N / 8), d0, dim));
                    if (!kScaled && DP != dim && 32 * ks + 8 * quarter >= dim)
                        f = __builtin_bit_cast(bf16x8, uintx4{0, 0, 0, 0});
                    small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, q[ks][2], small[t], 0, 0,
                                                                       0);
                    small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, q[ks][1], small[t], 0, 0,
                                                                       0);
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, q[ks][0], sc[t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) sc[t] += small[t];
            // Past the end the last row again: on a condition the table's entry would be copied, and
            // waited for, where the paths meet.
            find();
            load(p0 + kTilePositions);
            ask(p0 + 2 * kTilePositions);
            if constexpr (kScaled) {
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[t] *= scales(0, t);
            }
            if (tail) {
                asm volatile("");  // a branch: as selects in every step, 16 instructions
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
            top = largest_of_rows(top);
            const float shift = top == -INFINITY ? 0.0f : top;
            const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - shift);
            m = top;
            float w[8], part_sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] = __builtin_amdgcn_exp2f(sc[j / 4][j % 4] - shift);
                part_sum += w[j];
            }
            l = __builtin_fmaf(l, keep, part_sum);
            if constexpr (kScaled) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const floatx4 by = scales(1, t);
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[4 * t + r] *= by[r];
                }
            }
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
        // Head `col`, values 16 i + 4 quarter + r.
        bad = __any(bad);
        l = with_half(with_row_pair(l));
        bool fine = l > 0.0f && l < INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) fine = fine && fabsf(o[i][r]) < INFINITY;
        const uint64_t lanes = __ballot(!fine) | apart;
        uint32_t again = uint32_t(lanes | lanes >> 32);
        again = (again | again >> 16) & 0xffffu & ((1u << count) - 1u);
        const int64_t at = part_of<SHARED>(a, seg, worker, kv, h0, col < count ? col : 0);
        if (bad) l = NAN;
        if (col < count && (bad || !(again >> col & 1))) {
            if (quarter == 0) {
                // As the other parts and sums, 2^-24 of what they are.
                if (!seg.whole) a.part_stats[at] = float2{m, l * 0x1p-24f};
                else if (a.lse != nullptr) a.lse[s * a.heads + h0 + col] = lse_of(m, l * 0x1p-24f);
            }
            float* const to = seg.whole ? a.out + s * a.ld_out + int64_t(h0 + col) * dim
                                        : a.part_out + at * dim;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int d = 16 * i + 4 * quarter;
                floatx4u y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = seg.whole ? o[i][r] / l : o[i][r] * 0x1p-24f;
                if (d + (WIDE ? 0 : 3) < dim) {
                    *reinterpret_cast<floatx4u*>(to + d) = y;
                } else if (!WIDE) {
#pragma unroll
                    for (int r = 0; r < 3; ++r)
                        if (d + r < dim) to[d + r] = y[r];
                }
            }
        }
        if (bad) continue;
        while (again != 0) {
            const Again<AGAIN> some(again);
            const float* rows[AGAIN];
#pragma unroll
            for (int i = 0; i < AGAIN; ++i) rows[i] = query_row<SHARED>(a, seg, kv, h0, some.row[i]);
            float top[AGAIN], sum[AGAIN], y[AGAIN][2];
            part_by_formula<T, DP, AGAIN>(a, s, rows, kv, begin, end, top, sum, y);
#pragma unroll
            for (int i = 0; i < AGAIN; ++i) {
                const int g = some.row[i];
                const int64_t place = part_of<SHARED>(a, seg, worker, kv, h0, g);
                if (i < some.count && lane == 0) {
                    if (!seg.whole) a.part_stats[place] = float2{top[i], sum[i]};
                    else if (a.lse != nullptr)
                        a.lse[s * a.heads + h0 + g] = lse_of(top[i], sum[i]);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = lane + 64 * e;
                    if (i >= some.count || d >= dim) continue;
                    if (!seg.whole) a.part_out[place * dim + d] = y[i][e];
                    else a.out[s * a.ld_out + int64_t(h0 + g) * dim + d] = y[i][e] / sum[i];
                }
            }
        }
    }
}

template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_part_mfma(Paged a) {
    __shared__ PartLds<DP> lds;
    part_by_waves<T, DP, WIDE, false, 4>(a, blockIdx.x, lds);
}

// Parts of a row, `stride` rows apart.
struct Parts {
    const float2* stats;
    const float* out;
    int count;
    int64_t stride;
};

// What a sequence's own parts are found by, read at once, before any of it is used: a join is a
// chain of reads.
struct Own {
    int length, start, tiles, first, end;
};
__device__ __forceinline__ Own own_of(const Paged& a, int64_t s) {
    return Own{a.lengths[s], start_of(a, s), a.first[a.c.sequences], a.first[s], a.first[s + 1]};
}

// The sequence's own parts of a head (stats null: of none). One that is its only one is whole.
__device__ __forceinline__ Parts own_parts(const Paged& a, const Own& x, int64_t s, int h) {
    if (x.first == x.end) return Parts{nullptr, nullptr, 0, 1};
    const int w0 = worker_of(a, x.first, x.tiles);
    const int64_t from = int64_t(h) * (a.workers + a.c.sequences) + w0 + s;
    return Parts{a.part_stats + from, a.part_out + from * a.c.dim,
                 worker_of(a, x.end - 1, x.tiles) - w0 + 1, 1};
}

// Row (s, h) of the results from its parts, by WAVES waves that take them in turn: one where the
// rows fill the card, as each finds the parts' places by itself (2752 rows of some eleven parts: 10
// us against 17 with four). Lane d has values d and d + 64. Every thread calls it.
template <int WAVES>
__device__ __forceinline__ void join_parts(const Paged& a, int64_t s, int h, const Parts (&p)[2],
                                           float (*sh)[kMaxDim + 1]) {
    const int lane = int(threadIdx.x) & 63, wave = WAVES > 1 ? int(threadIdx.x) / 64 : 0;
    const int dim = int(a.c.dim);
    const int d0 = lane < dim ? lane : 0, d1 = lane + 64 < dim ? lane + 64 : 0;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        for (int i = lane; i < p[k].count; i += 64)
            top = fmaxf(top, p[k].stats[i * p[k].stride].x);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    float sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll 4
        for (int i = wave; i < p[k].count; i += WAVES) {
            const float2 z = p[k].stats[i * p[k].stride];
            const float* const from = p[k].out + i * p[k].stride * dim;
            const float x0 = from[d0], x1 = from[d1];
            const float keep = z.x == -INFINITY ? (z.y != z.y ? NAN : 0.0f)
                                                : __builtin_amdgcn_exp2f(z.x - top);
            sum += z.y * keep;
            y0 = __builtin_fmaf(x0, keep, y0);
            y1 = __builtin_fmaf(x1, keep, y1);
        }
    }
    if (WAVES > 1) {
        sh[wave][lane] = y0;
        sh[wave][lane + 64] = y1;
        if (lane == 0) sh[wave][kMaxDim] = sum;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            sum += sh[w][kMaxDim];
            y0 += sh[w][lane];
            y1 += sh[w][lane + 64];
        }
    }
    float* const out = a.out + s * a.ld_out + int64_t(h) * dim;
    if (lane < dim) out[lane] = y0 / sum;
    if (lane + 64 < dim) out[lane + 64] = y1 / sum;
    if (lane == 0 && a.lse != nullptr) a.lse[s * a.heads + h] = lse_of(top, sum);
}

// The row of a sequence without positions, or of a length that is none.
template <int WAVES>
__device__ __forceinline__ void empty_row(const Paged& a, int64_t s, int h, int n) {
    const int t = int(threadIdx.x) % (64 * WAVES);
    float* const out = a.out + s * a.ld_out + int64_t(h) * a.c.dim;
    for (int d = t; d < int(a.c.dim); d += 64 * WAVES) out[d] = n < 0 ? NAN : 0.0f;
    if (t == 0 && a.lse != nullptr) a.lse[s * a.heads + h] = n < 0 ? NAN : -INFINITY;
}

// ---------------------------------------------------------------- host checks

constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

inline int check(const char* name, const ehip_cache_t* c, Cache& out) {
    if (c == nullptr) return fail(EHIP_EINVAL, "%s: null cache", name);
    if (c->type < EHIP_CACHE_F32 || c->type > EHIP_CACHE_I8 || c->pages < 0 ||
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
    out = Cache{c->k_pages,  c->v_pages,     c->pages,     c->page_size, c->kv_heads, c->head_dim,
                c->table,    c->ld_table,    c->table_width, c->sequences, nullptr,     nullptr, -1};
    if ((c->page_size & (c->page_size - 1)) == 0)
        out.page_shift = __builtin_ctzll(uint64_t(c->page_size));
    if (c->type == EHIP_CACHE_I8) {
        if (c->head_dim > kMaxDim)
            return fail(EHIP_EINVAL, "%s: heads of %lld values in 8 bits", name,
                        (long long)c->head_dim);
        if (c->pages > 0 && (c->k_scales == nullptr || c->v_scales == nullptr))
            return fail(EHIP_EINVAL, "%s: null scales", name);
        out.k_scales = c->k_scales;
        out.v_scales = c->v_scales;
    }
    return EHIP_OK;
}

// Positions count on past a length by less than that again in 32 bits; pages may repeat in a table,
// so the pool's extent does not bound a length.
constexpr int64_t kMaxLength = int64_t(1) << 30;

inline int check_heads(const char* name, const Cache& c, int64_t heads, int64_t longest) {
    if (c.dim > kMaxDim || heads < 1 || heads % c.kv_heads != 0 || longest < 0)
        return fail(EHIP_EINVAL, "%s: %lld heads over %lld of %lld values, length %lld", name,
                    (long long)heads, (long long)c.kv_heads, (long long)c.dim, (long long)longest);
    if (heads > kMaxBlocks || c.sequences * heads > kMaxBlocks || longest > kMaxLength ||
        c.sequences * ceil_div(longest, kTile) > INT32_MAX)
        return fail(EHIP_EINVAL, "%s: %lld sequences of %lld heads of length %lld are too many",
                    name, (long long)c.sequences, (long long)heads, (long long)longest);
    return EHIP_OK;
}

// Parts of a head, and the bytes of all heads' and of the sequences' first tiles.
inline size_t part_bytes(const Cache& c, int64_t heads, int workers) {
    return size_t(heads) * size_t(workers + c.sequences) *
               (sizeof(float2) + size_t(c.dim) * sizeof(float)) +
           size_t(c.sequences + 1) * sizeof(int);
}

// How the work of a call is cut: by the matrix instructions' kernel, of waves, or the vector one.
struct Cut {
    bool waves;
    int tile, workers;
};

// bf16 and 8 bits, exact in one part, go by the matrix instructions.
inline bool by_waves(int type) { return type != EHIP_CACHE_F32; }
// Rows of whole units at 16 bytes.
inline bool whole_rows(const Cache& c, int values) {
    return c.dim % values == 0 && aligned16(c.k) && aligned16(c.v);
}
// Positions that so many rows of work of at most `longest` are cut by.
inline int tile_of(bool waves, int64_t rows, int64_t longest) {
    return waves && rows * ceil_div(longest, kWaveTile) <= INT32_MAX ? kWaveTile : kTile;
}

// Waves of a row that is joined: one where the rows fill the card, many for few rows of many parts
// (16 rows of 128 parts of 64 values: with the parts 14.3 us by 4 waves, 13.3 by 16; 128 of up to 128
// 16.1 and 15.2; 16 of 16 10.1 and 10.9).
constexpr int kManyJoinWaves = 16;
constexpr int join_threads(int waves) { return waves > kPagedWaves ? 64 * waves : kPagedThreads; }
inline int join_waves(int64_t rows, int64_t parts) {
    if (rows >= 1024) return 1;
    return rows <= 256 && parts >= 64 ? kManyJoinWaves : kPagedWaves;
}

// The cut of the sequences' own positions, and the launch over them (attention_paged.hip).
Cut cut_of(const Cache& c, int64_t heads, int64_t longest, bool waves);
int launch_parts(const Paged& a, int type, bool waves, hipStream_t s);

}  // namespace paged
}  // namespace ehip

#endif  // EHIP_ATTENTION_PAGED_HPP
