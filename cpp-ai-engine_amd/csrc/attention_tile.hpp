// attention_tile.hpp -- the pieces of attention on the matrix instructions: rows of fp32 values in
// three bf16 parts (gemm_split.hpp: 24 bits, six of the nine part products, fp32 sums), in
// registers for the rows that a wave owns and in LDS for the rows that stream past.
//
// v_mfma_f32_32x32x16_bf16, D = A B + C: lane l holds A(l % 32, 8 (l / 32) + 0..7), B(8 (l / 32) +
// 0..7, l % 32) and D(8 (r / 4) + 4 (l / 32) + r % 4, l % 32) in register r. A wave's own rows are
// the columns of every product, so a lane has one of them throughout: row sums are sums over the
// lane's registers and its partner's (l ^ 32), and a product's D is the next one's B as it stands,
// but for the order of its 16 rows, which the next one's A follows (RowTile::columns).
#ifndef EHIP_ATTENTION_TILE_HPP
#define EHIP_ATTENTION_TILE_HPP

#include "gemm_split.hpp"

namespace ehip {
namespace attention {

using gemm_detail::bf16x8;
using gemm_detail::floatx4u;
using gemm_detail::global_bytes;
using gemm_detail::global_load;
using gemm_detail::split_pair;
using gemm_detail::uintx4;

typedef float floatx16 __attribute__((ext_vector_type(16)));

// The six part products, the smallest first.
constexpr int kPart[6][2] = {{1, 1}, {2, 0}, {0, 2}, {0, 1}, {1, 0}, {0, 0}};

// Eight values in three parts, eight bf16 to a register quadruple. Unlike a product's tile they are
// not scaled: values below 2^-110 lose what is below 2^-133.
__device__ __forceinline__ void split8(const float* x, bf16x8 (&part)[3]) {
    uintx4 h, m, l;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t hj, mj, lj;
        split_pair(x[2 * j], x[2 * j + 1], hj, mj, lj);
        h[j] = hj;
        m[j] = mj;
        l[j] = lj;
    }
    part[0] = __builtin_bit_cast(bf16x8, h);
    part[1] = __builtin_bit_cast(bf16x8, m);
    part[2] = __builtin_bit_cast(bf16x8, l);
}

// Keeps LDS reads and matrix instructions in the order of the source: the next block's operands are
// asked for before the products of this one, whose six instructions (192 cycles) cover an LDS read.
// Left alone the compiler reads them one or two instructions ahead. Other instructions may cross.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x0216); }

// d += the five smaller part products of two blocks of 32 x 16, or the first parts' alone. The
// matrix instruction drops the low bits of its sums towards minus infinity: of a chain of six
// products a block each drops as much as the first parts' do, unless those come last, when the sum
// is still small (scores of 64 values: 4 instructions at full size in place of 24; the outputs'
// error against 64 bits, sequences of 64 to 1537, went down by a fifth, at no cost in time).
__device__ __forceinline__ void multiply_small(floatx16& d, const bf16x8 (&a)[3],
                                               const bf16x8 (&b)[3]) {
#pragma unroll
    for (int q = 0; q < 5; ++q)
        d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[kPart[q][0]], b[kPart[q][1]], d, 0, 0, 0);
}
__device__ __forceinline__ void multiply_first(floatx16& d, const bf16x8& a, const bf16x8& b) {
    d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, d, 0, 0, 0);
}

__device__ __forceinline__ floatx16 zeros() {
    floatx16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}

// Row (of 32) of register r of a lane's D.
__device__ __forceinline__ int row_of(int r) {
    return 8 * (r / 4) + 4 * ((int(threadIdx.x) & 63) / 32) + r % 4;
}

// How a row's `dim` values are read: one by one (fewer than four), four at a time (a multiple of
// four), or four at a time with the row's last four where a group of four passes its end, which are
// put in their places afterwards (heads of 77 values, 25 sequences of 120: backward 314 us one by
// one, 196 clamped, 168 for heads of 80).
enum Reads { kSingle, kFours, kClamped };

// First of the four values that are read for those from d on.
template <int READS>
__device__ __forceinline__ int clamped(int d, int dim) {
    return READS == kClamped ? (d < dim - 4 ? d : dim - 4) : (d < dim ? d : 0);
}
// Those from d on, of the four that were read for them; what is past the row's end is anything.
template <int READS>
__device__ __forceinline__ void in_place(float* x, int d, int dim) {
    if (READS != kClamped) return;
    const int over = d + 4 - dim;
    const float x1 = x[1], x2 = x[2], x3 = x[3];
    if (over == 1) x[0] = x1, x[1] = x2, x[2] = x3;
    if (over == 2) x[0] = x2, x[1] = x3;
    if (over == 3) x[0] = x3;
}

// The lane's own row (a pointer to its `dim` values) as the B operand of products over the head's
// values: DP / 16 blocks.
template <int DP, int READS>
__device__ __forceinline__ void own_row(const float* row, int dim, float factor,
                                        bf16x8 (&b)[DP / 16][3]) {
    const int half = (int(threadIdx.x) & 63) / 32;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int d0 = 16 * ks + 8 * half;
        float x[8];
        if (READS != kSingle) {
#pragma unroll
            for (int g = 0; g < 8; g += 4) {
                const int d = d0 + g;
                const floatx4u u =
                    *reinterpret_cast<const floatx4u*>(row + clamped<READS>(d, dim));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[g + j] = u[j];
                in_place<READS>(x + g, d, dim);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    x[g + j] = d + (READS == kFours ? 0 : j) < dim ? x[g + j] * factor : 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = d0 + j < dim;
                const float v = row[in ? d0 + j : 0];
                x[j] = in ? v * factor : 0.0f;
            }
        }
        split8(x, b[ks]);
    }
}

// The product of the lane's own rows of two tensors, each of the two lanes that hold it over half
// of the values.
template <int DP, int READS>
__device__ __forceinline__ float own_dot(const float* x, const float* y, int dim) {
    const int half = (int(threadIdx.x) & 63) / 32;
    float s = 0.0f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int d0 = 16 * ks + 8 * half;
        if (READS == kFours) {
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                if (d0 + j >= dim) continue;
                const floatx4u u = *reinterpret_cast<const floatx4u*>(x + d0 + j);
                const floatx4u v = *reinterpret_cast<const floatx4u*>(y + d0 + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = __builtin_fmaf(u[e], v[e], s);
            }
        } else if (READS == kClamped) {
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const int d = d0 + j, first = clamped<READS>(d, dim);
                const floatx4u u = *reinterpret_cast<const floatx4u*>(x + first);
                const floatx4u v = *reinterpret_cast<const floatx4u*>(y + first);
#pragma unroll
                for (int e = 0; e < 4; ++e)  // of those before d another group has the products
                    if (first + e >= d) s = __builtin_fmaf(u[e], v[e], s);
            }
        } else {
            for (int j = 0; j < 8; ++j)
                if (d0 + j < dim) s = __builtin_fmaf(x[d0 + j], y[d0 + j], s);
        }
    }
    return s + __shfl_xor(s, 32);
}

// Block db (32 values) of the lane's own row of a result, held as a D.
template <int READS>
__device__ __forceinline__ void store_own(float* row, int dim, int db, const floatx16& x) {
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const int d = 32 * db + row_of(r);
        if (READS == kFours ? d < dim : READS == kClamped && d + 4 <= dim) {
            *reinterpret_cast<floatx4u*>(row + d) = floatx4u{x[r], x[r + 1], x[r + 2], x[r + 3]};
        } else if (READS != kFours) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < dim) row[d + e] = x[r + e];
        }
    }
}

// ROWS streamed rows as the A operand of products over the head's values: LDS in three planes, each
// in blocks of 32 rows x 16 values as the instruction takes them, 1 KiB, 16 bytes a lane: a
// conflict-free ds_read_b128. The row's place within its half block is permuted by its group of
// eight values, so that a transposed read's eight rows of two groups fall on all banks, twice, and
// the writes of a row's groups, which neighbouring threads hold, on no bank more than twice either;
// few address bits depend on the lane and the block both, so few addresses are kept. A thread
// stages up to kUnits units of one row by 8 values.
template <int ROWS, int DP, int THREADS, int READS>
struct RowTile {
    static constexpr int kGroups = DP / 8;
    static constexpr int kUnits = (ROWS * kGroups + THREADS - 1) / THREADS;
    static constexpr int kPlane = ROWS * DP * 2;
    static constexpr int kBytes = 3 * kPlane;
    static_assert(ROWS % 32 == 0 && DP % 32 == 0, "tile shape");

    float v[kUnits][8];
    uint32_t o[kUnits];  // byte offsets of the units from the tile's first row

    __device__ __forceinline__ static int row(int u) {
        return (int(threadIdx.x) + u * THREADS) / kGroups;
    }
    __device__ __forceinline__ static int group(int u) {
        return (int(threadIdx.x) + u * THREADS) % kGroups;
    }
    __device__ __forceinline__ static int slot(int r, int g) {
        const int place = (r & 7) | (r >> 4 & 1) << 3 | (r >> 3 & 1) << 4;
        return ((r / 32) * (DP / 16) + g / 2) * 1024 + (g & 1) * 512 +
               ((place ^ (g & 3) ^ (g & 1) << 3) << 4);
    }
    // Rows are ld floats apart, at most kMaxLd: offsets within a tile are below 2^31.
    __device__ __forceinline__ RowTile(int ld, int dim) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int r = row(u) < ROWS ? row(u) : 0, d = 8 * group(u);
            o[u] = 4u * uint32_t(r * ld + clamped<READS>(d, dim));
        }
    }
    // The first `left` rows from `base` (left >= 1; rows past them repeat the last).
    __device__ __forceinline__ void load(const float* base, int ld, int left, int dim) {
        const auto at = (global_bytes)base;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (READS != kSingle) {
                const int d = 8 * group(u);
                uint32_t from = o[u];
                if (left < ROWS) {
                    const int r = row(u) < left ? row(u) : left - 1;
                    from = 4u * uint32_t(r * ld + clamped<READS>(d, dim));
                }
                const floatx4u x = global_load<floatx4u>(at + from);
                const uint32_t next =
                    READS == kFours
                        ? (d + 4 < dim ? 16 : 0)
                        : 4u * uint32_t(clamped<READS>(d + 4, dim) - clamped<READS>(d, dim));
                const floatx4u y = global_load<floatx4u>(at + from + next);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[u][j] = x[j];
                    v[u][4 + j] = y[j];
                }
            } else {
                const int r = row(u) < left ? row(u) : left - 1, d = 8 * group(u);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[u][j] = global_load<float>(
                        at + 4u * uint32_t(r * ld + (d + j < dim ? d + j : 0)));
            }
        }
    }
    // CLEAN: every row and value of the tile is there.
    template <bool CLEAN>
    __device__ __forceinline__ void store_as(char* lds, int left, int dim) const {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if ((u + 1) * THREADS > ROWS * kGroups && row(u) >= ROWS) continue;  // no unit
            const bool in = row(u) < left;
            const int d = 8 * group(u);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = v[u][j];
            in_place<READS>(x, d, dim);
            in_place<READS>(x + 4, d + 4, dim);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[j] = CLEAN || (in && d + (READS == kFours ? j & 4 : j) < dim) ? x[j] : 0.0f;
            bf16x8 part[3];
            split8(x, part);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<bf16x8*>(lds + p * kPlane + slot(row(u), group(u))) = part[p];
        }
    }
    __device__ __forceinline__ void store(char* lds, int left, int dim) const {
        if (left >= ROWS && dim == DP) store_as<true>(lds, left, dim);
        else store_as<false>(lds, left, dim);
    }
    // Part p of the transposed block (db, t): values 32 db .. of rows 16 t .., as the A operand of
    // products over the rows, the rows in the order that registers 8 (t % 2) .. of a D hold them:
    // half h of the lanes has rows 16 t + 4 h + {0..3, 8..11}. A transposed read gives sixteen
    // lanes one value each of four rows from the sixteen places of four values that they name.
    __device__ __forceinline__ static bf16x8 columns(const char* lds, int db, int t, int p) {
        typedef short shortx4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) shortx4* Rows;
        const int lane = int(threadIdx.x) & 63, i = lane & 15;
        const int r = 16 * t + 4 * (lane / 32) + i / 4;
        const int g = 4 * db + 2 * (lane / 16 % 2) + i % 4 / 2;
        const char* at = lds + p * kPlane + slot(r, g) + 8 * (i & 1);
        struct {
            shortx4 x, y;
        } f = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((Rows)at),
               __builtin_amdgcn_ds_read_tr16_b64_v4i16((Rows)(at + 256))};  // 8 rows on
        return __builtin_bit_cast(bf16x8, f);
    }
    // Part p of block (rb, ks) of the tile.
    __device__ __forceinline__ static bf16x8 block(const char* lds, int rb, int ks, int p) {
        const int lane = int(threadIdx.x) & 63;
        return *reinterpret_cast<const bf16x8*>(
            lds + slot(32 * rb + (lane & 31), 2 * ks + lane / 32) + p * kPlane);
    }
};

// s[b] = rows 32 b .. of the tile times the lane's own row: NB x 32 scores. fetch(ks) is called
// before own[ks] is used whole.
template <class Tile, int NB, int KS, class Fetch>
__device__ __forceinline__ void scores(floatx16 (&s)[NB], const char* lds, bf16x8 (&own)[KS][3],
                                       Fetch fetch) {
    constexpr int N = NB * KS;
    bf16x8 f[2][3];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = zeros();
#pragma unroll
    for (int p = 0; p < 3; ++p) f[0][p] = Tile::block(lds, 0, 0, p);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (n % NB == 0) fetch(n / NB);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            if (n + 1 < N) f[(n + 1) & 1][p] = Tile::block(lds, (n + 1) % NB, (n + 1) / NB, p);
            else if (p < N) f[N & 1][p] = Tile::block(lds, p % NB, p / NB, 0);
        }
        keep_order();
        multiply_small(s[n % NB], f[n & 1], own[n / NB]);
        keep_order();
    }
    // The first parts once more, three blocks ahead.
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int at = 3 * (N & 1) + n, ahead = at + 3;
        if (n + 3 < N)
            f[ahead / 3 % 2][ahead % 3] = Tile::block(lds, (n + 3) % NB, (n + 3) / NB, 0);
        keep_order();
        multiply_first(s[n % NB], f[at / 3 % 2][at % 3], own[n / NB][0]);
        keep_order();
    }
}

// For blocks first .. first + count - 1 (at most DB) of values: add(block - first, the tile's
// transposed block times the weights w of its rows, 16 NU of them).
template <class Tile, int DB, int NU, class Add>
__device__ __forceinline__ void weighted(const char* lds, int first, int count,
                                         const bf16x8 (&w)[NU][3], Add add) {
    bf16x8 h[NU], f[2][2];  // first parts, the others
    const auto ask = [&](int n) {
        const int db = n / NU, u = n % NU;
        h[u] = Tile::columns(lds, first + db, u, 0);
#pragma unroll
        for (int p = 1; p < 3; ++p) f[n & 1][p - 1] = Tile::columns(lds, first + db, u, p);
    };
    if (count > 0) ask(0);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
        if (db >= count) break;
        floatx16 x = zeros();
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int n = db * NU + u;
            if (u + 1 < NU) ask(n + 1);
            keep_order();
            const bf16x8 a[3] = {h[u], f[n & 1][0], f[n & 1][1]};
            multiply_small(x, a, w[u]);
            keep_order();
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            multiply_first(x, h[u], w[u][0]);
            if (u == 0 && db + 1 < DB) {  // its h is free now
                keep_order();
                if (db + 1 < count) ask((db + 1) * NU);
                keep_order();
            }
        }
        add(db, x);
    }
}

}  // namespace attention
}  // namespace ehip

#endif  // EHIP_ATTENTION_TILE_HPP
