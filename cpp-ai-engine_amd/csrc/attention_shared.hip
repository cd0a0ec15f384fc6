// attention_shared.hip -- attention of one new token per sequence over the paged cache where the
// sequences of a group share their first positions (answers to one prompt): those are passed once
// for the group, by all of its sequences' query heads together, each sequence's own after them, and
// the parts of both joined.

#include "attention_paged.hpp"

namespace ehip {

using namespace paged;

namespace {

using attention::bf16x8;
using attention::floatx4u;
using attention::keep_order;
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- many rows

// A thread's values of a row that is staged, in up to three bf16 parts of eight each.
template <class T, int DP, bool WIDE>
struct Staged {  // bf16 and 8 bits, exact in one part
    static constexpr int kParts = 1;
    static constexpr int N = sizeof(T) == 1 && DP > 64 ? 16 : 8;
    Piece<T, N, WIDE> x;
    __device__ __forceinline__ void load(const T* row, int d0, int dim) { x.load(row, d0, dim); }
    // in: a position that is there; others are nothing, whatever was read.
    __device__ __forceinline__ void parts(int i, int d0, int dim, bool in, bf16x8 (&p)[1]) const {
        uintx4 y = x.bf16(i, d0, dim);
        if (sizeof(T) == 2 && (!in || d0 + 8 * i >= dim)) y = uintx4{0, 0, 0, 0};
        p[0] = __builtin_bit_cast(bf16x8, y);
    }
};
template <int DP, bool WIDE>
struct Staged<float, DP, WIDE> {
    static constexpr int kParts = 3;
    static constexpr int N = 8;
    float x[8];
    __device__ __forceinline__ void load(const float* row, int d0, int dim) {
#pragma unroll
        for (int g = 0; g < 8; g += 4) {
            const int d = d0 + g;
            if (WIDE) {
                const floatx4u y = *reinterpret_cast<const floatx4u*>(row + (d < dim ? d : 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[g + e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[g + e] = row[d + e < dim ? d + e : 0];
            }
        }
    }
    __device__ __forceinline__ void parts(int, int d0, int dim, bool in, bf16x8 (&p)[3]) const {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = in && d0 + e < dim ? x[e] : 0.0f;
        attention::split8(y, p);
    }
};

// d0, d1 += the products of a block each of K or V in its parts with one of q or the weights in
// three, but for the first parts', which go into a sum of their own: the matrix instruction drops
// the low bits of its sums, least where they are small. Two chains at a time, as a product waits for
// the one before.
template <int PARTS>
__device__ __forceinline__ void multiply_small(floatx4& d0, const bf16x8 (&x0)[PARTS], floatx4& d1,
                                               const bf16x8 (&x1)[PARTS], const bf16x8 (&y0)[3],
                                               const bf16x8 (&y1)[3]) {
    using attention::kPart;
#pragma unroll
    for (int i = 0; i < (PARTS == 3 ? 5 : 2); ++i) {
        const int a = PARTS == 3 ? kPart[i][0] : 0, b = PARTS == 3 ? kPart[i][1] : 2 - i;
        d0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x0[a], y0[b], d0, 0, 0, 0);
        d1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x1[a], y1[b], d1, 0, 0, 0);
    }
}

// The shared positions of groups with many rows: a block takes 64 of them, 16 a wave in its registers
// as in part_by_waves, and stages 32 positions at a time for all in LDS. So the cache is read, and
// made bf16, once for 64 rows in place of 16. K lies in blocks of 16 positions by 32 values as the
// instruction takes them, 1 KiB, the positions' places permuted by the values' so that neighbouring
// threads write to different banks; V in rows as there. Of 256 rows over 30000 positions, 8 key heads
// of 128 values in 8 bits, 130 us: 230 TFLOP/s of the 470 that three products for one leave; matrix
// instructions take 35 % of the time and vector ones half of it, with two waves a SIMD.
constexpr int kKeys = 32;  // positions of a step
// Rows that are formed a second time together. Four want registers of the tiles (32 heads over 8 of 128, us:
// 8 groups of up to 16 over up to 6000 positions in bf16, two 64.6, four 65.6; 64 over 30000 in 8 bits
// 128 and 130; 64 over 16000, heads of 100, 91 and 94; an infinity in the first value, 2 groups of 32
// over 4000 in 8 bits, 407 and 344).
constexpr int kSharedAgain = 2;

template <class T, int DP>
struct alignas(16) RowsLds {
    static constexpr int kParts = Staged<T, DP, true>::kParts, kBuffers = kParts == 1 ? 2 : 1;
    static constexpr int kKeyPlane = kKeys * DP * 2, kValuePlane = kKeys * value_pitch(DP);
    char tile[kBuffers][kParts * (kKeyPlane + kValuePlane)];
    float scales[kBuffers][2][kKeys];
};

template <class T, int DP, bool WIDE>
__device__ __forceinline__ void part_by_rows(const Paged& a, uint32_t block,
                                             RowsLds<T, DP>& lds) {
    using Unit = Staged<T, DP, WIDE>;
    using Lds = RowsLds<T, DP>;
    constexpr bool kScaled = sizeof(T) == 1;
    constexpr int kParts = Unit::kParts, N = Unit::N, KS = DP / 32, NV = DP / 16;
    constexpr int kPieces = DP / N, kUnits = kKeys * kPieces / kPagedThreads;
    constexpr int kBuffers = Lds::kBuffers, kPitch = value_pitch(DP);
    constexpr int kKeyPlane = Lds::kKeyPlane, kValuePlane = Lds::kValuePlane;
    static_assert(kKeys * kPieces % kPagedThreads == 0, "whole units");
    static_assert(!kScaled || kUnits == 1, "a thread has one position's scale");
    const int lane = int(threadIdx.x) & 63, col = lane & 15, quarter = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int dim = int(a.c.dim), kv_heads = int(a.c.kv_heads);
    const int kv = int(block % uint32_t(kv_heads));
    const int worker = int(block / uint32_t(kv_heads));
    const T* const k = static_cast<const T*>(a.c.k) + int64_t(kv) * dim;
    const T* const v = static_cast<const T*>(a.c.v) + int64_t(kv) * dim;
    const uint32_t pitch = uint32_t(kv_heads * dim);
    const float c2 = a.scale * 1.44269504088896340736f;
    Items among;
    for (Segment seg = first_segment<true>(a, block, worker, among); seg.t < seg.t_end;
         next_segment<true>(a, seg, among)) {
        const int64_t s = seg.s;
        const int begin = seg.begin, end = seg.end;
        const int count = rows_of<true>(a, seg, 0);
        const int mine = 16 * wave + col;  // the lane's row
        const bool some = 16 * wave < count;
        bool bad = false;  // a page outside the pool

        // The table's entries of the thread's units, asked for a step before their rows are read,
        // past the end the last again.
        Entry entry[kUnits];
        uint32_t row[kUnits];
        int64_t place = 0;
        Unit kx[kUnits], vx[kUnits];
        float scale = 0.0f;
        const auto ask = [&](int p0) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int j = (int(threadIdx.x) + u * kPagedThreads) / kPieces;
                entry[u] = entry_of(a.c, s, uint32_t(min(p0 + j, end - 1)));
            }
        };
        const auto find = [&] {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                int64_t r = row_of_entry(a.c, entry[u]);
                if (r < 0) {
                    bad = true;
                    r = 0;
                }
                row[u] = uint32_t(r);
            }
            // Of its position's piece 0 a thread has the key's scale too, of piece 1 the value's.
            if constexpr (kScaled)
                place = scale_of(a.c, row[0], row[0] != 0 ? entry[0].off : 0, kv);
        };
        const auto load = [&](int p0) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int d0 = (int(threadIdx.x) + u * kPagedThreads) % kPieces * N;
                kx[u].load(k + uint64_t(row[u]) * pitch, d0, dim);
                vx[u].load(v + uint64_t(row[u]) * pitch, d0, dim);
            }
            if constexpr (kScaled) {
                const float* const from =
                    int(threadIdx.x) % kPieces == 0 ? a.c.k_scales : a.c.v_scales;
                scale = p0 + int(threadIdx.x) / kPieces < end ? from[place] : 0.0f;
            }
        };
        const auto store = [&](int p0, char* to, float (*scales)[kKeys]) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int unit = int(threadIdx.x) + u * kPagedThreads;
                const int j = unit / kPieces, d0 = unit % kPieces * N;
                const bool in = p0 + j < end;
#pragma unroll
                for (int i = 0; i < N / 8; ++i) {
                    const int g = d0 / 8 + i;
                    char* const at = to + (j / 16 * KS + g / 4) * 1024 + (g % 4) * 256 +
                                     ((j % 16) ^ (g % 16)) * 16;
                    bf16x8 part[kParts];
                    kx[u].parts(i, d0, dim, in, part);
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
                        *reinterpret_cast<bf16x8*>(at + p * kKeyPlane) = part[p];
                    vx[u].parts(i, d0, dim, in, part);
#pragma unroll
                    for (int p = 0; p < kParts; ++p)
                        *reinterpret_cast<bf16x8*>(to + kParts * kKeyPlane + p * kValuePlane +
                                                   j * kPitch + 16 * g) = part[p];
                }
            }
            if constexpr (kScaled)
                if (int(threadIdx.x) % kPieces < 2)
                    scales[int(threadIdx.x) % kPieces][int(threadIdx.x) / kPieces] = scale;
        };
        ask(begin);
        bf16x8 q[KS][3];
        uint64_t apart = 0;  // rows for the formula
        {
            const float* const from = query_row<true>(a, seg, kv, 0, mine < count ? mine : 0);
            float y[KS][8];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (!WIDE) {
                    ask_eight(from, 32 * ks + 8 * quarter, dim, y[ks]);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {  // a head is a multiple of four values
                    const int d0 = 32 * ks + 8 * quarter + e / 4 * 4;
                    y[ks][e] = from[(d0 < dim ? d0 : 0) + e % 4];
                }
            }
            find();
            load(begin);
            ask(begin + kKeys);
            float largest = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (!WIDE) eight_in_place(y[ks], 32 * ks + 8 * quarter, dim);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = 32 * ks + 8 * quarter + e;
                    y[ks][e] = d < dim && mine < count ? y[ks][e] : 0.0f;
                    largest = fmaxf(largest, fabsf(y[ks][e]));
                }
            }
            apart = __ballot(out_of_parts<T>(largest_of_rows(largest) * fabsf(c2)));
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[ks][e] *= c2;
                attention::split8(y[ks], q[ks]);
            }
        }
        floatx4 o[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        store(begin, lds.tile[0], lds.scales[0]);
        int buffer = 0;
        __syncthreads();
        for (int p0 = begin; p0 < end; p0 += kKeys) {
            find();
            load(p0 + kKeys);
            ask(p0 + 2 * kKeys);
            if (some) {
                const char* const keys = lds.tile[buffer];
                const char* const values = keys + kParts * kKeyPlane;
                const auto scales = [&](int which, int t) {  // of a lane's scores
                    return *reinterpret_cast<const floatx4*>(
                        &lds.scales[buffer][which][16 * t + 4 * quarter]);
                };
                floatx4 sc[2], small[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[t] = small[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                // LDS is read a block ahead of the products.
                bf16x8 f[2][2][kParts];
                const auto ask_keys = [&](int ks) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const char* const at = keys + (t * KS + ks) * 1024 + quarter * 256 +
                                               (col ^ (4 * ks + quarter) % 16) * 16;
#pragma unroll
                        for (int p = 0; p < kParts; ++p)
                            f[ks & 1][t][p] =
                                *reinterpret_cast<const bf16x8*>(at + p * kKeyPlane);
                    }
                };
                ask_keys(0);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (ks + 1 < KS) ask_keys(ks + 1);
                    keep_order();
                    multiply_small<kParts>(small[0], f[ks & 1][0], small[1], f[ks & 1][1], q[ks],
                                           q[ks]);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[ks & 1][t][0], q[ks][0],
                                                                        sc[t], 0, 0, 0);
                    keep_order();
                }
                float w[8], top = m;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    sc[t] += small[t];
                    if constexpr (kScaled) sc[t] *= scales(0, t);
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[4 * t + r] = sc[t][r];
                }
                if (p0 + kKeys > end) {
                    asm volatile("");  // a branch: as selects in every step, 16 instructions
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (p0 + 16 * (j / 4) + 4 * quarter + j % 4 >= end) w[j] = -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, w[j]);
                top = largest_of_rows(top);
                const float shift = top == -INFINITY ? 0.0f : top;
                const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - shift);
                m = top;
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = __builtin_amdgcn_exp2f(w[j] - shift);
                    sum += w[j];
                }
                l = __builtin_fmaf(l, keep, sum);
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
                // Two blocks of 16 values at a time.
                const auto ask_values = [&](int i) {
                    typedef __attribute__((address_space(3))) shortx4* Rows;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            const char* const from = values + part * kValuePlane +
                                                     (4 * quarter + col / 4) * kPitch +
                                                     32 * (i + t) + 8 * (col % 4);
                            struct {
                                shortx4 x, y;
                            } g = {
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((Rows)from),
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((Rows)(from + 16 * kPitch))};
                            f[i / 2 & 1][t][part] = __builtin_bit_cast(bf16x8, g);
                        }
                };
                ask_values(0);
                if (kBuffers > 1) store(p0 + kKeys, lds.tile[buffer ^ 1], lds.scales[buffer ^ 1]);
                floatx4 y[2][2];
                const auto sum_up = [&](int i) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            o[i + t][r] = __builtin_fmaf(o[i + t][r], keep, y[i / 2 & 1][t][r]);
                };
#pragma unroll
                for (int i = 0; i < NV; i += 2) {
                    if (i + 2 < NV) ask_values(i + 2);
                    keep_order();
                    auto& x = f[i / 2 & 1];
                    auto& z = y[i / 2 & 1];
#pragma unroll
                    for (int t = 0; t < 2; ++t) z[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                    multiply_small<kParts>(z[0], x[0], z[1], x[1], p, p);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        z[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[t][0], p[0], z[t], 0, 0,
                                                                       0);
                    if (i > 0) sum_up(i - 2);  // while these products are formed
                    keep_order();
                }
                sum_up(NV - 2);
            } else if (kBuffers > 1) {
                store(p0 + kKeys, lds.tile[buffer ^ 1], lds.scales[buffer ^ 1]);
            }
            if (kBuffers == 1) {
                __syncthreads();  // all have read
                store(p0 + kKeys, lds.tile[0], lds.scales[0]);
            } else {
                buffer ^= 1;
            }
            __syncthreads();
        }
        // The lane's row, values 16 i + 4 quarter + r; rows whose sums are not finite by the formula.
        bad = __syncthreads_or(bad);
        l = with_half(with_row_pair(l));
        bool fine = l > 0.0f && l < INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) fine = fine && fabsf(o[i][r]) < INFINITY;
        const uint64_t lanes = __ballot(!fine && mine < count) | apart;
        uint32_t again = uint32_t(lanes | lanes >> 32);
        again = (again | again >> 16) & 0xffffu;
        again = __builtin_amdgcn_readfirstlane(bad ? 0u : again);
        const int64_t part0 = part_of<true>(a, seg, worker, kv, 0, 0);
        if (mine < count && !(again >> col & 1)) {
            const int64_t at = part0 + mine;
            if (quarter == 0) a.part_stats[at] = float2{m, bad ? NAN : l * 0x1p-24f};
            float* const to = a.part_out + at * dim;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int d = 16 * i + 4 * quarter;
                floatx4u y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = o[i][r] * 0x1p-24f;  // as the other parts
                if (d + 4 <= dim) {
                    *reinterpret_cast<floatx4u*>(to + d) = y;
                } else {
#pragma unroll
                    for (int r = 0; r < 3; ++r)
                        if (d + r < dim) to[d + r] = y[r];
                }
            }
        }
        while (again != 0) {
            const Again<kSharedAgain> next(again);
            const float* rows[kSharedAgain];
#pragma unroll
            for (int i = 0; i < kSharedAgain; ++i)
                rows[i] = query_row<true>(a, seg, kv, 0, 16 * wave + next.row[i]);
            float top[kSharedAgain], sum[kSharedAgain], y[kSharedAgain][2];
            part_by_formula<T, DP, kSharedAgain>(a, s, rows, kv, begin, end, top, sum, y);
#pragma unroll
            for (int i = 0; i < kSharedAgain; ++i) {
                const int64_t at = part0 + 16 * wave + next.row[i];
                if (i < next.count && lane == 0) a.part_stats[at] = float2{top[i], sum[i]};
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (i < next.count && lane + 64 * e < dim)
                        a.part_out[at * dim + lane + 64 * e] = y[i][e];
            }
        }
    }
}

// The shared positions' parts, after those of the sequences' own: one launch, whose blocks of the one
// kind begin where blocks of the other end. ROWS: part_by_rows. (8 groups of up to 64 rows over up to
// 6000 shared positions and 1024 own ones, 32 heads over 8 of 128, bf16: 171 MB in 52 us, 3.3 TB/s.)
// bf16 heads of up to 64 are held to three waves a SIMD, a register or two below what they take (8 groups
// of 16 over 4000, 32 heads over 8 of 64: 46.5 us, two waves 48.7; one of 64 over 16000 62.1, 60.2; 8 bits
// have three as they are).
template <class T, int DP, bool WIDE, bool ROWS>
__global__ __launch_bounds__(kPagedThreads, sizeof(T) == 2 && DP <= 64 && WIDE ? 3 : 2) void
shared_parts(Paged own, Paged a, uint32_t own_blocks) {
    __shared__ union Lds {
        PartLds<DP> part;
        RowsLds<T, DP> rows;
    } lds;
    if (blockIdx.x < own_blocks)
        part_by_waves<T, DP, WIDE, false, kSharedAgain>(own, blockIdx.x, lds.part);
    else if constexpr (ROWS)
        part_by_rows<T, DP, WIDE>(a, blockIdx.x - own_blocks, lds.rows);
    else
        part_by_waves<T, DP, WIDE, true, kSharedAgain>(a, blockIdx.x - own_blocks, lds.part);
}

// Apart where the own positions go by the vector kernel.
template <class T, int DP, bool WIDE>
__global__ __launch_bounds__(kPagedThreads, 2) void shared_rows(Paged a) {
    __shared__ RowsLds<T, DP> lds;
    part_by_rows<T, DP, WIDE>(a, blockIdx.x, lds);
}

// --------------------------------------------------------------------- join

constexpr int kPlanThreads = 1024;

// The last group that begins at sequence s or before.
__device__ __forceinline__ int group_of(const int* cu, int groups, int s) {
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cu[mid] <= s) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The parts of rows, of their own and of the group's positions, where the row is not one part of its
// own.
template <int WAVES>
__global__ __launch_bounds__(kPagedThreads) void shared_join(Paged own, Paged a,
                                                             const int* __restrict__ group) {
    __shared__ float sh[WAVES][kMaxDim + 1];
    const int64_t at =
        int64_t(blockIdx.x) * (kPagedWaves / WAVES) + int(threadIdx.x) / (64 * WAVES);
    if (at >= a.c.sequences * a.heads) return;
    const int64_t s = at / a.heads;
    const Own x = own_of(own, s);
    const int g = group[s], group_rows = a.heads / int(a.c.kv_heads);
    const int h = int(at % a.heads), n = length_from(own, x.length);
    if (n <= 0) {
        empty_row<WAVES>(a, s, h, n);
        return;
    }
    Parts p[2] = {own_parts(own, x, s, h), Parts{nullptr, nullptr, 0, 1}};
    if (x.start == 0 && p[0].count == 1) return;  // the sequence was one segment
    if (x.start > 0) {
        const int kv = h / group_rows;
        const int row = int(s - group_begin(a, g)) * group_rows + h % group_rows;
        const int tile = row / a.rows, each = tiles_of(a, shared_of(a, g));
        const int tiles = a.first[a.groups], t0 = a.first[g] + tile * each;
        const int w0 = worker_of(a, t0, tiles);
        const int place = w0 + row_tile_base(a, g) + tile;
        const int64_t from = (int64_t(kv) * a.places + place) * a.rows + row % a.rows;
        p[1] = Parts{a.part_stats + from, a.part_out + from * a.c.dim,
                     worker_of(a, t0 + each - 1, tiles) - w0 + 1, a.rows};
    }
    join_parts<WAVES>(a, s, h, p, sh);
}

// One block. The groups' offsets, in range and ascending whatever came in; what each shares, nothing
// where it has no two sequences or the number is none that its table row could have; the sequences'
// first own positions, 0 for those of no group or shorter than what theirs shares, and their groups.
__global__ __launch_bounds__(kPlanThreads) void shared_plan(Paged a, const int32_t* group_cu,
                                                            const int32_t* shared,
                                                            int longest_shared, int* cu,
                                                            int* counts, int* starts,
                                                            int* group) {
    __shared__ int sh[kPlanThreads / 64];
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) / 64;
    const int sequences = int(a.c.sequences);
    int before = 0;  // the largest offset so far
    for (int base = 0; base <= a.groups; base += kPlanThreads) {
        const int g = base + int(threadIdx.x);
        int x = g <= a.groups ? min(max(group_cu[g], 0), sequences) : 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int y = __shfl_up(x, d);
            x = lane >= d ? max(x, y) : x;
        }
        if (lane == 63) sh[wave] = x;
        __syncthreads();
        x = max(x, before);
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) x = max(x, sh[w]);
            before = max(before, sh[w]);
        }
        if (g <= a.groups) cu[g] = x;
        __syncthreads();
    }
    for (int g = int(threadIdx.x); g < a.groups; g += kPlanThreads) {
        const int n = shared[g];
        const bool fits = n > 0 && n <= longest_shared && n <= a.c.width * a.c.page_size;
        counts[g] = fits && a.c.pages > 0 && cu[g + 1] - cu[g] > 1 ? n : 0;
    }
    __syncthreads();
    for (int s = int(threadIdx.x); s < sequences; s += kPlanThreads) {
        int start = 0, g = 0;
        if (a.groups > 0) {
            g = group_of(cu, a.groups, s);
            if (cu[g] <= s && s < cu[g + 1] && length_of(a, s) >= counts[g]) start = counts[g];
        }
        starts[s] = start;
        group[s] = g;
    }
}

// ---------------------------------------------------------------- host checks

int check_groups(const char* name, const Cache& c, int64_t heads, int64_t groups,
                 int64_t longest_shared) {
    if (groups < 0 || groups > kMaxBlocks || longest_shared < 0 || longest_shared > kMaxLength)
        return fail(EHIP_EINVAL, "%s: %lld groups that share %lld positions", name,
                    (long long)groups, (long long)longest_shared);
    const int64_t rows = c.sequences * (heads / c.kv_heads);
    if ((rows + groups) * ceil_div(longest_shared, kTile) > INT32_MAX)
        return fail(EHIP_EINVAL, "%s: %lld sequences of %lld heads that share %lld positions are "
                                 "too many",
                    name, (long long)c.sequences, (long long)heads, (long long)longest_shared);
    return EHIP_OK;
}

// Whether part_by_rows passes the shared positions: else, of groups of up to 32 rows in the mean, do
// waves of their own (8 groups of 4000 shared positions and 100 own ones, 32 heads over 8 of 128,
// us, waves : rows, for 8, 16, 32 and 64 rows; 8 bits 38 : 49, 42 : 48, 52 : 57, 73 : 64; bf16 41 :
// 47, 47 : 48, 57 : 57, 78 : 67).
bool by_rows(int type, int64_t rows) { return !by_waves(type) || rows > 32; }

struct Plan {
    Cut own, shared;
    bool by_rows;
    int rows, places;
    size_t own_bytes, part_bytes, first_bytes, bytes;
};

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

Plan plan_of(const Cache& c, int type, int64_t heads, int64_t longest, int64_t groups,
             int64_t longest_shared) {
    Plan p{};
    p.own = cut_of(c, heads, longest, by_waves(type));
    const int64_t rows = c.sequences * (heads / c.kv_heads);
    p.by_rows = by_rows(type, groups > 0 ? rows / groups : 0);
    p.rows = p.by_rows ? 64 : 16;
    const int64_t row_tiles = rows / p.rows + groups;
    const bool waves = !p.by_rows;
    const int tile = tile_of(true, row_tiles, longest_shared);
    const int64_t most = std::max<int64_t>(1, row_tiles * ceil_div(longest_shared, tile));
    const int64_t resident = waves ? 2048 : 512;
    p.shared = Cut{waves, tile,
                   int(std::min(most, std::max<int64_t>(1, resident / c.kv_heads)))};
    p.places = int(p.shared.workers + row_tiles + 1);
    p.own_bytes = round16(part_bytes(c, heads, p.own.workers));
    p.part_bytes = round16(size_t(c.kv_heads) * size_t(p.places) * size_t(p.rows) *
                           (sizeof(float2) + size_t(c.dim) * sizeof(float)));
    // The parts of both; the groups' first tiles, offsets and shared positions, and the sequences'
    // own starts and groups.
    p.first_bytes = round16(size_t(groups + 1) * sizeof(int));
    p.bytes = p.own_bytes + p.part_bytes + 3 * p.first_bytes + 2 * size_t(c.sequences) * sizeof(int);
    return p;
}

template <class T, int DP, bool WIDE>
int launch_rows(const Paged& a, hipStream_t s) {
    EHIP_LAUNCH("attention_shared", (shared_rows<T, DP, WIDE>),
                dim3(unsigned(a.workers * a.c.kv_heads)), dim3(kPagedThreads), 0, s, a);
    return EHIP_OK;
}

template <class T, bool WIDE>
int launch_rows_dim(const Paged& a, hipStream_t s) {
    return a.c.dim <= 64 ? launch_rows<T, 64, WIDE>(a, s) : launch_rows<T, 128, WIDE>(a, s);
}

// Where the vector kernel takes the own positions: the shared ones before them.
int launch_apart(const Paged& own, const Paged& a, hipStream_t s) {
    const bool wide = aligned16(a.c.k) && aligned16(a.c.v) && a.c.dim % 4 == 0;
    const int rc = wide ? launch_rows_dim<float, true>(a, s) : launch_rows_dim<float, false>(a, s);
    return rc != EHIP_OK ? rc : launch_parts(own, EHIP_CACHE_F32, false, s);
}

template <class T, int DP, bool WIDE, bool ROWS>
int launch_both(const Paged& own, const Paged& a, hipStream_t s) {
    const int64_t group = a.heads / a.c.kv_heads;
    const int64_t own_blocks =
        ceil_div(own.workers * ceil_div(group, 16) * a.c.kv_heads, kPagedWaves);
    const int64_t units = a.workers * a.c.kv_heads;
    EHIP_LAUNCH("attention_shared", (shared_parts<T, DP, WIDE, ROWS>),
                dim3(unsigned(own_blocks + (ROWS ? units : ceil_div(units, kPagedWaves)))),
                dim3(kPagedThreads), 0, s, own, a, uint32_t(own_blocks));
    return EHIP_OK;
}

template <class T, int DP, bool WIDE>
int launch_kind(const Paged& own, const Paged& a, bool rows, hipStream_t s) {
    return rows ? launch_both<T, DP, WIDE, true>(own, a, s)
                : launch_both<T, DP, WIDE, false>(own, a, s);
}

template <class T, bool WIDE>
int launch_dim(const Paged& own, const Paged& a, bool rows, hipStream_t s) {
    return a.c.dim <= 64 ? launch_kind<T, 64, WIDE>(own, a, rows, s)
                         : launch_kind<T, 128, WIDE>(own, a, rows, s);
}

int launch_shared(const Paged& own, const Paged& a, int type, bool rows, hipStream_t s) {
    if (!by_waves(type)) return launch_apart(own, a, s);
    const bool aligned = aligned16(a.c.k) && aligned16(a.c.v);
    const bool wide = aligned && a.c.dim % (type == EHIP_CACHE_BF16 ? 8 : 16) == 0;
    if (type == EHIP_CACHE_BF16)
        return wide ? launch_dim<Bf16, true>(own, a, rows, s)
                    : launch_dim<Bf16, false>(own, a, rows, s);
    return wide ? launch_dim<Int8, true>(own, a, rows, s) : launch_dim<Int8, false>(own, a, rows, s);
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int64_t ehip_attention_shared_workspace(const ehip_cache_t* cache, int64_t heads, int64_t longest,
                                        int64_t groups, int64_t longest_shared) {
    Cache c;
    if (check("attention_shared", cache, c) || check_heads("attention_shared", c, heads, longest) ||
        check_groups("attention_shared", c, heads, groups, longest_shared))
        return -1;
    return c.sequences == 0
               ? 0
               : int64_t(plan_of(c, cache->type, heads, longest, groups, longest_shared).bytes);
}

int ehip_attention_shared_f32(const ehip_cache_t* cache, const float* q, int64_t ld_q,
                              int64_t heads, const int32_t* lengths, int64_t longest,
                              const int32_t* group_cu, const int32_t* shared, int64_t groups,
                              int64_t longest_shared, float scale, float* out, int64_t ld_out,
                              float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    EHIP_READY();
    Cache c;
    if (int rc = check("attention_shared", cache, c)) return rc;
    if (int rc = check_heads("attention_shared", c, heads, longest)) return rc;
    if (int rc = check_groups("attention_shared", c, heads, groups, longest_shared)) return rc;
    if (ld_q < heads * c.dim || ld_out < heads * c.dim)
        return fail(EHIP_EINVAL, "attention_shared: leading dimension below the row's length");
    if (c.sequences == 0) return EHIP_OK;
    if (q == nullptr || lengths == nullptr || out == nullptr || group_cu == nullptr ||
        (groups > 0 && shared == nullptr))
        return fail(EHIP_EINVAL, "attention_shared: null tensor");
    const Plan p = plan_of(c, cache->type, heads, longest, groups, longest_shared);
    if (workspace == nullptr || workspace_bytes < p.bytes || !aligned16(workspace))
        return fail(EHIP_EINVAL, "attention_shared: needs %zu bytes of 16-byte aligned workspace",
                    p.bytes);
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
    Paged own = a;
    char* at = static_cast<char*>(workspace);
    own.tile = p.own.tile;
    own.workers = p.own.workers;
    const int64_t parts = heads * (own.workers + c.sequences);
    own.part_stats = reinterpret_cast<float2*>(at);
    own.part_out = reinterpret_cast<float*>(own.part_stats + parts);
    own.first = reinterpret_cast<int*>(own.part_out + parts * c.dim);
    at += p.own_bytes;
    a.tile = p.shared.tile;
    a.workers = p.shared.workers;
    a.rows = p.rows;
    a.places = p.places;
    a.groups = int(groups);
    a.part_stats = reinterpret_cast<float2*>(at);
    a.part_out = reinterpret_cast<float*>(a.part_stats + c.kv_heads * int64_t(p.places) * p.rows);
    at += p.part_bytes;
    a.first = reinterpret_cast<int*>(at);
    int* const cu = reinterpret_cast<int*>(at + p.first_bytes);
    int* const counts = reinterpret_cast<int*>(at + 2 * p.first_bytes);
    int* const starts = reinterpret_cast<int*>(at + 3 * p.first_bytes);
    int* const of = starts + c.sequences;
    a.group_cu = cu;
    a.shared = counts;
    own.starts = starts;
    hipStream_t s = as_stream(stream);
    EHIP_LAUNCH("attention_shared_plan", shared_plan, dim3(1), dim3(kPlanThreads), 0, s, a,
                group_cu, shared, int(longest_shared), cu, counts, starts, of);
    if (groups > 0) {
        if (int rc = launch_shared(own, a, cache->type, p.by_rows, s)) return rc;
    } else {
        if (int rc = launch_parts(own, cache->type, p.own.waves, s)) return rc;
    }
    const int64_t rows = c.sequences * heads;
    if (join_waves(rows, 0) == 1)
        EHIP_LAUNCH("attention_shared_join", shared_join<1>,
                    dim3(unsigned(ceil_div(rows, kPagedWaves))), dim3(kPagedThreads), 0, s, own,
                    a, of);
    else
        EHIP_LAUNCH("attention_shared_join", shared_join<kPagedWaves>, dim3(unsigned(rows)),
                    dim3(kPagedThreads), 0, s, own, a, of);
    return EHIP_OK;
}

}  // extern "C"
