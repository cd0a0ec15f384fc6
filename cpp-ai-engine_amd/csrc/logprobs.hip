// logprobs.hip -- log probabilities of given tokens, the entropy of each row's distribution and
// its largest logits, and the gradient of the first two:
//
//   lse = log sum_j exp(x_j), logprob = x_t - lse, H = lse - sum_j p_j x_j, p_j = exp(x_j - lse)
//   dx_j = g_lp ([j = t] - p_j) - g_H p_j (x_j - lse + H)
//
// HBM bounds both directions. A block takes a run of a row's segments, kSegment logits in registers
// at a time, and reads each once: with the running maximum m go the sums of e = exp(x - m) and of
// e (x - m), from which lse = m + log(sum e) and H = log(sum e) - sum e (x - m) / sum e without the
// cancellation of two numbers of lse's size. Rows that are few are cut over several blocks, whose
// results a second launch joins. 8192 rows of 32000: forward 206 us, 5.1 TB/s, backward 344, 6.1.

#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace ehip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kVectors = 8;                           // of four logits, a thread and segment
constexpr int kSegment = kThreads * kVectors * 4;     // logits of a segment
constexpr int kMaxTop = 128;
constexpr float kLog2e = 1.44269504088896340736f;

// Four floats at any float's address.
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

// Maximum, sum of exp(x - m) and sum of exp(x - m) (x - m) of some logits. m = -inf: none but -inf.
struct Sums {
    float m, l, w;
};

// The sums of a about another maximum m >= a.m.
__device__ __forceinline__ Sums about(const Sums& a, float m) {
    const float d = a.m - m;
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    // Of nothing but -inf (l = 0), or too far below m: whatever d is. A NaN stays.
    if (a.l == 0.0f || (f == 0.0f && a.l == a.l)) return Sums{m, 0.0f, 0.0f};
    return Sums{m, a.l * f, f * __builtin_fmaf(a.l, d, a.w)};
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

// The sums of all threads of the block, in each of them. Every thread calls it.
__device__ __forceinline__ Sums block_sums(const Sums& mine, Sums* sh) {
    const float m = wave_max(mine.m);
    Sums a = about(mine, m);
    a.l = wave_sum(a.l);
    a.w = wave_sum(a.w);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x / 64] = a;
    __syncthreads();
    float top = sh[0].m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sh[w].m);
    Sums all{top, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const Sums b = about(sh[w], top);
        all.l += b.l;
        all.w += b.w;
    }
    return all;
}

// A row's results from its sums.
struct RowOut {
    const float* logits;
    int64_t ld;
    const int32_t* targets;
    int64_t vocab;
    float *logprob, *entropy, *lse;
    int top;
    float* top_logprob;
    int32_t* top_index;
};

__device__ __forceinline__ float lse_of(const Sums& a) {
    return a.m == -INFINITY && a.l == 0.0f ? -INFINITY : a.m + logf(a.l);
}

__device__ __forceinline__ void finish_row(const RowOut& o, int64_t r, const Sums& a) {
    const float z = lse_of(a);
    o.lse[r] = z;
    if (o.entropy != nullptr) o.entropy[r] = z == -INFINITY ? 0.0f : logf(a.l) - a.w / a.l;
    if (o.logprob != nullptr) {
        const int64_t t = o.targets[r];
        o.logprob[r] = t < 0 || t >= o.vocab ? NAN
                       : z == -INFINITY      ? -INFINITY
                                             : o.logits[r * o.ld + t] - z;
    }
}

// ------------------------------------------------------------------ the top

// A logit's place in the order (-0 as 0, NaN above all; 0 is none) and, with its index from above
// in the low half, a key that no other of the row has: larger keys come first.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    const uint32_t y = b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
    return x != x ? 0xffffffffu : y;
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t index) {
    return uint64_t(order) << 32 | uint32_t(~index);
}

constexpr int kOffer = 4 * kVectors;  // keys that a thread offers at once

// The largest keys so far, and room for what may join them: all keys of kMaxTop threads.
constexpr int kRoom = kMaxTop * kOffer;
struct Top {
    uint64_t list[kMaxTop];  // in order; 0 where there are fewer
    uint64_t found[kMaxTop + kRoom];
    uint64_t largest[kThreads];
    uint64_t limit;
    uint32_t limits[kWaves];
    int count;
};

__device__ __forceinline__ void clear(Top& sh, int top) {
    for (int i = int(threadIdx.x); i < top; i += kThreads) sh.list[i] = 0;
    __syncthreads();
}

// list = the largest `top` of found[0 .. n), which all differ, 0 after them. Every thread calls it.
__device__ __forceinline__ void list_found(Top& sh, int n, int top) {
    for (int i = int(threadIdx.x); i < top; i += kThreads)
        if (i >= n) sh.list[i] = 0;
    for (int i = int(threadIdx.x); i < n; i += kThreads) {
        const uint64_t k = sh.found[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += sh.found[j] > k;
        if (rank < top) sh.list[rank] = k;  // the order of arrival does not matter
    }
    __syncthreads();
}

// Adds the list to the n found keys, and makes them the list. Every thread calls it.
__device__ __forceinline__ void join_found(Top& sh, int n, int top, bool full) {
    for (int i = int(threadIdx.x); i < top; i += kThreads)
        if (sh.list[i] != 0) sh.found[n + i] = sh.list[i];
    // The list is full from its first batch on, or what is in it was all there is.
    if (full) n += top;
    else
        for (int i = 0; i < top && sh.list[i] != 0; ++i) ++n;
    __syncthreads();
    list_found(sh, n, top);
}

// Takes the kOffer keys key(0) .. of every thread (0: none; all others differ from each other and
// from the list's) into the list of the `top` largest. Every thread calls it.
template <class Key>
__device__ __forceinline__ void offer(Top& sh, int top, Key key) {
    const uint64_t last = sh.list[top - 1];
    uint64_t largest = 0;
#pragma unroll
    for (int i = 0; i < kOffer; ++i) {
        const uint64_t k = key(i);
        largest = k > largest ? k : largest;
    }
    if (threadIdx.x == 0) sh.count = 0;
    const int threads = __syncthreads_count(largest > last);
    if (threads == 0) return;
    // At most `top` threads hold keys of the new list. Where more of them have one above the last:
    // the `top`-th of the threads' largest is a lower limit of the list, and as many threads reach
    // it.
    uint64_t limit = 0;
    if (threads > top) {
        // The wave's order first: only its first `top` can be among the block's.
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < 64; ++i) {
            const uint64_t other =
                uint64_t(uint32_t(__builtin_amdgcn_readlane(int(largest >> 32), i))) << 32 |
                uint32_t(__builtin_amdgcn_readlane(int(uint32_t(largest)), i));
            rank += other > largest;
        }
        const int each = top < 64 ? top : 64;
        const bool mine = rank < each && largest != 0;
        sh.largest[threadIdx.x] = 0;
        __syncthreads();
        if (mine) sh.largest[int(threadIdx.x) / 64 * each + rank] = largest;
        __syncthreads();
        if (mine) {
            rank = 0;
#pragma unroll 4
            for (int i = 0; i < kWaves * each; ++i) rank += sh.largest[i] > largest;
            if (rank == top - 1) sh.limit = largest;
        }
        __syncthreads();
        limit = sh.limit;
    }
    if (largest > last && largest >= limit) {
#pragma unroll
        for (int i = 0; i < kOffer; ++i) {
            const uint64_t k = key(i);
            if (k > last && k >= limit) sh.found[atomicAdd(&sh.count, 1)] = k;
        }
    }
    __syncthreads();
    join_found(sh, sh.count, top, last != 0);
}

// The same for the logits x of a segment (all indices above the list's), `largest` each thread's
// largest, special where the thread has met a NaN or +inf: a key is made for the few that may be in
// the list only (155 rows of 91471, top 20: 32 us, 46 with keys for all). A lower limit of the
// list's orders is the least over the row's n waves of the ceil(top / n)-th largest of their lanes'
// largest, its lowest 12 bits as 0: found by counting the lanes above it, a bit at a time. Where
// that limit does not separate enough of them, as many are equal or the row has little but -inf,
// all keys are offered.
__device__ __forceinline__ void offer_logits(Top& sh, int top, const float (&x)[kVectors][4],
                                             float largest, bool special, uint32_t base,
                                             int left) {
    const auto key = [&](int i) {
        const int at = 4 * (i / 4 * kThreads + int(threadIdx.x)) + i % 4;
        return at < left ? key_of(order_of(x[i / 4][i % 4]), base + uint32_t(at)) : 0;
    };
    const uint64_t last = sh.list[top - 1];
    const uint32_t floor = uint32_t(last >> 32), mine = order_of(largest);
    if (threadIdx.x == 0) sh.count = 0;
    const int threads = __syncthreads_count(mine > floor);
    if (!__syncthreads_or(special)) {
        if (threads == 0) return;
        uint32_t limit = floor + 1;
        if (threads > top) {
            // Of a short row the waves that are full, or the first one.
            const int waves = max(1, min(left / 4, kThreads) / 64);
            const int each = (top + waves - 1) / waves;
            uint32_t upto = 0;
#pragma unroll
            for (int b = 31; b >= 12; --b) {
                const uint32_t next = upto | 1u << b;
                upto = __popcll(__ballot(mine >= next)) >= each ? next : upto;
            }
            if ((threadIdx.x & 63) == 0) sh.limits[threadIdx.x / 64] = upto;
            __syncthreads();
            uint32_t least = sh.limits[0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w)
                if (w < waves) least = min(least, sh.limits[w]);
            limit = max(limit, least);
        }
        if (limit > order_of(-INFINITY)) {
            if (mine >= limit) {
#pragma unroll
                for (int i = 0; i < kOffer; ++i) {
                    if (order_of(x[i / 4][i % 4]) < limit) continue;
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < kRoom) sh.found[at] = key(i);
                }
            }
            __syncthreads();
            const int n = sh.count;
            if (n <= kRoom) {
                join_found(sh, n, top, last != 0);
                return;
            }
        }
    }
    __syncthreads();  // all have read the count
    offer(sh, top, key);
}

// ------------------------------------------------------------------ forward

struct Parts {
    int per_row;       // blocks of a row; 1: they write the row's results
    bool stream;       // more than the caches hold: read past them
    Sums* sums;        // (rows, per_row)
    uint64_t* tops;    // (rows, per_row, top)
};

template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprob_rows(RowOut o, Parts p) {
    __shared__ Sums sh[kWaves];
    __shared__ std::conditional_t<TOP, Top, char> st;
    const int64_t r = blockIdx.x / p.per_row;
    const int part = int(blockIdx.x % p.per_row);
    const int segments = int((o.vocab + kSegment - 1) / kSegment);
    const int s0 = int(int64_t(part) * segments / p.per_row);
    const int s1 = int(int64_t(part + 1) * segments / p.per_row);
    const float* row = o.logits + r * o.ld;
    Sums mine{-INFINITY, 0.0f, 0.0f};
    if constexpr (TOP) clear(st, o.top);
    for (int s = s0; s < s1; ++s) {
        const int64_t base = int64_t(s) * kSegment;
        const int left = int(std::min<int64_t>(o.vocab - base, kSegment));
        const int vectors = (left + 4 * kThreads - 1) / (4 * kThreads);
        const float* from = row + base + 4 * threadIdx.x;
        float x[kVectors][4];
        if (left == kSegment) {
            floatx4u v[kVectors];
            if (p.stream) {
#pragma unroll
                for (int j = 0; j < kVectors; ++j)
                    v[j] = __builtin_nontemporal_load(
                        reinterpret_cast<const floatx4u*>(from + j * 4 * kThreads));
            } else {
#pragma unroll
                for (int j = 0; j < kVectors; ++j)
                    v[j] = *reinterpret_cast<const floatx4u*>(from + j * 4 * kThreads);
            }
#pragma unroll
            for (int j = 0; j < kVectors; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = v[j][e];
        } else {
#pragma unroll
            for (int j = 0; j < kVectors; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = -INFINITY;
                const int at = 4 * (j * kThreads + int(threadIdx.x));
                if (at + 4 <= left) {
                    const floatx4u v =
                        *reinterpret_cast<const floatx4u*>(from + j * 4 * kThreads);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = v[e];
                } else if (at < left) {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (at + e < left) x[j][e] = from[j * 4 * kThreads + e];
                }
            }
        }
        float largest = -INFINITY;
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) largest = fmaxf(largest, x[j][e]);
        const float m = fmaxf(mine.m, largest);
        mine = about(mine, m);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
            if (j >= vectors) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = x[j][e] - ref;
                const float y = __builtin_amdgcn_exp2f(d * kLog2e);
                mine.l += y;
                mine.w = __builtin_fmaf(y, fmaxf(d, -200.0f), mine.w);  // not 0 times -inf
            }
        }
        if constexpr (TOP)
            offer_logits(st, o.top, x, largest, mine.l != mine.l, uint32_t(base), left);
    }
    const Sums all = block_sums(mine, sh);
    if (p.per_row > 1) {
        if (threadIdx.x == 0) p.sums[blockIdx.x] = all;
        if constexpr (TOP)
            for (int i = int(threadIdx.x); i < o.top; i += kThreads)
                p.tops[int64_t(blockIdx.x) * o.top + i] = st.list[i];
        return;
    }
    if (threadIdx.x == 0) finish_row(o, r, all);
    if constexpr (TOP) {
        const float z = lse_of(all);
        for (int i = int(threadIdx.x); i < o.top; i += kThreads) {
            const uint32_t j = ~uint32_t(st.list[i]);
            o.top_index[r * o.top + i] = int32_t(j);
            o.top_logprob[r * o.top + i] = z == -INFINITY ? -INFINITY : row[j] - z;
        }
    }
}

// A row's parts: a block a row.
template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprob_join(RowOut o, Parts p) {
    __shared__ Sums sh[kWaves];
    __shared__ std::conditional_t<TOP, Top, char> st;
    const int64_t r = blockIdx.x;
    Sums mine{-INFINITY, 0.0f, 0.0f};
    for (int i = int(threadIdx.x); i < p.per_row; i += kThreads) {
        const Sums b = p.sums[r * p.per_row + i];
        const float m = fmaxf(mine.m, b.m);
        const Sums c = about(mine, m), d = about(b, m);
        mine = Sums{m, c.l + d.l, c.w + d.w};
    }
    const Sums all = block_sums(mine, sh);
    if (threadIdx.x == 0) finish_row(o, r, all);
    if constexpr (TOP) {
        clear(st, o.top);
        const uint64_t* keys = p.tops + r * p.per_row * o.top;
        const int n = p.per_row * o.top;
        if (n <= kThreads) {  // few enough to rank as they are
            if (int(threadIdx.x) < n) {
                const uint64_t key = keys[threadIdx.x];
                // Parts shorter than the list leave zeros; made to differ, they come last.
                st.found[threadIdx.x] = key != 0 ? key : uint64_t(threadIdx.x) + 1;
            }
            __syncthreads();
            list_found(st, n, o.top);
        }
        for (int base = 0; n > kThreads && base < n; base += kThreads * kOffer)
            offer(st, o.top, [&](int i) {
                const int at = base + i * kThreads + int(threadIdx.x);
                return at < n ? keys[at] : 0;
            });
        const float z = lse_of(all);
        for (int i = int(threadIdx.x); i < o.top; i += kThreads) {
            const uint32_t j = ~uint32_t(st.list[i]);
            o.top_index[r * o.top + i] = int32_t(j);
            o.top_logprob[r * o.top + i] = z == -INFINITY ? -INFINITY : o.logits[r * o.ld + j] - z;
        }
    }
}

// ----------------------------------------------------------------- backward

// Block = row, segment. Each logit is read before its gradient is written, by one thread.
__global__ __launch_bounds__(kThreads) void logprob_rows_backward(
    const float* logits, int64_t ld, const int32_t* __restrict__ targets,
    const float* __restrict__ lse, const float* __restrict__ entropy,
    const float* __restrict__ g_logprob, const float* __restrict__ g_entropy, float* dlogits,
    int64_t ld_dlogits, int64_t vocab, int segments) {
    const int64_t r = blockIdx.x / segments;
    const int64_t base = int64_t(blockIdx.x % segments) * kSegment;
    const int left = int(std::min<int64_t>(vocab - base, kSegment));
    const float z = lse[r], g = g_logprob[r];
    const float ge = g_entropy != nullptr ? g_entropy[r] : 0.0f;
    const float h = g_entropy != nullptr ? entropy[r] : 0.0f;
    const int64_t target = targets[r];
    const bool bad = target < 0 || target >= vocab;
    const int64_t t = target - base;
    const float* from = logits + r * ld + base + 4 * threadIdx.x;
    float* to = dlogits + r * ld_dlogits + base + 4 * threadIdx.x;
    const auto gradient = [&](float x, int at) {
        const float d = x - z;
        const float p = __builtin_amdgcn_exp2f(d * kLog2e);
        float y = p == 0.0f ? 0.0f : -p * __builtin_fmaf(ge, d + h, g);
        if (at == t) y += g;
        if (z == -INFINITY) y = 0.0f;
        return bad ? NAN : y;
    };
    if (left == kSegment) {
        floatx4u x[kVectors];
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
            x[j] = __builtin_nontemporal_load(
                reinterpret_cast<const floatx4u*>(from + j * 4 * kThreads));
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
            const int at = 4 * (j * kThreads + int(threadIdx.x));
            floatx4u y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = gradient(x[j][e], at + e);
            __builtin_nontemporal_store(y, reinterpret_cast<floatx4u*>(to + j * 4 * kThreads));
        }
        return;
    }
    for (int j = 0; j < kVectors; ++j) {
        const int at = 4 * (j * kThreads + int(threadIdx.x));
        if (at + 4 <= left) {
            const floatx4u x = *reinterpret_cast<const floatx4u*>(from + j * 4 * kThreads);
            floatx4u y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = gradient(x[e], at + e);
            *reinterpret_cast<floatx4u*>(to + j * 4 * kThreads) = y;
        } else {
            for (int e = 0; e < 4; ++e)
                if (at + e < left)
                    to[j * 4 * kThreads + e] = gradient(from[j * 4 * kThreads + e], at + e);
        }
    }
}

// ---------------------------------------------------------------- host checks

constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;
constexpr int64_t kStream = int64_t(1) << 26;  // logits: 256 MiB, the last cache's size

int check(const char* name, int64_t rows, int64_t vocab, int64_t top) {
    if (rows < 0 || vocab < 1 || vocab > INT32_MAX || top < 0 || top > kMaxTop || top > vocab)
        return fail(EHIP_EINVAL, "%s: %lld rows of %lld logits, top %lld", name, (long long)rows,
                    (long long)vocab, (long long)top);
    if (rows > kMaxBlocks || rows * ceil_div(vocab, kSegment) > kMaxBlocks)
        return fail(EHIP_EINVAL, "%s: %lld rows of %lld logits are too many", name,
                    (long long)rows, (long long)vocab);
    return EHIP_OK;
}

// Blocks of a row: one from 512 rows (two a CU) on, else what makes some 1024 of them.
int parts_of(int64_t rows, int64_t vocab) {
    if (rows == 0 || rows >= 512) return 1;
    return int(std::min(ceil_div(vocab, kSegment), ceil_div(1024, rows)));
}

size_t part_bytes(int64_t rows, int parts, int64_t top) {
    return parts > 1 ? size_t(rows) * size_t(parts) *
                           (sizeof(Sums) + 4 + size_t(top) * sizeof(uint64_t))
                     : 0;
}

template <bool TOP>
int launch_forward(const RowOut& o, const Parts& p, int64_t rows, hipStream_t s) {
    EHIP_LAUNCH("token_logprobs", logprob_rows<TOP>, dim3(unsigned(rows * p.per_row)),
                dim3(kThreads), 0, s, o, p);
    if (p.per_row > 1)
        EHIP_LAUNCH("token_logprobs_join", logprob_join<TOP>, dim3(unsigned(rows)), dim3(kThreads),
                    0, s, o, p);
    return EHIP_OK;
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int64_t ehip_token_logprobs_workspace(int64_t rows, int64_t vocab, int64_t top) {
    if (check("token_logprobs", rows, vocab, top)) return -1;
    return int64_t(part_bytes(rows, parts_of(rows, vocab), top));
}

int ehip_token_logprobs_f32(const float* logits, int64_t ld, const int32_t* targets, int64_t rows,
                            int64_t vocab, float* logprob, float* entropy, float* lse, int64_t top,
                            float* top_logprob, int32_t* top_index, void* workspace,
                            size_t workspace_bytes, void* stream) {
    EHIP_READY();
    if (int rc = check("token_logprobs", rows, vocab, top)) return rc;
    if (ld < vocab) return fail(EHIP_EINVAL, "token_logprobs: rows of %lld logits %lld apart",
                                (long long)vocab, (long long)ld);
    if (rows == 0) return EHIP_OK;
    if (logits == nullptr || lse == nullptr || (logprob != nullptr && targets == nullptr) ||
        (top > 0 && (top_logprob == nullptr || top_index == nullptr)))
        return fail(EHIP_EINVAL, "token_logprobs: null tensor");
    Parts p{parts_of(rows, vocab), rows * vocab >= kStream, nullptr, nullptr};
    const size_t need = part_bytes(rows, p.per_row, top);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(EHIP_EINVAL, "token_logprobs: needs %zu bytes of 16-byte aligned workspace",
                    need);
    p.tops = static_cast<uint64_t*>(workspace);
    p.sums = reinterpret_cast<Sums*>(p.tops + size_t(rows) * size_t(p.per_row) * size_t(top));
    const RowOut o{logits,  ld,  targets,  vocab,       logprob,
                   entropy, lse, int(top), top_logprob, top_index};
    return top > 0 ? launch_forward<true>(o, p, rows, as_stream(stream))
                   : launch_forward<false>(o, p, rows, as_stream(stream));
}

int ehip_token_logprobs_backward_f32(const float* logits, int64_t ld, const int32_t* targets,
                                     const float* lse, const float* entropy,
                                     const float* g_logprob, const float* g_entropy,
                                     float* dlogits, int64_t ld_dlogits, int64_t rows,
                                     int64_t vocab, void* stream) {
    EHIP_READY();
    if (int rc = check("token_logprobs_backward", rows, vocab, 0)) return rc;
    if (ld < vocab || ld_dlogits < vocab)
        return fail(EHIP_EINVAL, "token_logprobs_backward: rows of %lld logits %lld and %lld apart",
                    (long long)vocab, (long long)ld, (long long)ld_dlogits);
    if (rows == 0) return EHIP_OK;
    if (logits == nullptr || targets == nullptr || lse == nullptr || g_logprob == nullptr ||
        dlogits == nullptr || (g_entropy != nullptr && entropy == nullptr))
        return fail(EHIP_EINVAL, "token_logprobs_backward: null tensor");
    const int64_t segments = ceil_div(vocab, kSegment);
    EHIP_LAUNCH("token_logprobs_backward", logprob_rows_backward, dim3(unsigned(rows * segments)),
                dim3(kThreads), 0, as_stream(stream), logits, ld, targets, lse, entropy, g_logprob,
                g_entropy, dlogits, ld_dlogits, vocab, int(segments));
    return EHIP_OK;
}

}  // extern "C"
