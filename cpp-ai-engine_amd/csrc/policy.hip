// policy.hip -- the clipped policy loss of sampled tokens with a KL term and an entropy bonus, and
// its gradient with respect to their log probabilities and entropies. For a token of log probability
// p, under the sampling policy o and under a reference f, with advantage A and entropy H:
//
//   d = p - o, ratio = exp(d); surrogate = min(ratio, 1 + high) A, or max(ratio, 1 - low) A for A < 0
//   kl = exp(f - p) - (f - p) - 1
//   loss = sum_t w_t (-surrogate + beta kl - c H), w_t the mean's over tokens or over sequences
//   dp = w (-[not clipped] ratio A + beta (1 - exp(f - p))), dH = -c w
//
// HBM bounds long batches, latency short ones. Over 2 million tokens of 2048 sequences with all
// tensors the sums take 18 us (42 MB, 2.4 TB/s), joining them 7, the gradient 14 (50 MB, 3.7 TB/s);
// the arithmetic of some 60 to 80 operations a token is not hidden by the loads altogether. The
// flat tokens are cut into chunks of kChunk and a wave takes what one sequence has of one chunk, a
// segment. The segment of chunk c and sequence s has place c + s, no other's: from one to the next
// at least one of them grows. So a wave finds its segment by searching the offsets, without a list
// of them.

#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace ehip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunk = 512;          // tokens of a wave
constexpr int kBatch = 4;            // tokens of a lane that are read together
constexpr int kJoinThreads = 256;    // sequences of a joining block
constexpr int kOwn = 16;             // segments that a thread adds up by itself
constexpr int kFewThreads = 1024;
constexpr int kFew = 64;             // places that one block takes

// Sums of a segment, a sequence or all, in 64 bits: up to 2^31 terms.
struct Sums {
    double loss, kl, ratio;
    int clipped, tokens;
};

struct BlockSums {
    double loss, kl, ratio, clipped, tokens, count;
};

struct Policy {
    const float *logprob, *old, *advantage, *ref, *entropy;
    const uint8_t* mask;
    const int32_t* cu;
    int sequences, tokens;
    bool advantage_by_sequence, mean_by_sequence;
    double log_low, log_high;  // clipped where d is below, above
    double low, high;          // the ratio there
    float kl_weight, entropy_weight;
    int64_t places;
};

__device__ __forceinline__ int offset(const Policy& a, int s) {
    return min(max(a.cu[s], 0), a.tokens);
}

struct Segment {
    int s, begin, end;
};

// The segment of a place (begin == end: none). Every lane of the wave calls it.
__device__ __forceinline__ Segment segment_of(const Policy& a, int64_t place) {
    if (a.sequences == 0) return Segment{0, 0, 0};
    // The last sequence whose first place is not past it: 64 candidates at a time, a lane each.
    const int lane = int(threadIdx.x) & 63;
    int lo = 0, n = a.sequences;
    while (true) {
        const int step = (n + 63) / 64, at = lane * step;
        const int s = at < n ? lo + at : lo;
        const int64_t first = int64_t(offset(a, s) / kChunk) + s;
        const int c = __popcll(__ballot(at < n && first <= place));
        if (c > 0) lo += (c - 1) * step;
        n = c > 0 ? min(n - (c - 1) * step, step) : 1;
        if (step == 1 || c == 0) break;
    }
    Segment g{lo, 0, 0};
    const int64_t chunk = place - lo;
    const int64_t begin = offset(a, lo), end = offset(a, lo + 1);
    const int64_t from = std::max(begin, chunk * kChunk), to = std::min(end, (chunk + 1) * kChunk);
    if (chunk >= 0 && from < to) {
        g.begin = int(from);
        g.end = int(to);
    }
    return g;
}

// exp(x) - x - 1 below one in magnitude, by its series, whose next term is 2^-35 of it: the difference
// would have few digits.
__device__ __forceinline__ float kl_series(float x) {
    float s = 1.0f;
#pragma unroll
    for (int n = 13; n >= 3; --n) s = __builtin_fmaf(x * (1.0f / float(n)), s, 1.0f);
    return 0.5f * x * x * s;
}
// 2^-40 of the same of any x: past fp32 up to x = 115, which is more than a mean over all the tokens that
// there can be brings back. The exponential is the square of that of the half. (In 64 bits the kernel
// of 2 million tokens took 19.2 us in place of 17.9.)
constexpr float kKlUnit = 0x1p-40f;
__device__ __forceinline__ float kl_of(float x) {
    const float h = expf(0.5f * x) * 0x1p-20f;
    const float kl = __builtin_fmaf(h, h, -kKlUnit) - fminf(x, 1e30f) * kKlUnit;  // not inf - inf
    return fabsf(x) < 1.0f ? kl_series(x) * kKlUnit : kl;
}

// exp(x): 2^n exp(f), |f| <= ln 2 / 2, by Taylor's series, whose next term is 2^-37 of it. A third of
// the library's instructions, which has 53 bits.
__device__ __forceinline__ double exp36(double x) {
    x = x < -800.0 ? -800.0 : x > 800.0 ? 800.0 : x;  // 0 and infinity; NaN stays
    const double n = rint(x * 1.44269504088896340736);
    const double f = __builtin_fma(-n, 0.693147180559945309417, x);
    double s = 1.0;
#pragma unroll
    for (int i = 9; i >= 1; --i) s = __builtin_fma(f * (1.0 / double(i)), s, 1.0);
    return ldexp(s, x == x ? int(n) : 0);
}

// Tokens t, t + 64, ... of a segment as they are read: all together, those that do not count too,
// whose values are then not used (2 million tokens of 2048 sequences, in
// 32 bits: 19 us one by one, 14 like this, 15 by eight).
struct Tokens {
    float p[kBatch], old[kBatch], advantage[kBatch], ref[kBatch], entropy[kBatch];
    bool counts[kBatch];
};

template <bool ENTROPY>
__device__ __forceinline__ void load(const Policy& a, const Segment& g, int t, Tokens& x) {
    uint8_t mask[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const int at = min(t + 64 * i, g.end - 1);
        mask[i] = a.mask != nullptr ? a.mask[at] : 1;
        x.p[i] = a.logprob[at];
        x.old[i] = a.old[at];
        x.advantage[i] = a.advantage[a.advantage_by_sequence ? g.s : at];
        x.ref[i] = a.ref != nullptr ? a.ref[at] : 0.0f;
        if (ENTROPY) x.entropy[i] = a.entropy != nullptr ? a.entropy[at] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x.counts[i] = mask[i] != 0 && t + 64 * i < g.end;
}

// Whether the ratio is clipped goes by the difference in 64 bits.
__device__ __forceinline__ bool clipped(const Policy& a, double d, float advantage) {
    return advantage < 0.0f ? d < a.log_low : d > a.log_high;
}

// A token's terms. The loss's sum takes 64 bits, as it has terms of both signs (340 tokens' of about 1
// have come to 10^-3; 17 us in place of the 14 in 32 bits).
struct Token {
    double ratio, surrogate;
    float kl;  // kKlUnit of it
    bool clipped;
};

__device__ __forceinline__ Token token_of(const Policy& a, const Tokens& from, int i) {
    Token x;
    const float advantage = from.advantage[i];
    const double d = double(from.p[i]) - double(from.old[i]);
    x.ratio = exp36(d);
    x.clipped = clipped(a, d, advantage);
    x.surrogate = (x.clipped ? (advantage < 0.0f ? a.low : a.high) : x.ratio) * double(advantage);
    x.kl = a.ref != nullptr ? kl_of(float(double(from.ref[i]) - double(from.p[i]))) : 0.0f;
    return x;
}

// The gradient of a token of weight w by its log probability, in 32 bits. An exponential past fp32, or
// below its normal numbers, may not be once it has the weight: the weight takes the square root twice.
__device__ __forceinline__ float gradient_of(const Policy& a, const Tokens& from, int i, float w) {
    const float advantage = from.advantage[i];
    const double d = double(from.p[i]) - double(from.old[i]);
    const float h = expf(0.5f * float(d));
    float y = clipped(a, d, advantage) ? 0.0f : -(w * advantage * h * h);
    if (a.ref != nullptr && a.kl_weight != 0.0f) {
        const float x = float(double(from.ref[i]) - double(from.p[i])), r = expf(0.5f * x);
        const float by = w * a.kl_weight;
        y -= fabsf(x) < 1.0f ? by * (x + kl_series(x)) : by * r * r - by;
    }
    return y;
}

template <class T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// The sums of a place's segment. Every lane of the wave calls it.
__device__ __forceinline__ void sum_segment(const Policy& a, int64_t place, Sums* sums) {
    const int lane = int(threadIdx.x) & 63;
    const Segment g = segment_of(a, place);
    if (g.begin == g.end) return;
    Sums x{};
    for (int t = g.begin; t < g.end; t += 64 * kBatch) {
        Tokens all;
        load<true>(a, g, t + lane, all);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (t + 64 * i >= g.end) break;
            const Token y = token_of(a, all, i);
            double loss = -y.surrogate;
            const double kl = double(y.kl) * (1.0 / kKlUnit);
            if (a.kl_weight != 0.0f) loss = __builtin_fma(double(a.kl_weight), kl, loss);
            if (a.entropy_weight != 0.0f)
                loss = __builtin_fma(-double(a.entropy_weight), double(all.entropy[i]), loss);
            const bool counts = all.counts[i];
            x.loss += counts ? loss : 0.0;
            x.kl += counts ? kl : 0.0;
            x.ratio += counts ? y.ratio : 0.0;
            x.clipped += counts && y.clipped;
            x.tokens += counts;
        }
    }
    x.loss = wave_sum(x.loss);
    x.kl = wave_sum(x.kl);
    x.ratio = wave_sum(x.ratio);
    x.clipped = wave_sum(x.clipped);
    x.tokens = wave_sum(x.tokens);
    if (lane == 0) sums[place] = x;
}

__global__ __launch_bounds__(kThreads) void policy_segments(Policy a, Sums* sums) {
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int64_t place = int64_t(blockIdx.x) * kWaves + wave;
    if (place < a.places) sum_segment(a, place, sums);
}

__device__ __forceinline__ void add(Sums& x, const Sums& y) {
    x.loss += y.loss;
    x.kl += y.kl;
    x.ratio += y.ratio;
    x.clipped += y.clipped;
    x.tokens += y.tokens;
}

__device__ __forceinline__ void finish(const Policy& a, const BlockSums& x, float* loss,
                                       float* stats, float* weights) {
    const bool none = x.tokens == 0.0;
    loss[0] = none ? 0.0f : float(x.loss / x.count);
    if (stats != nullptr) {
        stats[0] = none ? 0.0f : float(x.kl / x.tokens);
        stats[1] = none ? 0.0f : float(x.clipped / x.tokens);
        stats[2] = none ? 0.0f : float(x.ratio / x.tokens);
    }
    weights[a.sequences] = none ? 0.0f : float(1.0 / x.count);
}

// The sums of all threads of the block in thread 0. Every thread calls it.
template <int THREADS>
__device__ __forceinline__ BlockSums block_sums(const BlockSums& mine, BlockSums* sh) {
    const BlockSums x{wave_sum(mine.loss),    wave_sum(mine.kl),     wave_sum(mine.ratio),
                      wave_sum(mine.clipped), wave_sum(mine.tokens), wave_sum(mine.count)};
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x / 64] = x;
    __syncthreads();
    BlockSums all{};
    if (threadIdx.x == 0)
        for (int w = 0; w < THREADS / 64; ++w) {
            all.loss += sh[w].loss;
            all.kl += sh[w].kl;
            all.ratio += sh[w].ratio;
            all.clipped += sh[w].clipped;
            all.tokens += sh[w].tokens;
            all.count += sh[w].count;
        }
    return all;
}

// The sums and weights of a block's sequences, a thread each; a sequence of many segments by its
// wave. Returns all sequences' sums in thread 0. Every thread of the block calls it.
template <int THREADS>
__device__ __forceinline__ BlockSums sum_sequences(const Policy& a, int s, const Sums* sums,
                                                   float* weights, BlockSums* sh) {
    const int lane = int(threadIdx.x) & 63;
    int64_t first = 0;
    int count = 0;
    if (s < a.sequences) {
        const int begin = offset(a, s), end = offset(a, s + 1);
        first = int64_t(begin / kChunk) + s;
        count = begin < end ? (end - 1) / kChunk - begin / kChunk + 1 : 0;
    }
    Sums x{};
    if (count <= kOwn) {
#pragma unroll 4
        for (int i = 0; i < count; ++i) add(x, sums[first + i]);
    }
    for (uint64_t many = __ballot(count > kOwn); many != 0; many &= many - 1) {
        const int from = __builtin_ctzll(many);
        const int64_t at = __shfl(first, from);
        const int n = __shfl(count, from);
        Sums y{};
        for (int i = lane; i < n; i += 64) add(y, sums[at + i]);
        y.loss = wave_sum(y.loss);
        y.kl = wave_sum(y.kl);
        y.ratio = wave_sum(y.ratio);
        y.clipped = wave_sum(y.clipped);
        y.tokens = wave_sum(y.tokens);
        if (lane == from) x = y;
    }
    const double n = double(x.tokens);
    double w = 1.0;
    if (a.mean_by_sequence) w = x.tokens > 0 ? 1.0 / n : 0.0;
    if (s < a.sequences) weights[s] = float(w);
    const BlockSums mine{x.tokens > 0 ? x.loss * w : 0.0,
                         x.kl,
                         x.ratio,
                         double(x.clipped),
                         n,
                         a.mean_by_sequence ? double(x.tokens > 0) : n};
    return block_sums<THREADS>(mine, sh);
}

// One block writes the results, several their sums for policy_finish.
__global__ __launch_bounds__(kJoinThreads) void policy_sequences(Policy a, const Sums* sums,
                                                                 BlockSums* blocks, float* loss,
                                                                 float* stats, float* weights) {
    __shared__ BlockSums sh[kJoinThreads / 64];
    const int s = int(blockIdx.x) * kJoinThreads + int(threadIdx.x);
    const BlockSums all = sum_sequences<kJoinThreads>(a, s, sums, weights, sh);
    if (threadIdx.x != 0) return;
    if (gridDim.x > 1) blocks[blockIdx.x] = all;
    else finish(a, all, loss, stats, weights);
}

// All in one block, for up to kFew places: a launch less (32 sequences, 340 tokens in all, with the
// gradient, from Python: 28 us with two, 22 like this, and with fewer tensors made).
__global__ __launch_bounds__(kFewThreads) void policy_few(Policy a, Sums* sums, float* loss,
                                                          float* stats, float* weights) {
    __shared__ BlockSums sh[kFewThreads / 64];
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    for (int64_t place = wave; place < a.places; place += kFewThreads / 64)
        sum_segment(a, place, sums);
    __syncthreads();
    const BlockSums all = sum_sequences<kFewThreads>(a, int(threadIdx.x), sums, weights, sh);
    if (threadIdx.x == 0) finish(a, all, loss, stats, weights);
}

__global__ __launch_bounds__(kJoinThreads) void policy_finish(Policy a, const BlockSums* blocks,
                                                              int count, float* loss, float* stats,
                                                              float* weights) {
    __shared__ BlockSums sh[kJoinThreads / 64];
    BlockSums x{};
    for (int i = int(threadIdx.x); i < count; i += kJoinThreads) {
        const BlockSums y = blocks[i];
        x.loss += y.loss;
        x.kl += y.kl;
        x.ratio += y.ratio;
        x.clipped += y.clipped;
        x.tokens += y.tokens;
        x.count += y.count;
    }
    x = block_sums<kJoinThreads>(x, sh);
    if (threadIdx.x == 0) finish(a, x, loss, stats, weights);
}

__global__ __launch_bounds__(kThreads) void policy_backward(Policy a,
                                                            const float* __restrict__ weights,
                                                            const float* __restrict__ grad,
                                                            float* g_logprob, float* g_entropy) {
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int lane = int(threadIdx.x) & 63;
    const int64_t place = int64_t(blockIdx.x) * kWaves + wave;
    if (place >= a.places) return;
    // Tokens of the place's chunk that are of no sequence.
    const int64_t base = place * kChunk, stop = std::min<int64_t>(base + kChunk, a.tokens);
    const int begin = offset(a, 0), end = offset(a, a.sequences);
    if (base < begin || stop > end) {
        for (int64_t t = base + lane; t < stop; t += 64) {
            if (t >= begin && t < end) continue;
            if (g_logprob != nullptr) g_logprob[t] = 0.0f;
            if (g_entropy != nullptr) g_entropy[t] = 0.0f;
        }
    }
    const Segment g = segment_of(a, place);
    if (g.begin == g.end) return;
    const float w = grad[0] * (weights[g.s] * weights[a.sequences]);
    for (int t = g.begin; t < g.end; t += 64 * kBatch) {
        Tokens all;
        load<false>(a, g, t + lane, all);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = t + 64 * i + lane;
            if (at - lane >= g.end) break;
            if (at >= g.end) continue;
            const float y = gradient_of(a, all, i, w);
            if (g_logprob != nullptr) g_logprob[at] = all.counts[i] ? y : 0.0f;
            if (g_entropy != nullptr)
                g_entropy[at] = all.counts[i] ? -a.entropy_weight * w : 0.0f;
        }
    }
}

// ---------------------------------------------------------------- host checks

constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

int check(const char* name, const ehip_policy_t* d, Policy& a) {
    if (d == nullptr) return fail(EHIP_EINVAL, "%s: null descriptor", name);
    if (d->sequences < 0 || d->tokens < 0 || d->sequences > kMaxBlocks ||
        d->tokens > INT32_MAX - kChunk)
        return fail(EHIP_EINVAL, "%s: %lld sequences of %lld tokens", name,
                    (long long)d->sequences, (long long)d->tokens);
    if (!(d->clip_low >= 0.0) || !(d->clip_high >= 0.0))
        return fail(EHIP_EINVAL, "%s: clipped by %g and %g", name, d->clip_low, d->clip_high);
    if (!std::isfinite(d->kl_weight) || !std::isfinite(d->entropy_weight))
        return fail(EHIP_EINVAL, "%s: weights %g and %g", name, double(d->kl_weight),
                    double(d->entropy_weight));
    if ((d->kl_weight != 0.0f && d->ref_logprob == nullptr && d->tokens > 0) ||
        (d->entropy_weight != 0.0f && d->entropy == nullptr && d->tokens > 0))
        return fail(EHIP_EINVAL, "%s: a weighted term without its tensor", name);
    a = Policy{};
    a.logprob = d->logprob;
    a.old = d->old_logprob;
    a.advantage = d->advantage;
    a.ref = d->ref_logprob;
    a.entropy = d->entropy;
    a.mask = d->mask;
    a.cu = d->cu;
    a.sequences = int(d->sequences);
    a.tokens = int(d->tokens);
    a.advantage_by_sequence = d->advantage_by_sequence != 0;
    a.mean_by_sequence = d->mean_by_sequence != 0;
    a.log_low = d->clip_low < 1.0 ? std::log1p(-d->clip_low) : -INFINITY;
    a.log_high = std::log1p(d->clip_high);
    a.low = 1.0 - d->clip_low;
    a.high = 1.0 + d->clip_high;
    a.kl_weight = d->kl_weight;
    a.entropy_weight = d->entropy_weight;
    a.places = a.tokens / kChunk + 1 + a.sequences;
    return EHIP_OK;
}

int check_tensors(const char* name, const Policy& a) {
    const bool advantages = !a.advantage_by_sequence || a.sequences > 0;
    if (a.cu == nullptr || (a.tokens > 0 && (a.logprob == nullptr || a.old == nullptr ||
                                             (advantages && a.advantage == nullptr))))
        return fail(EHIP_EINVAL, "%s: null tensor", name);
    return EHIP_OK;
}

int64_t join_blocks(const Policy& a) {
    return std::max<int64_t>(1, ceil_div(a.sequences, kJoinThreads));
}

size_t part_bytes(const Policy& a) {
    return size_t(a.places) * sizeof(Sums) + size_t(join_blocks(a)) * sizeof(BlockSums);
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int64_t ehip_policy_loss_workspace(const ehip_policy_t* desc) {
    Policy a;
    return check("policy_loss", desc, a) ? -1 : int64_t(part_bytes(a));
}

int ehip_policy_loss_f32(const ehip_policy_t* desc, float* loss, float* stats, float* weights,
                         void* workspace, size_t workspace_bytes, void* stream) {
    EHIP_READY();
    Policy a;
    if (int rc = check("policy_loss", desc, a)) return rc;
    if (int rc = check_tensors("policy_loss", a)) return rc;
    if (loss == nullptr || weights == nullptr)
        return fail(EHIP_EINVAL, "policy_loss: null tensor");
    const size_t need = part_bytes(a);
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))
        return fail(EHIP_EINVAL, "policy_loss: needs %zu bytes of 16-byte aligned workspace", need);
    BlockSums* const blocks = static_cast<BlockSums*>(workspace);
    const int64_t joins = join_blocks(a);
    Sums* const sums = reinterpret_cast<Sums*>(blocks + joins);
    hipStream_t s = as_stream(stream);
    if (a.places <= kFew) {
        EHIP_LAUNCH("policy_loss", policy_few, dim3(1), dim3(kFewThreads), 0, s, a, sums, loss,
                    stats, weights);
        return EHIP_OK;
    }
    if (a.tokens > 0 && a.sequences > 0)
        EHIP_LAUNCH("policy_loss", policy_segments, dim3(unsigned(ceil_div(a.places, kWaves))),
                    dim3(kThreads), 0, s, a, sums);
    EHIP_LAUNCH("policy_loss_sequences", policy_sequences, dim3(unsigned(joins)),
                dim3(kJoinThreads), 0, s, a, sums, blocks, loss, stats, weights);
    if (joins > 1)
        EHIP_LAUNCH("policy_loss_finish", policy_finish, dim3(1), dim3(kJoinThreads), 0, s, a,
                    blocks, int(joins), loss, stats, weights);
    return EHIP_OK;
}

int ehip_policy_loss_backward_f32(const ehip_policy_t* desc, const float* weights,
                                  const float* grad, float* g_logprob, float* g_entropy,
                                  void* stream) {
    EHIP_READY();
    Policy a;
    if (int rc = check("policy_loss_backward", desc, a)) return rc;
    if (int rc = check_tensors("policy_loss_backward", a)) return rc;
    if (weights == nullptr || grad == nullptr)
        return fail(EHIP_EINVAL, "policy_loss_backward: null tensor");
    if (a.tokens == 0 || (g_logprob == nullptr && g_entropy == nullptr)) return EHIP_OK;
    EHIP_LAUNCH("policy_loss_backward", policy_backward,
                dim3(unsigned(ceil_div(a.places, kWaves))), dim3(kThreads), 0, as_stream(stream), a,
                weights, grad, g_logprob, g_entropy);
    return EHIP_OK;
}

}  // extern "C"
