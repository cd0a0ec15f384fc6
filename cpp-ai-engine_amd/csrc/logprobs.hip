// logprobs.hip -- log probabilities of given tokens, the entropy of each row's distribution and
// its largest logits, and the gradient of the first two:
//
//   lse = log sum_j exp(x_j), logprob = x_t - lse, H = lse - sum_j p_j x_j, p_j = exp(x_j - lse)
//   dx_j = g_lp ([j = t] - p_j) - g_H p_j (x_j - lse + H)

#include "common.hpp"

#include <cmath>

namespace ehip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 128;

__device__ __forceinline__ float block_max(float x, float* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x / 64] = x;
    __syncthreads();
    x = sh[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) x = fmaxf(x, sh[w]);
    return x;
}
__device__ __forceinline__ float block_sum(float x, float* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x / 64] = x;
    __syncthreads();
    x = sh[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) x += sh[w];
    return x;
}

// A logit and its index as one number that is larger the earlier it comes among the top: the
// logit's order (-0 as 0, NaN above all) in the high half, the index from above in the low one.
// Every key of a row is above 0.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
    uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    b = x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
    return uint64_t(b) << 32 | uint32_t(~index);
}

// A block a row: the maximum, the sums, then the top one by one, each the largest key below the
// last.
__global__ __launch_bounds__(kThreads) void logprob_rows(
    const float* __restrict__ logits, int64_t ld, const int32_t* __restrict__ targets,
    int64_t vocab, float* logprob, float* entropy, float* lse, int top, float* top_logprob,
    int32_t* top_index) {
    __shared__ float sh[kThreads / 64];
    __shared__ uint64_t best[kThreads];
    const int64_t r = blockIdx.x;
    const float* x = logits + r * ld;
    float m = -INFINITY;
    bool bad = false;
    for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
        m = fmaxf(m, x[j]);
        bad |= x[j] != x[j];
    }
    m = block_max(m, sh);
    bad = __syncthreads_or(bad) || m == INFINITY;
    float sum = 0.0f, wsum = 0.0f;
    for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
        const float d = x[j] - m, e = m == -INFINITY ? 0.0f : expf(d);
        sum += e;
        wsum += e == 0.0f ? 0.0f : e * d;
    }
    sum = block_sum(sum, sh);
    wsum = block_sum(wsum, sh);
    const bool empty = m == -INFINITY && !bad;
    const float z = bad ? NAN : (empty ? -INFINITY : m + logf(sum));
    if (threadIdx.x == 0) {
        lse[r] = z;
        if (entropy != nullptr) entropy[r] = bad ? NAN : (empty ? 0.0f : logf(sum) - wsum / sum);
        if (logprob != nullptr) {
            const int64_t t = targets[r];
            logprob[r] = t < 0 || t >= vocab ? NAN : (empty ? -INFINITY : x[t] - z);
        }
    }
    uint64_t below = ~uint64_t(0);
    for (int n = 0; n < top; ++n) {
        uint64_t mine = 0;
        for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
            const uint64_t key = order_key(x[j], uint32_t(j));
            if (key < below && key > mine) mine = key;
        }
        __syncthreads();
        best[threadIdx.x] = mine;
        __syncthreads();
        for (int i = 0; i < kThreads; ++i) mine = best[i] > mine ? best[i] : mine;
        below = mine;
        if (threadIdx.x == 0) {
            const uint32_t j = ~uint32_t(mine);
            top_index[r * top + n] = int32_t(j);
            top_logprob[r * top + n] = empty ? -INFINITY : x[j] - z;
        }
    }
}

__global__ __launch_bounds__(kThreads) void logprob_rows_backward(
    const float* logits, int64_t ld, const int32_t* __restrict__ targets,
    const float* __restrict__ lse, const float* __restrict__ entropy,
    const float* __restrict__ g_logprob, const float* __restrict__ g_entropy, float* dlogits,
    int64_t ld_dlogits, int64_t vocab) {
    const int64_t r = blockIdx.x;
    const float z = lse[r], g = g_logprob[r];
    const float ge = g_entropy != nullptr ? g_entropy[r] : 0.0f;
    const float h = g_entropy != nullptr ? entropy[r] : 0.0f;
    const int64_t t = targets[r];
    const bool bad = t < 0 || t >= vocab;
    for (int64_t j = threadIdx.x; j < vocab; j += kThreads) {
        const float d = logits[r * ld + j] - z;
        float y = 0.0f;
        if (z != -INFINITY) {
            const float p = expf(d);
            y = p == 0.0f ? 0.0f : -p * (g + ge * (d + h));
            if (j == t) y += g;
        }
        dlogits[r * ld_dlogits + j] = bad ? NAN : y;
    }
}

constexpr int64_t kMaxRows = (int64_t(1) << 24) - 1;

int check(const char* name, int64_t rows, int64_t vocab, int64_t top) {
    if (rows < 0 || vocab < 1 || vocab > INT32_MAX || top < 0 || top > kMaxTop || top > vocab)
        return fail(EHIP_EINVAL, "%s: %lld rows of %lld logits, top %lld", name, (long long)rows,
                    (long long)vocab, (long long)top);
    if (rows > kMaxRows)
        return fail(EHIP_EINVAL, "%s: %lld rows are too many", name, (long long)rows);
    return EHIP_OK;
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int64_t ehip_token_logprobs_workspace(int64_t rows, int64_t vocab, int64_t top) {
    return check("token_logprobs", rows, vocab, top) ? -1 : 0;
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
    EHIP_LAUNCH("token_logprobs", logprob_rows, dim3(unsigned(rows)), dim3(kThreads), 0,
                as_stream(stream), logits, ld, targets, vocab, logprob, entropy, lse, int(top),
                top_logprob, top_index);
    return EHIP_OK;
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
    EHIP_LAUNCH("token_logprobs_backward", logprob_rows_backward, dim3(unsigned(rows)),
                dim3(kThreads), 0, as_stream(stream), logits, ld, targets, lse, entropy, g_logprob,
                g_entropy, dlogits, ld_dlogits, vocab);
    return EHIP_OK;
}

}  // extern "C"
