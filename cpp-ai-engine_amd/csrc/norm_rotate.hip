// norm_rotate.hip -- the norm of every query and key head and its rotation by the token's position,
// in one pass, and the gradient. For a head's values x, its weight w and the angles t_i = position
// f_i of its pairs (a, b):
//
//   r = 1 / sqrt(mean x^2 + eps)    y = x r w
//   out_a = y_a cos t_i - y_b sin t_i    out_b = y_b cos t_i + y_a sin t_i    out = y elsewhere
//   u = grad turned by -t    dx = r (w u - x r^2 mean(w u x))    dw = sum of u x r
//
// HBM bounds it: a head is read once, in registers of a few lanes, and written. The angles are
// formed here, in 64 bits from the product to the quarter turn (a position of a million is some
// 10^5 turns, whose fraction fp32 does not have), once for a wave's heads of a token. 369 MB of
// query and key heads of 96 take 87 us, 4.2 TB/s; 134 MB of heads of 64 26 us, 5.2 TB/s, and back
// 201 MB 44 us, 4.6 TB/s, with 5 for the weights' gradients.

#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace ehip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxDim = 256;
constexpr int kMaxParts = 1024;  // blocks of the backward, each with a share of dw

// Four floats at any float's address.
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

struct Side {  // the queries or the keys
    const float *x, *grad, *weight;
    float* out;
    int64_t ld, ld_grad, ld_out;
};

struct Args {
    Side q, k;
    int heads, total_heads;  // of the queries; of both
    int dim, half;           // half: pairs
    bool interleaved;
    const int32_t* positions;
    const double* freqs;
    float eps;
    int64_t tokens;
    int per, chunks;  // heads of a wave, shares of a token
    int each;         // tokens of a wave, where it holds several tokens' heads at a time
    int64_t units;    // waves' worth of work
    float* parts;     // (blocks, 2, dim): shares of the weights' gradients
};

// The places of a lane's eight values in a head, two runs of up to four: value j of the first and
// of the second, or neighbours, are a pair; the lanes past the pairs hold what is not rotated.
struct Places {
    int a, b, na, nb;
    bool pairs;
};

__device__ __forceinline__ int upto4(int n) { return n < 0 ? 0 : n < 4 ? n : 4; }

__device__ __forceinline__ Places places(const Args& a, int u) {
    const int units = (a.half + 3) / 4, rotary = 2 * a.half;
    Places p;
    p.pairs = u < units;
    if (p.pairs && !a.interleaved) {
        p.a = 4 * u;
        p.b = a.half + 4 * u;
        p.na = p.nb = upto4(a.half - 4 * u);
    } else {
        p.a = p.pairs ? 8 * u : rotary + 8 * (u - units);
        p.b = p.a + 4;
        const int end = p.pairs ? rotary : a.dim;
        p.na = upto4(end - p.a);
        p.nb = upto4(end - p.b);
    }
    return p;
}

__device__ __forceinline__ void load4(const float* row, int at, int n, float* x) {
    if (n == 4) {
        const floatx4u v = *reinterpret_cast<const floatx4u*>(row + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = e < n ? row[at + e] : 0.0f;
    }
}
__device__ __forceinline__ void store4(float* row, int at, int n, const float* x) {
    if (n == 4) {
        *reinterpret_cast<floatx4u*>(row + at) = floatx4u{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < n) row[at + e] = x[e];
    }
}
__device__ __forceinline__ void load8(const float* row, const Places& p, float (&x)[8]) {
    load4(row, p.a, p.na, x);
    load4(row, p.b, p.nb, x + 4);
}
__device__ __forceinline__ void store8(float* row, const Places& p, const float (&x)[8]) {
    store4(row, p.a, p.na, x);
    store4(row, p.b, p.nb, x + 4);
}

// Sine and cosine of an angle in 64 bits: less the nearest number of quarter turns (pi / 2 in two
// parts), then their Taylor series, whose next terms are below 2^-28 at pi / 4, in fp32.
__device__ __forceinline__ void sine_cosine(double angle, float& sine, float& cosine) {
    const double n = rint(angle * 0.63661977236758134308);
    double f = __builtin_fma(-n, 1.57079632679489655800, angle);
    f = __builtin_fma(-n, 6.12323399573676603587e-17, f);
    const float x = float(f), z = x * x;
    float s = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
    s = __builtin_fmaf(z, s, 1.0f / 120.0f);
    s = __builtin_fmaf(z, s, -1.0f / 6.0f);
    s = __builtin_fmaf(x * z, s, x);
    float c = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = __builtin_fmaf(z, c, -1.0f / 720.0f);
    c = __builtin_fmaf(z, c, 1.0f / 24.0f);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.0f);
    const int quarter = int(n - 4.0 * floor(n * 0.25));  // 0 .. 3
    const float x0 = quarter & 1 ? c : s, x1 = quarter & 1 ? s : c;
    sine = quarter & 2 ? -x0 : x0;
    cosine = quarter == 1 || quarter == 2 ? -x1 : x1;
}

// Turns the lane's pairs by the angles, or back.
__device__ __forceinline__ void turn(const Places& p, bool interleaved, const float (&cosine)[4],
                                     const float (&sine)[4], float sign, float (&x)[8]) {
    if (!p.pairs) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float xa = interleaved ? x[2 * j] : x[j], xb = interleaved ? x[2 * j + 1] : x[4 + j];
        const float s = sign * sine[j];
        const float ya = __builtin_fmaf(xa, cosine[j], -(xb * s));
        const float yb = __builtin_fmaf(xb, cosine[j], xa * s);
        // Written once for each layout: an index that depends on it would put x into memory.
        x[2 * j] = interleaved ? ya : x[2 * j];
        x[2 * j + 1] = interleaved ? yb : x[2 * j + 1];
        if (!interleaved) {
            x[j] = ya;
            x[4 + j] = yb;
        }
    }
}

template <int CONTROL>
__device__ __forceinline__ float moved(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CONTROL, 15, 15, true));
}

// The sum over a head's G lanes, in each of them.
template <int G>
__device__ __forceinline__ float head_sum(float x) {
    x += moved<0xb1>(x);                // quad_perm 1 0 3 2
    x += moved<0x4e>(x);                // quad_perm 2 3 0 1
    if (G > 4) x += moved<0x141>(x);    // row_half_mirror
    if (G > 8) x += moved<0x140>(x);    // row_mirror
    if (G > 16) x += __shfl_xor(x, 16);
    if (G > 32) x += __shfl_xor(x, 32);
    return x;
}

// A wave has `per` heads of a token, 64 / G at a time, each in G lanes of eight values, or all heads
// of several tokens. The lanes of a head read all of it before they write, so the output may be the
// input.
template <int G, bool BACK>
__global__ __launch_bounds__(kThreads) void norm_rotate(Args a) {
    constexpr int kSlots = 64 / G;
    const int lane = int(threadIdx.x) & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int slot = lane / G, u = lane % G;
    const Places p = places(a, u);
    const int sub = a.each > 1 ? slot / a.total_heads : 0;  // the slot's token and head
    const int head = slot - sub * a.total_heads;
    const float each = 1.0f / float(a.dim);
    float dw[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.0f;
    for (int64_t unit = int64_t(blockIdx.x) * kWaves + wave; unit < a.units;
         unit += int64_t(gridDim.x) * kWaves) {
        const int64_t t = unit / a.chunks * a.each + sub;
        const int first = int(unit % a.chunks) * a.per;
        const int end = sub < a.each && t < a.tokens ? min(first + a.per, a.total_heads) : 0;
        float cosine[4], sine[4];
        if (a.half > 0) {
            const double at = double(a.positions[t < a.tokens ? t : a.tokens - 1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * u + j;
                sine_cosine(at * a.freqs[i < a.half ? i : 0], sine[j], cosine[j]);
            }
        }
        for (int h = first + head; h < end; h += kSlots) {
            const bool key = h >= a.heads;
            // Chosen field by field: a reference to either would be read through memory.
            const Side side{key ? a.k.x : a.q.x,         key ? a.k.grad : a.q.grad,
                            key ? a.k.weight : a.q.weight, key ? a.k.out : a.q.out,
                            key ? a.k.ld : a.q.ld,       key ? a.k.ld_grad : a.q.ld_grad,
                            key ? a.k.ld_out : a.q.ld_out};
            const int64_t column = int64_t(key ? h - a.heads : h) * a.dim;
            float x[8], w[8], g[8];
            const bool norm = side.weight != nullptr;
            if (!BACK || norm) load8(side.x + t * side.ld + column, p, x);
            if (BACK) load8(side.grad + t * side.ld_grad + column, p, g);
            if (norm) load8(side.weight, p, w);
            float r = 1.0f;
            if (norm) {
                float s = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[e], x[e], s);
                r = 1.0f / sqrtf(__builtin_fmaf(head_sum<G>(s), each, a.eps));
            }
            if (!BACK) {
                if (norm) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
                }
                turn(p, a.interleaved, cosine, sine, 1.0f, x);
                store8(side.out + t * side.ld_out + column, p, x);
                continue;
            }
            turn(p, a.interleaved, cosine, sine, -1.0f, g);
            if (norm) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] *= r;
                    const float y = g[e] * x[e];
                    dw[0][e] += key ? 0.0f : y;
                    dw[1][e] += key ? y : 0.0f;
                    g[e] *= w[e];
                    m = __builtin_fmaf(g[e], x[e], m);
                }
                m = head_sum<G>(m) * each;
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = r * __builtin_fmaf(-x[e], m, g[e]);
            }
            if (side.out != nullptr) store8(side.out + t * side.ld_out + column, p, g);
        }
    }
    if (!BACK || a.parts == nullptr) return;
    // The block's share: its heads' lanes of the same values.
    __shared__ float sh[kWaves][2][kMaxDim + 8];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float x = dw[s][e];
#pragma unroll
            for (int d = G; d < 64; d *= 2) x += __shfl_xor(x, d);
            dw[s][e] = x;
        }
        if (slot == 0) store8(sh[wave][s], p, dw[s]);
    }
    __syncthreads();
    for (int i = int(threadIdx.x); i < 2 * a.dim; i += kThreads) {
        const int s = i >= a.dim, d = s ? i - a.dim : i;
        float x = sh[0][s][d];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) x += sh[v][s][d];
        a.parts[int64_t(blockIdx.x) * 2 * a.dim + i] = x;
    }
}

// The weights' gradients from the blocks' shares, in their order: sixteen columns a
// block, sixty-four threads of shares each.
constexpr int kJoinThreads = 1024;

__global__ __launch_bounds__(kJoinThreads) void norm_rotate_join(const float* __restrict__ parts,
                                                             int count, int dim, float* dq,
                                                             float* dk) {
    __shared__ float sh[kJoinThreads];
    const int column = int(blockIdx.x) * 16 + int(threadIdx.x) % 16, share = int(threadIdx.x) / 16;
    float x = 0.0f;
    if (column < 2 * dim) {
#pragma unroll 8
        for (int b = share; b < count; b += kJoinThreads / 16)
            x += parts[int64_t(b) * 2 * dim + column];
    }
    sh[threadIdx.x] = x;
    __syncthreads();
    if (share != 0 || column >= 2 * dim) return;
#pragma unroll
    for (int s = 1; s < kJoinThreads / 16; ++s) x += sh[s * 16 + int(threadIdx.x)];
    float* const out = column < dim ? dq : dk;
    if (out != nullptr) out[column < dim ? column : column - dim] = x;
}

// ---------------------------------------------------------------- host checks

constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;

int check(const char* name, const ehip_norm_rotate_t* d) {
    if (d == nullptr) return fail(EHIP_EINVAL, "%s: null descriptor", name);
    if (d->tokens < 0 || d->heads < 0 || d->kv_heads < 0 || d->heads + d->kv_heads < 1 ||
        d->head_dim < 1 || d->head_dim > kMaxDim || d->rotary < 0 || d->rotary > d->head_dim ||
        d->rotary % 2 != 0 || !(d->eps >= 0.0f))
        return fail(EHIP_EINVAL,
                    "%s: %lld tokens of %lld and %lld heads of %lld values, %lld rotated, eps %g",
                    name, (long long)d->tokens, (long long)d->heads, (long long)d->kv_heads,
                    (long long)d->head_dim, (long long)d->rotary, double(d->eps));
    if (d->tokens > INT32_MAX || d->heads > kMaxBlocks || d->kv_heads > kMaxBlocks)
        return fail(EHIP_EINVAL, "%s: extents past the index range", name);
    if (d->ld_q < d->heads * d->head_dim || d->ld_k < d->kv_heads * d->head_dim)
        return fail(EHIP_EINVAL, "%s: leading dimension below the row's length", name);
    return EHIP_OK;
}

int check_tensors(const char* name, const ehip_norm_rotate_t* d) {
    if ((d->heads > 0 && d->q == nullptr) || (d->kv_heads > 0 && d->k == nullptr) ||
        (d->rotary > 0 && (d->positions == nullptr || d->freqs == nullptr)))
        return fail(EHIP_EINVAL, "%s: null tensor", name);
    return EHIP_OK;
}

int lanes_of(const Args& a) {
    const int units = (a.half + 3) / 4 + (a.dim - 2 * a.half + 7) / 8;
    int g = 4;
    while (g < units) g *= 2;
    return g;
}

Args arguments(const ehip_norm_rotate_t* d) {
    Args a{};
    a.q = Side{d->q, nullptr, d->q_weight, nullptr, d->ld_q, 0, 0};
    a.k = Side{d->k, nullptr, d->k_weight, nullptr, d->ld_k, 0, 0};
    a.heads = int(d->heads);
    a.total_heads = int(d->heads + d->kv_heads);
    a.dim = int(d->head_dim);
    a.half = int(d->rotary / 2);
    a.interleaved = d->interleaved != 0;
    a.positions = d->positions;
    a.freqs = d->freqs;
    a.eps = d->eps;
    // Shares of a token for some 16 waves a CU; one share's heads share the angles.
    const int slots = 64 / lanes_of(a);
    const int64_t most = ceil_div(a.total_heads, slots);
    const int64_t want = std::min(most, ceil_div(4096, std::max<int64_t>(1, d->tokens)));
    a.per = int(ceil_div(most, want)) * slots;
    a.chunks = int(ceil_div(a.total_heads, a.per));
    // Tokens whose heads leave half of a wave or more without work share it (65536 tokens, us, a
    // wave a token : like this; two heads of 24 values 43 : 13, of 64 44 : 17, of 128 44 : 29; four
    // of 64 with the gradient 114 : 75).
    a.each = std::max(1, slots / a.total_heads);
    a.tokens = d->tokens;
    a.units = ceil_div(d->tokens, a.each) * a.chunks;
    return a;
}

int64_t blocks_of(const Args& a) {
    return std::min<int64_t>(kMaxParts, ceil_div(a.units, kWaves));
}

template <bool BACK>
int launch(const Args& a, hipStream_t s) {
    const int64_t blocks = BACK ? blocks_of(a) : std::min(kMaxBlocks, ceil_div(a.units, kWaves));
    const dim3 grid{unsigned(blocks)}, block{kThreads};
    const char* name = BACK ? "norm_rotate_backward" : "norm_rotate";
    switch (lanes_of(a)) {
        case 4: EHIP_LAUNCH(name, (norm_rotate<4, BACK>), grid, block, 0, s, a); break;
        case 8: EHIP_LAUNCH(name, (norm_rotate<8, BACK>), grid, block, 0, s, a); break;
        case 16: EHIP_LAUNCH(name, (norm_rotate<16, BACK>), grid, block, 0, s, a); break;
        case 32: EHIP_LAUNCH(name, (norm_rotate<32, BACK>), grid, block, 0, s, a); break;
        default: EHIP_LAUNCH(name, (norm_rotate<64, BACK>), grid, block, 0, s, a);
    }
    return EHIP_OK;
}

// Bytes of the blocks' shares, where a weight has a gradient.
size_t part_bytes(const Args& a) {
    return a.q.weight != nullptr || a.k.weight != nullptr
               ? size_t(blocks_of(a)) * 2 * size_t(a.dim) * sizeof(float)
               : 0;
}

}  // namespace
}  // namespace ehip

using namespace ehip;

extern "C" {

int ehip_norm_rotate_f32(const ehip_norm_rotate_t* desc, float* q_out, int64_t ld_q_out,
                         float* k_out, int64_t ld_k_out, void* stream) {
    EHIP_READY();
    if (int rc = check("norm_rotate", desc)) return rc;
    if (ld_q_out < desc->heads * desc->head_dim || ld_k_out < desc->kv_heads * desc->head_dim)
        return fail(EHIP_EINVAL, "norm_rotate: leading dimension below the row's length");
    if (desc->tokens == 0) return EHIP_OK;
    if (int rc = check_tensors("norm_rotate", desc)) return rc;
    if ((desc->heads > 0 && q_out == nullptr) || (desc->kv_heads > 0 && k_out == nullptr))
        return fail(EHIP_EINVAL, "norm_rotate: null tensor");
    Args a = arguments(desc);
    a.q.out = q_out;
    a.q.ld_out = ld_q_out;
    a.k.out = k_out;
    a.k.ld_out = ld_k_out;
    return launch<false>(a, as_stream(stream));
}

int64_t ehip_norm_rotate_backward_workspace(const ehip_norm_rotate_t* desc) {
    if (check("norm_rotate_backward", desc)) return -1;
    return desc->tokens == 0 ? 0 : int64_t(part_bytes(arguments(desc)));
}

int ehip_norm_rotate_backward_f32(const ehip_norm_rotate_t* desc, const float* grad_q,
                                  int64_t ld_grad_q, const float* grad_k, int64_t ld_grad_k,
                                  float* dq, int64_t ld_dq, float* dk, int64_t ld_dk,
                                  float* dq_weight, float* dk_weight, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    EHIP_READY();
    if (int rc = check("norm_rotate_backward", desc)) return rc;
    const int64_t row_q = desc->heads * desc->head_dim, row_k = desc->kv_heads * desc->head_dim;
    if (ld_grad_q < row_q || ld_grad_k < row_k || (dq != nullptr && ld_dq < row_q) ||
        (dk != nullptr && ld_dk < row_k))
        return fail(EHIP_EINVAL, "norm_rotate_backward: leading dimension below the row's length");
    if ((dq_weight != nullptr && desc->q_weight == nullptr) ||
        (dk_weight != nullptr && desc->k_weight == nullptr))
        return fail(EHIP_EINVAL, "norm_rotate_backward: the gradient of a weight that is not there");
    hipStream_t s = as_stream(stream);
    if (desc->tokens > 0) {
        if (int rc = check_tensors("norm_rotate_backward", desc)) return rc;
        if ((desc->heads > 0 && grad_q == nullptr) || (desc->kv_heads > 0 && grad_k == nullptr))
            return fail(EHIP_EINVAL, "norm_rotate_backward: null tensor");
    }
    Args a = arguments(desc);
    const bool weights = dq_weight != nullptr || dk_weight != nullptr;
    const size_t need = weights && desc->tokens > 0 ? part_bytes(a) : 0;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
        return fail(EHIP_EINVAL,
                    "norm_rotate_backward: needs %zu bytes of 16-byte aligned workspace", need);
    if (desc->tokens > 0) {
        a.q.grad = grad_q;
        a.q.ld_grad = ld_grad_q;
        a.q.out = dq;
        a.q.ld_out = ld_dq;
        a.k.grad = grad_k;
        a.k.ld_grad = ld_grad_k;
        a.k.out = dk;
        a.k.ld_out = ld_dk;
        a.parts = weights ? static_cast<float*>(workspace) : nullptr;
        if (int rc = launch<true>(a, s)) return rc;
    }
    if (weights)
        EHIP_LAUNCH("norm_rotate_backward_join", norm_rotate_join,
                    dim3(unsigned(ceil_div(2 * a.dim, 16))), dim3(kJoinThreads), 0, s, a.parts,
                    desc->tokens > 0 ? int(blocks_of(a)) : 0, a.dim, dq_weight, dk_weight);
    return EHIP_OK;
}

}  // extern "C"
