// attention_shared.hip -- attention of one new token per sequence over the paged cache where the
// sequences of a group share their first positions (answers to one prompt): those are passed once
// for the group, by all of its sequences' query heads together, each sequence's own after them, and
// the parts of both joined.

#include "attention_paged.hpp"

namespace ehip {

using namespace paged;

namespace {

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

// Whole answers for rows without a shared part, joined ones for the others. Thread d % 128 has a
// value, two threads for alternate parts.
__global__ __launch_bounds__(256) void shared_join(Paged own, Paged a) {
    __shared__ float sh[2][kMaxDim], sh_l[2];
    const int64_t at = blockIdx.x, s = at / a.heads;
    const int h = int(at % a.heads), dim = int(a.c.dim);
    const int d = int(threadIdx.x) % kMaxDim, half = int(threadIdx.x) / kMaxDim;
    const int n = length_of(own, s), start = start_of(own, s);
    if (n <= 0) {
        if (half == 0 && d < dim)
            a.out[s * a.ld_out + int64_t(h) * dim + d] = n < 0 ? NAN : 0.0f;
        if (threadIdx.x == 0 && a.lse != nullptr) a.lse[at] = n < 0 ? NAN : -INFINITY;
        return;
    }
    // The parts of the sequence's own positions.
    int parts = 0;
    int64_t from = 0;
    if (n > start) {
        const int tiles = own.first[a.c.sequences];
        const int w0 = worker_of(own, own.first[s], tiles);
        parts = worker_of(own, own.first[s + 1] - 1, tiles) - w0 + 1;
        if (start == 0 && parts == 1) return;  // the sequence was one segment
        from = int64_t(h) * (own.workers + a.c.sequences) + w0 + s;
    }
    // Those of the group's.
    int shared_parts = 0;
    int64_t shared_from = 0;
    if (start > 0) {
        const int lo = group_of(a.group_cu, a.groups, int(s));
        const int group = a.heads / int(a.c.kv_heads), kv = h / group;
        const int row = int(s - group_begin(a, lo)) * group + h % group;
        const int tile = row / a.rows, each = tiles_of(a, shared_of(a, lo));
        const int tiles = a.first[a.groups], t0 = a.first[lo] + tile * each;
        const int w0 = worker_of(a, t0, tiles);
        shared_parts = worker_of(a, t0 + each - 1, tiles) - w0 + 1;
        const int place = w0 + row_tile_base(a, lo) + tile;
        shared_from = (int64_t(kv) * a.places + place) * a.rows + row % a.rows;
    }
    const float2* const stats = own.part_stats + from;
    const float2* const shared_stats = a.part_stats + shared_from;
    float top = -INFINITY;
    for (int i = int(threadIdx.x) & 63; i < parts; i += 64) top = fmaxf(top, stats[i].x);
    for (int i = int(threadIdx.x) & 63; i < shared_parts; i += 64)
        top = fmaxf(top, shared_stats[int64_t(i) * a.rows].x);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    float sum = 0.0f, y = 0.0f;
    const auto add = [&](const float2& z, float value) {
        const float keep = z.x == -INFINITY ? (z.y != z.y ? NAN : 0.0f)
                                            : __builtin_amdgcn_exp2f(z.x - top);
        sum += z.y * keep;
        y = __builtin_fmaf(value, keep, y);
    };
    const int column = d < dim ? d : 0;
#pragma unroll 8
    for (int i = half; i < parts; i += 2)
        add(stats[i], own.part_out[(from + i) * dim + column]);
#pragma unroll 8
    for (int i = half; i < shared_parts; i += 2)
        add(shared_stats[int64_t(i) * a.rows],
            a.part_out[(shared_from + int64_t(i) * a.rows) * dim + column]);
    sh[half][d] = y;
    if (d == 0) sh_l[half] = sum;
    __syncthreads();
    if (half != 0) return;
    sum = sh_l[0] + sh_l[1];
    y += sh[1][d];
    if (d < dim) a.out[s * a.ld_out + int64_t(h) * dim + d] = y / sum;
    if (d == 0 && a.lse != nullptr) a.lse[at] = lse_of(top, sum);
}

// One block. The groups' offsets, in range and ascending whatever came in; what each shares, nothing
// where it has no two sequences or the number is none that its table row could have; the sequences'
// first own positions, 0 for those of no group or shorter than what theirs shares.
__global__ __launch_bounds__(kPlanThreads) void shared_plan(Paged a, const int32_t* group_cu,
                                                            const int32_t* shared,
                                                            int longest_shared, int* cu,
                                                            int* counts, int* starts) {
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
        int start = 0;
        if (a.groups > 0) {
            const int g = group_of(cu, a.groups, s);
            if (cu[g] <= s && s < cu[g + 1] && length_of(a, s) >= counts[g]) start = counts[g];
        }
        starts[s] = start;
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

struct Plan {
    Cut own, shared;
    int rows, places;
    size_t own_bytes, part_bytes, first_bytes, bytes;
};

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

Plan plan_of(const Cache& c, int type, int64_t heads, int64_t longest, int64_t groups,
             int64_t longest_shared) {
    Plan p{};
    p.own = cut_of(c, heads, longest, type);
    const bool waves = p.own.waves;
    p.rows = waves ? 16 : kMaxGroup;
    const int64_t row_tiles = c.sequences * (heads / c.kv_heads) / p.rows + groups;
    const int tile = tile_of(waves, row_tiles, longest_shared);
    const int64_t most = std::max<int64_t>(1, row_tiles * ceil_div(longest_shared, tile));
    const int64_t resident = waves ? 2048 : 512;
    p.shared = Cut{waves, tile,
                   int(std::min(most, std::max<int64_t>(1, resident / c.kv_heads)))};
    p.places = int(p.shared.workers + row_tiles + 1);
    p.own_bytes = round16(part_bytes(c, heads, p.own.workers));
    p.part_bytes = round16(size_t(c.kv_heads) * size_t(p.places) * size_t(p.rows) *
                           (sizeof(float2) + size_t(c.dim) * sizeof(float)));
    // The parts of both; the groups' first tiles, offsets and shared positions, and the sequences'
    // own starts.
    p.first_bytes = round16(size_t(groups + 1) * sizeof(int));
    p.bytes = p.own_bytes + p.part_bytes + 3 * p.first_bytes + size_t(c.sequences) * sizeof(int);
    return p;
}

template <class T, int LPP, bool VEC>
int launch_vector(const Paged& a, hipStream_t s) {
    EHIP_LAUNCH("attention_shared", (paged_part<T, LPP, kMaxGroup, VEC, true>),
                dim3(unsigned(a.workers * a.c.kv_heads)), dim3(kPagedThreads), 0, s, a);
    return EHIP_OK;
}

template <class T, bool VEC>
int launch_lanes(const Paged& a, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    if (a.c.dim <= 32) return launch_vector<T, 32 / N, VEC>(a, s);
    if (a.c.dim <= 64) return launch_vector<T, 64 / N, VEC>(a, s);
    return launch_vector<T, 128 / N, VEC>(a, s);
}

template <class T, int DP, bool WIDE>
int launch_part_mfma(const Paged& a, hipStream_t s) {
    EHIP_LAUNCH("attention_shared", (paged_part_mfma<T, DP, WIDE, true>),
                dim3(unsigned(ceil_div(a.workers * a.c.kv_heads, kPagedWaves))), dim3(kPagedThreads), 0, s, a);
    return EHIP_OK;
}

template <class T, bool WIDE>
int launch_mfma(const Paged& a, hipStream_t s) {
    if (a.c.dim <= 32) return launch_part_mfma<T, 32, WIDE>(a, s);
    if (a.c.dim <= 64) return launch_part_mfma<T, 64, WIDE>(a, s);
    return launch_part_mfma<T, 128, WIDE>(a, s);
}

// Reads of whole pieces in 8 bits: of 16 values, or of 8 in heads of up to 32.
int launch_parts_i8(const Paged& a, bool aligned, hipStream_t s) {
    return aligned && a.c.dim % (a.c.dim <= 32 ? 8 : 16) == 0 ? launch_mfma<Int8, true>(a, s)
                                                              : launch_mfma<Int8, false>(a, s);
}

int launch_shared(const Paged& a, int type, hipStream_t s) {
    const bool aligned = aligned16(a.c.k) && aligned16(a.c.v);
    if (type == EHIP_CACHE_I8) return launch_parts_i8(a, aligned, s);
    if (type == EHIP_CACHE_BF16)
        return by_waves(a.c, type) ? launch_mfma<Bf16, true>(a, s)
                                   : launch_lanes<Bf16, false>(a, s);
    return aligned && a.c.dim % 4 == 0 ? launch_lanes<float, true>(a, s)
                                       : launch_lanes<float, false>(a, s);
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
    a.group_cu = cu;
    a.shared = counts;
    own.starts = starts;
    hipStream_t s = as_stream(stream);
    EHIP_LAUNCH("attention_shared_plan", shared_plan, dim3(1), dim3(kPlanThreads), 0, s, a,
                group_cu, shared, int(longest_shared), cu, counts, starts);
    if (groups > 0)
        if (int rc = launch_shared(a, cache->type, s)) return rc;
    if (int rc = launch_parts(own, cache->type, s)) return rc;
    EHIP_LAUNCH("attention_shared_join", shared_join, dim3(unsigned(c.sequences * heads)),
                dim3(256), 0, s, own, a);
    return EHIP_OK;
}

}  // extern "C"
