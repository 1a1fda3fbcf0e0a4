// Log probabilities of given tokens, entropy and top alternatives of rows of logits (nnhip_token_log_probs).
//
// With m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//     ln p[t] = (x_t - m) - ln S,    entropy = ln S - T / S.
// S is a sum in 64 bits: the largest logit adds exactly 1 to it, so S - 1 keeps the digits that the entropy and the log
// probability of a near-certain row consist of.  (T's terms all have one sign: 16 of them meet in FP32, those sums in 64 bits.)
//
// Bound by reading the logits once.  A row is cut into segments for as many workgroups as fill the device; a wave takes
// pieces of 1024 logits of its segment, in rising order, with the next piece on its way, and keeps
//   - m of the wave, S and T of every lane relative to it (a new maximum is rare: the sums are rescaled then);
//   - the best logits so far, sorted, one a lane.  Only a piece whose largest logit exceeds the last of them is looked at
//     again; equal logits keep the order of their indexes because candidates come in rising order and have to be greater.
// A second launch adds the segments of a row up, if there are several.
#include "nnhip_internal.h"

namespace nnhip {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kPiece = 16, kPieceLogits = kPiece * 64;      // logits a lane / a wave has in hand
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;

struct LogProbArgs {
    nnhip_log_probs_desc d;
    int segments, segment;      // segments of a row, logits of one (a multiple of kPieceLogits)
    double* sums;               // [row][segment][2]: S, T
    float* tops;                // [row][segment]: m
    float* values;              // [row][segment][top]
    int32_t* ids;
};

__device__ __forceinline__ float no_number() { return __uint_as_float(0x7fc00000u); }

__device__ __forceinline__ float wave_max(float x)
{
    for (int y = 32; y > 0; y >>= 1) x = fmaxf(x, __shfl_xor(x, y));
    return x;
}
__device__ __forceinline__ double wave_sum(double x)
{
    for (int y = 32; y > 0; y >>= 1) x += __shfl_xor(x, y);
    return x;
}

// The `top` largest logits a wave has seen, sorted, entry i in lane i; empty entries are NaN, which no comparison counts.
struct Best {
    float value;
    int32_t id;
    float last;                 // entry top - 1: what a candidate has to exceed (NaN: there is room)

    __device__ __forceinline__ void clear()
    {
        value = last = no_number();
        id = -1;
    }
    // Offers the logits of the lanes in `mask`, in lane order.
    __device__ __forceinline__ void offer(uint64_t mask, float x, int32_t index, int top)
    {
        const int lane = threadIdx.x & 63;
        while (mask) {
            const int from = __builtin_ctzll(mask);
            mask &= mask - 1;
            float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), from));
            if (v != v) v = INFINITY;                           // in the order a NaN counts as +infinity
            if (v <= last) continue;
            const int32_t i = __builtin_amdgcn_readlane(index, from);
            const int place = __popcll(__ballot(value >= v));
            const float above = __shfl_up(value, 1);
            const int32_t above_id = __shfl_up(id, 1);
            value = lane < place ? value : lane == place ? v : above;
            id = lane < place ? id : lane == place ? i : above_id;
            last = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(value), top - 1));
        }
    }
};

// The sums of some logits relative to m.
struct Sums {
    float m;
    double S, T;

    __device__ __forceinline__ void clear()
    {
        m = kLowest;
        S = T = 0.0;
    }
    __device__ __forceinline__ void rescale(float next)
    {
        if (next == m) return;
        const double by = static_cast<double>(m) - static_cast<double>(next), e = exp(by);
        // (by * S first: by may be -infinity only where e is 0 and S is 0 or not a number)
        T = e == 0.0 ? 0.0 * S : e * (T + by * S);
        S *= e;
        m = next;
    }
};

// The four waves' results -> thread 0's sums and the `top` best of the workgroup in LDS: every candidate counts those that
// come before it.
struct Joined {
    float m[kWaves];
    double S[kWaves], T[kWaves];
    float value[kWaves * NNHIP_LOG_PROBS_MAX_TOP], best[NNHIP_LOG_PROBS_MAX_TOP];
    int32_t id[kWaves * NNHIP_LOG_PROBS_MAX_TOP], best_id[NNHIP_LOG_PROBS_MAX_TOP];
};

__device__ void join_waves(Joined& j, Sums& sums, const Best& best, int top)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    sums.S = wave_sum(sums.S);
    sums.T = wave_sum(sums.T);
    if (lane == 0) {
        j.m[wave] = sums.m;
        j.S[wave] = sums.S;
        j.T[wave] = sums.T;
    }
    if (lane < top) {
        j.value[wave * top + lane] = best.value;
        j.id[wave * top + lane] = best.id;
    }
    __syncthreads();
    const float m = fmaxf(fmaxf(j.m[0], j.m[1]), fmaxf(j.m[2], j.m[3]));
    double S = 0.0, T = 0.0;
    for (int w = 0; w < kWaves; ++w) {
        Sums x{j.m[w], j.S[w], j.T[w]};
        x.rescale(m);
        S += x.S;
        T += x.T;
    }
    sums = Sums{m, S, T};
    if (tid < kWaves * top && j.id[tid] >= 0) {
        const float v = j.value[tid];
        const int32_t id = j.id[tid];
        int before = 0;
        for (int k = 0; k < kWaves * top; ++k)
            before += j.id[k] >= 0 && (j.value[k] > v || (j.value[k] == v && j.id[k] < id)) ? 1 : 0;
        if (before < top) {
            j.best[before] = v;
            j.best_id[before] = id;
        }
    }
    __syncthreads();
}

// Results of one row from the sums over all of it and the best in LDS.
__device__ void write_row(const nnhip_log_probs_desc& d, int row, const Joined& j, const Sums& sums)
{
    const int tid = threadIdx.x;
    const bool defined = sums.S > 0.0 && sums.S < INFINITY;     // (a NaN or +infinity among the logits makes S NaN)
    const double log_sum = log1p(sums.S - 1.0), m = static_cast<double>(sums.m);
    if (tid < d.top) {
        const size_t at = static_cast<size_t>(row) * d.top + tid;
        d.top_ids[at] = j.best_id[tid];
        if (d.top_log_probs) d.top_log_probs[at] = defined ? static_cast<float>((static_cast<double>(j.best[tid]) - m) - log_sum) : no_number();
    }
    if (tid == 128 && d.entropy) d.entropy[row] = defined ? static_cast<float>(log_sum - sums.T / sums.S) : no_number();
    if (tid == 64 && d.log_probs) {
        const int32_t t = d.targets[row];
        float lp = no_number();
        if (defined && t >= 0 && t < d.vocabulary)
            lp = static_cast<float>((static_cast<double>(d.logits[static_cast<int64_t>(row) * d.row_stride + t]) - m) - log_sum);
        d.log_probs[row] = lp;
    }
}

template <bool TOP>
__global__ __launch_bounds__(kThreads) void log_probs_kernel(const LogProbArgs a)
{
    __shared__ Joined joined;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.segments)), part = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.segments));
    const float* x = a.d.logits + static_cast<int64_t>(row) * a.d.row_stride;
    const int64_t first = static_cast<int64_t>(part) * a.segment;
    const int end = static_cast<int>(first + a.segment < a.d.vocabulary ? first + a.segment : a.d.vocabulary);
    Sums sums;
    Best best;
    sums.clear();
    best.clear();
    float now[kPiece], next[kPiece];
    auto fetch = [&](float (&to)[kPiece], int64_t at) {
        if (at + kPieceLogits <= end) {
#pragma unroll
            for (int u = 0; u < kPiece; ++u) to[u] = __builtin_nontemporal_load(x + at + u * 64 + lane);
        } else {
#pragma unroll
            for (int u = 0; u < kPiece; ++u) to[u] = at + u * 64 + lane < end ? x[at + u * 64 + lane] : -INFINITY;
        }
    };
    int64_t at = first + wave * kPieceLogits;
    if (at < end) fetch(now, at);
    for (; at < end; at += kWaves * kPieceLogits) {
        if (at + kWaves * kPieceLogits < end) fetch(next, at + kWaves * kPieceLogits);
        float most = now[0];
#pragma unroll
        for (int u = 1; u < kPiece; ++u) most = fmaxf(most, now[u]);
        if (__any(most > sums.m)) sums.rescale(fmaxf(sums.m, wave_max(most)));
        float t = 0.0f;
#pragma unroll
        for (int u = 0; u < kPiece; ++u) {
            const float d = now[u] - sums.m, e = __builtin_amdgcn_exp2f(d * kLog2e);
            sums.S += static_cast<double>(e);
            t = fmaf(fmaxf(d, -200.0f), e, t);                  // (e is 0 long before: -infinity times 0 must not come up)
        }
        sums.T += static_cast<double>(t);
        if (TOP && __any(!(most <= best.last) || t != t)) {
#pragma unroll
            for (int u = 0; u < kPiece; ++u) {
                const int64_t index = at + u * 64 + lane;
                best.offer(__ballot(index < end && !(now[u] <= best.last)), now[u], static_cast<int32_t>(index), a.d.top);
            }
        }
#pragma unroll
        for (int u = 0; u < kPiece; ++u) now[u] = next[u];
    }
    join_waves(joined, sums, best, TOP ? a.d.top : 0);
    if (a.segments == 1) {
        write_row(a.d, row, joined, sums);
        return;
    }
    if (threadIdx.x == 0) {
        a.tops[blockIdx.x] = sums.m;
        a.sums[2 * static_cast<size_t>(blockIdx.x)] = sums.S;
        a.sums[2 * static_cast<size_t>(blockIdx.x) + 1] = sums.T;
    }
    if (TOP && static_cast<int>(threadIdx.x) < a.d.top) {
        const bool there = static_cast<int>(threadIdx.x) < end - first;         // the last segment may hold fewer than `top`
        const size_t to = static_cast<size_t>(blockIdx.x) * a.d.top + threadIdx.x;
        a.values[to] = there ? joined.best[threadIdx.x] : 0.0f;
        a.ids[to] = there ? joined.best_id[threadIdx.x] : -1;
    }
}

// The segments of one row: their sums, and their best as candidates in the order of the segments.
__global__ __launch_bounds__(kThreads) void log_probs_join_kernel(const LogProbArgs a)
{
    __shared__ Joined joined;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t from = static_cast<size_t>(blockIdx.x) * a.segments;
    Sums sums;
    Best best;
    sums.clear();
    best.clear();
    float m = kLowest;
    for (int k = tid; k < a.segments; k += kThreads) m = fmaxf(m, a.tops[from + k]);
    sums.m = wave_max(m);
    for (int k = tid; k < a.segments; k += kThreads) {
        Sums x{a.tops[from + k], a.sums[2 * (from + k)], a.sums[2 * (from + k) + 1]};
        x.rescale(sums.m);
        sums.S += x.S;
        sums.T += x.T;
    }
    const int all = a.segments * a.d.top, each = ((all + kWaves - 1) / kWaves + 63) / 64 * 64;
    for (int k0 = wave * each; k0 < all && k0 < (wave + 1) * each; k0 += 64) {
        const int k = k0 + lane;
        const size_t at = static_cast<size_t>(blockIdx.x) * all + k;
        const float v = k < all ? a.values[at] : 0.0f;
        const int32_t id = k < all ? a.ids[at] : -1;
        best.offer(__ballot(id >= 0 && !(v <= best.last)), v, id, a.d.top);
    }
    join_waves(joined, sums, best, a.d.top);
    write_row(a.d, blockIdx.x, joined, sums);
}

}  // namespace

LogProbPlan plan_token_log_probs(const nnhip_log_probs_desc& d, int compute_units)
{
    // Eight workgroups of four waves a compute unit, none with less than a piece for each wave where the row allows it.
    LogProbPlan p{};
    const int64_t pieces = (static_cast<int64_t>(d.vocabulary) + kPieceLogits - 1) / kPieceLogits;
    int64_t segments = 8 * static_cast<int64_t>(compute_units) / d.rows;
    if (segments > (pieces + kWaves - 1) / kWaves) segments = (pieces + kWaves - 1) / kWaves;
    if (segments < 1) segments = 1;
    const int64_t each = (pieces + segments - 1) / segments;
    p.segment = static_cast<int>(each * kPieceLogits < 0x7fffffff ? each * kPieceLogits : 0x7fffffff / kPieceLogits * kPieceLogits);
    p.segments = static_cast<int>((static_cast<int64_t>(d.vocabulary) + p.segment - 1) / p.segment);
    if (p.segments > 1) p.scratch_bytes = static_cast<size_t>(d.rows) * p.segments * (16 + 4 + 8 * static_cast<size_t>(d.top));
    return p;
}

hipError_t launch_token_log_probs(Lane* lane, const nnhip_log_probs_desc& d, const LogProbPlan& p, void* scratch)
{
    const size_t parts = static_cast<size_t>(d.rows) * p.segments;
    LogProbArgs a{d, p.segments, p.segment, static_cast<double*>(scratch), nullptr, nullptr, nullptr};
    a.tops = reinterpret_cast<float*>(a.sums + 2 * parts);
    a.values = a.tops + parts;
    a.ids = reinterpret_cast<int32_t*>(a.values + parts * d.top);
    if (d.top > 0)
        hipLaunchKernelGGL(log_probs_kernel<true>, dim3(static_cast<unsigned>(parts)), dim3(kThreads), 0, lane->stream, a);
    else
        hipLaunchKernelGGL(log_probs_kernel<false>, dim3(static_cast<unsigned>(parts)), dim3(kThreads), 0, lane->stream, a);
    if (p.segments > 1) hipLaunchKernelGGL(log_probs_join_kernel, dim3(d.rows), dim3(kThreads), 0, lane->stream, a);
    return hipGetLastError();
}

}  // namespace nnhip
