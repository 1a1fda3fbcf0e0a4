// Log probabilities of given tokens, entropy and top alternatives of rows of logits (nnhip_token_log_probs).
//
// With m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//     ln p[t] = (x_t - m) - ln S,    entropy = ln S - T / S.
// S is a sum in 64 bits: the largest logit adds exactly 1 to it, so S - 1 keeps the digits that the entropy and the log
// probability of a near-certain row consist of.  (T's terms all have one sign: 16 of them meet in FP32, those sums in 64 bits.)
//
// Bound by reading the logits once.  A row is cut into segments for as many workgroups as fill the device; a wave takes
// pieces of 1024 logits of its segment with the next piece on its way, keeps its maximum m, the sums S and T of every lane
// relative to it (a new maximum is rare: the sums are rescaled then), and writes down each piece's largest logit.
//
// The `top` best logits of a row lie in the `top` pieces with the largest maxima (equal maxima by index): any other piece has
// that many pieces before it, each with a logit that goes before all of its own.  So one workgroup a row picks those pieces and
// looks at them again, a few KB of the row, with the least of their maxima as the threshold: about as many logits pass as
// are wanted.  Keeping sorted candidates during the streaming pass instead cost eight times its memory time for 20 of
// 262144 (92 us for 32 rows).
#include "nnhip_internal.h"

namespace nnhip {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kHand = 16, kHandLogits = kHand * 64;         // logits a lane / a wave has in hand
constexpr int kMaxPieces = 512;                             // pieces of a row: 1024 logits each, more in rows above 524288
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;

struct LogProbArgs {
    nnhip_log_probs_desc d;
    int segments;               // of a row
    int64_t segment;            // logits of one (whole pieces)
    int pieces, piece;          // pieces of a row, logits of one (a multiple of kHandLogits)
    double* sums;               // [row][segment][2]: S, T
    float* tops;                // [row][segment]: m
    float* maxima;              // [row][piece]
};

__device__ __forceinline__ float no_number() { return __uint_as_float(0x7fc00000u); }

// Rotations within 16 lanes, then exchanges of 16 and 32: no LDS.
template <int CONTROL>
__device__ __forceinline__ float rotated(float x)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CONTROL, 0xf, 0xf, false));
}
__device__ __forceinline__ float wave_max(float x)
{
    x = fmaxf(x, rotated<0x128>(x));
    x = fmaxf(x, rotated<0x124>(x));
    x = fmaxf(x, rotated<0x122>(x));
    x = fmaxf(x, rotated<0x121>(x));
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
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

struct Joined {
    float m[kWaves];
    double S[kWaves], T[kWaves];
    float maxima[kMaxPieces];
    float value[kWaves * NNHIP_LOG_PROBS_MAX_TOP], best[NNHIP_LOG_PROBS_MAX_TOP];
    int32_t id[kWaves * NNHIP_LOG_PROBS_MAX_TOP], best_id[NNHIP_LOG_PROBS_MAX_TOP];
    int32_t chosen[NNHIP_LOG_PROBS_MAX_TOP], counts[kMaxPieces / 64];
    float threshold;
};

// The sums of the four waves, in their order; every thread gets them.
__device__ void join_sums(Joined& j, Sums& sums)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    sums.S = wave_sum(sums.S);
    sums.T = wave_sum(sums.T);
    if (lane == 0) {
        j.m[wave] = sums.m;
        j.S[wave] = sums.S;
        j.T[wave] = sums.T;
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
}

// The `top` best logits of a row whose pieces' maxima are in LDS -> j.best, j.best_id, in their order.
__device__ void find_best(Joined& j, const LogProbArgs& a, const float* x)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), top = a.d.top, pieces = a.pieces;
    const int wanted = top < pieces ? top : pieces;
    if (tid == 0) j.threshold = -INFINITY;                      // (fewer pieces than alternatives: every logit counts)
    __syncthreads();
    bool chosen[kMaxPieces / kThreads];
#pragma unroll
    for (int r = 0; r < kMaxPieces / kThreads; ++r) {
        const int p = r * kThreads + tid;
        chosen[r] = false;
        if (p < pieces) {                                       // the piece's place among all
            const float v = j.maxima[p];
            int before = 0;
            for (int q = 0; q < pieces; ++q) before += j.maxima[q] > v || (j.maxima[q] == v && q < p) ? 1 : 0;
            chosen[r] = before < wanted;
            if (before == wanted - 1 && wanted == top) j.threshold = v;
        }
        const uint64_t mask = __ballot(chosen[r]);
        if (lane == 0) j.counts[r * kWaves + wave] = __popcll(mask);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kMaxPieces / kThreads; ++r) {           // in rising order
        const uint64_t mask = __ballot(chosen[r]);
        int at = __popcll(mask & ((1ull << lane) - 1));
        for (int w = 0; w < r * kWaves + wave; ++w) at += j.counts[w];
        if (chosen[r]) j.chosen[at] = r * kThreads + tid;
    }
    __syncthreads();
    const float threshold = j.threshold;
    Best best;
    best.clear();
    for (int c = wave; c < wanted; c += kWaves) {
        const int64_t begin = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(j.chosen[c])) * a.piece;
        const int64_t end = begin + a.piece < a.d.vocabulary ? begin + a.piece : a.d.vocabulary;
        for (int64_t at = begin; at < end; at += kHandLogits) {
            float now[kHand];
#pragma unroll
            for (int u = 0; u < kHand; ++u) now[u] = at + u * 64 + lane < end ? x[at + u * 64 + lane] : 0.0f;
#pragma unroll
            for (int u = 0; u < kHand; ++u) {
                const int64_t index = at + u * 64 + lane;
                best.offer(__ballot(index < end && !(now[u] < threshold) && !(now[u] <= best.last)), now[u], static_cast<int32_t>(index), top);
            }
        }
    }
    if (lane < top) {
        j.value[wave * top + lane] = best.value;
        j.id[wave * top + lane] = best.id;
    }
    __syncthreads();
    if (tid < kWaves * top && j.id[tid] >= 0) {                 // a candidate's place among those of the four waves
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

__global__ __launch_bounds__(kThreads) void log_probs_kernel(const LogProbArgs a)
{
    __shared__ Joined joined;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.segments)), part = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.segments));
    const float* x = a.d.logits + static_cast<int64_t>(row) * a.d.row_stride;
    const int64_t first = static_cast<int64_t>(part) * a.segment;
    const int64_t end = first + a.segment < a.d.vocabulary ? first + a.segment : a.d.vocabulary;
    Sums sums;
    sums.clear();
    float now[kHand], next[kHand];
    auto fetch = [&](float (&to)[kHand], int64_t at) {
        const float* from = x + at;
        if (at + kHandLogits <= end) {
#pragma unroll
            for (int u = 0; u < kHand; ++u) to[u] = __builtin_nontemporal_load(from + u * 64 + lane);
        } else {
            const int left = static_cast<int>(end - at);
#pragma unroll
            for (int u = 0; u < kHand; ++u) to[u] = u * 64 + lane < left ? from[u * 64 + lane] : -INFINITY;
        }
    };
    // wave w takes the pieces w, w + 4, ... of the segment
    const int64_t step = static_cast<int64_t>(kWaves - 1) * a.piece;
    int64_t at = first + static_cast<int64_t>(wave) * a.piece, piece_end = at + a.piece;
    float largest = -INFINITY;
    if (at < end) fetch(now, at);
    while (at < end) {
        const int64_t following = at + kHandLogits == piece_end ? piece_end + step : at + kHandLogits;
        if (following < end) fetch(next, following);
        float most = now[0];
#pragma unroll
        for (int u = 1; u < kHand; ++u) most = fmaxf(most, now[u]);
        most = wave_max(most);
        if (most > sums.m) sums.rescale(most);
        float t = 0.0f;
#pragma unroll
        for (int u = 0; u < kHand; ++u) {
            const float d = now[u] - sums.m, e = __builtin_amdgcn_exp2f(d * kLog2e);
            sums.S += static_cast<double>(e);
            t = fmaf(fmaxf(d, -200.0f), e, t);                  // (e is 0 long before: -infinity times 0 must not come up)
        }
        sums.T += static_cast<double>(t);
        if (a.d.top > 0) {
            largest = __any(t != t) ? INFINITY : fmaxf(largest, most);          // a NaN counts as +infinity
            if (following != at + kHandLogits || following >= end) {
                const int piece = static_cast<int>((piece_end - 1) / a.piece);
                if (lane == 0) {
                    if (a.segments == 1)
                        joined.maxima[piece] = largest;
                    else
                        a.maxima[static_cast<size_t>(row) * a.pieces + piece] = largest;
                }
                largest = -INFINITY;
            }
        }
        if (following != at + kHandLogits) piece_end = following + a.piece;
        at = following;
#pragma unroll
        for (int u = 0; u < kHand; ++u) now[u] = next[u];
    }
    join_sums(joined, sums);
    if (a.segments == 1) {
        if (a.d.top > 0) find_best(joined, a, x);
        write_row(a.d, row, joined, sums);
    } else if (threadIdx.x == 0) {
        a.tops[blockIdx.x] = sums.m;
        a.sums[2 * static_cast<size_t>(blockIdx.x)] = sums.S;
        a.sums[2 * static_cast<size_t>(blockIdx.x) + 1] = sums.T;
    }
}

// One row: the sums of its segments, and its best logits.
__global__ __launch_bounds__(kThreads) void log_probs_join_kernel(const LogProbArgs a)
{
    __shared__ Joined joined;
    const int tid = threadIdx.x;
    const size_t from = static_cast<size_t>(blockIdx.x) * a.segments;
    if (a.d.top > 0)
        for (int p = tid; p < a.pieces; p += kThreads) joined.maxima[p] = a.maxima[static_cast<size_t>(blockIdx.x) * a.pieces + p];
    Sums sums;
    sums.clear();
    float m = kLowest;
    for (int k = tid; k < a.segments; k += kThreads) m = fmaxf(m, a.tops[from + k]);
    sums.m = wave_max(m);
    for (int k = tid; k < a.segments; k += kThreads) {
        Sums x{a.tops[from + k], a.sums[2 * (from + k)], a.sums[2 * (from + k) + 1]};
        x.rescale(sums.m);
        sums.S += x.S;
        sums.T += x.T;
    }
    join_sums(joined, sums);
    if (a.d.top > 0) find_best(joined, a, a.d.logits + static_cast<int64_t>(blockIdx.x) * a.d.row_stride);
    write_row(a.d, blockIdx.x, joined, sums);
}

}  // namespace

LogProbPlan plan_token_log_probs(const nnhip_log_probs_desc& d, int compute_units)
{
    // Eight workgroups of four waves a compute unit, none with less than a piece for each wave where the row allows it.
    LogProbPlan p{};
    const int64_t V = d.vocabulary, hands = (V + kHandLogits - 1) / kHandLogits;
    const int64_t piece = (hands + kMaxPieces - 1) / kMaxPieces, pieces = (hands + piece - 1) / piece;
    int64_t segments = 8 * static_cast<int64_t>(compute_units) / d.rows;
    if (segments > (pieces + kWaves - 1) / kWaves) segments = (pieces + kWaves - 1) / kWaves;
    if (segments < 1) segments = 1;
    const int64_t each = (pieces + segments - 1) / segments;
    p.piece = static_cast<int>(piece * kHandLogits);
    p.pieces = static_cast<int>(pieces);
    p.segments = static_cast<int>((pieces + each - 1) / each);
    p.segment = each * p.piece;
    if (p.segments > 1) p.scratch_bytes = static_cast<size_t>(d.rows) * (20 * static_cast<size_t>(p.segments) + 4 * static_cast<size_t>(pieces));
    return p;
}

hipError_t launch_token_log_probs(Lane* lane, const nnhip_log_probs_desc& d, const LogProbPlan& p, void* scratch)
{
    const size_t parts = static_cast<size_t>(d.rows) * p.segments;
    LogProbArgs a{d, p.segments, p.segment, p.pieces, p.piece, static_cast<double*>(scratch), nullptr, nullptr};
    if (scratch) {
        a.tops = reinterpret_cast<float*>(a.sums + 2 * parts);
        a.maxima = a.tops + parts;
    }
    hipLaunchKernelGGL(log_probs_kernel, dim3(static_cast<unsigned>(parts)), dim3(kThreads), 0, lane->stream, a);
    if (p.segments > 1) hipLaunchKernelGGL(log_probs_join_kernel, dim3(d.rows), dim3(kThreads), 0, lane->stream, a);
    return hipGetLastError();
}

}  // namespace nnhip
