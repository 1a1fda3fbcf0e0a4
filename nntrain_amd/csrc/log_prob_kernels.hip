// Log probabilities of given tokens, entropy and top alternatives of rows of logits (nnhip_token_log_probs).
//
// With m = max x, R = sum e^(x - m) over all logits but one that is m, T = sum (x - m) e^(x - m):
//     ln p[t] = (x_t - m) - ln(1 + R),    entropy = ln(1 + R) - T / (1 + R).
// The log probability and the entropy of a near-certain row consist of R alone, so the 1 of the largest logit never enters a
// sum: a wave leaves out one logit equal to its maximum, takes it in when a greater one comes, and so do waves and segments
// where their sums meet.  (T's terms all have one sign: 16 of them meet in FP32, those sums in 64 bits.)
//
// Bound by reading the logits once.  A row is cut into segments for as many workgroups as fill the device; a wave takes
// pieces of 1024 logits of its segment with the next piece on its way, keeps its maximum m, the sums R and T of every lane
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
constexpr float kLn2 = 0.693147180559945309417f, kLn2Low = static_cast<float>(0.693147180559945309417 - static_cast<double>(kLn2));
constexpr float kLowest = -3.402823466e38f;

struct LogProbArgs {
    nnhip_log_probs_desc d;
    int segments;               // of a row
    int64_t segment;            // logits of one (whole pieces)
    int pieces, piece;          // pieces of a row, logits of one (a multiple of kHandLogits)
    double* sums;               // [row][segment][2]: R, T
    float* tops;                // [row][segment]: m
    int32_t* maxima;            // [row][piece], order keys
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
template <int CONTROL>
__device__ __forceinline__ double rotated(double x)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), CONTROL, 0xf, 0xf, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), CONTROL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}
__device__ __forceinline__ double wave_sum(double x)
{
    x += rotated<0x128>(x);
    x += rotated<0x124>(x);
    x += rotated<0x122>(x);
    x += rotated<0x121>(x);
    uint64_t bits = __builtin_bit_cast(uint64_t, x);
    auto low = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(bits), static_cast<uint32_t>(bits), false, false);
    auto high = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(bits >> 32), static_cast<uint32_t>(bits >> 32), false, false);
    x = __builtin_bit_cast(double, static_cast<uint64_t>(high[0]) << 32 | low[0]) + __builtin_bit_cast(double, static_cast<uint64_t>(high[1]) << 32 | low[1]);
    bits = __builtin_bit_cast(uint64_t, x);
    low = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(bits), static_cast<uint32_t>(bits), false, false);
    high = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(bits >> 32), static_cast<uint32_t>(bits >> 32), false, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high[0]) << 32 | low[0]) + __builtin_bit_cast(double, static_cast<uint64_t>(high[1]) << 32 | low[1]);
}

// Integers in the order of the numbers (-0 and +0 the same; a NaN has been replaced by +infinity before).
__device__ __forceinline__ int32_t order_key(float x)
{
    const int32_t bits = static_cast<int32_t>(__float_as_uint(x + 0.0f));
    return bits ^ ((bits >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float order_value(int32_t key) { return __uint_as_float(static_cast<uint32_t>(key ^ ((key >> 31) & 0x7fffffff))); }
// One number for the order of candidates: greater logits first, equal ones by index.
__device__ __forceinline__ uint64_t candidate_key(float x, int32_t id)
{
    return static_cast<uint64_t>(static_cast<uint32_t>(order_key(x)) ^ 0x80000000u) << 32 | (0xffffffffu - static_cast<uint32_t>(id));
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
            const float above = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(value), 0x138, 0xf, 0xf, false));     // lane - 1
            const int32_t above_id = __builtin_amdgcn_update_dpp(0, id, 0x138, 0xf, 0xf, false);
            value = lane < place ? value : lane == place ? v : above;
            id = lane < place ? id : lane == place ? i : above_id;
            last = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(value), top - 1));
        }
    }
};

// The sums of some logits relative to m, the largest of them (kLowest if there is none above it).  R is without one logit that is
// m, in all the lanes together, unless m is kLowest: what one lane leaves out is not in another's.
struct Sums {
    float m;
    double R, T;

    __device__ __forceinline__ void clear()
    {
        m = kLowest;
        R = T = 0.0;
    }
    // Takes in the logit that was left out.
    __device__ __forceinline__ void whole()
    {
        if (m > kLowest) R += 1.0;
    }
    __device__ __forceinline__ void rescale(float next)
    {
        if (next == m) return;
        if (m == kLowest) {                                     // nothing yet, or nothing that counts beside a greater logit
            R *= 0.0;
            T = R;
            m = next;
            return;
        }
        const double by = static_cast<double>(m) - static_cast<double>(next), e = exp(by);
        // (by * R first: by may be -infinity only where e is 0 and R is 0 or not a number)
        T = e == 0.0 ? 0.0 * R : e * (T + by * R);
        R *= e;
        m = next;
    }
};

// What the W waves of a workgroup exchange.
template <int W>
struct Joined {
    float m[W];
    double R[W], T[W];
    alignas(16) int32_t maxima[kMaxPieces];                     // order keys
    float hand[W][kHandLogits];
    uint64_t candidates[W * NNHIP_LOG_PROBS_MAX_TOP], best[NNHIP_LOG_PROBS_MAX_TOP];
    int32_t before[kMaxPieces], chosen[NNHIP_LOG_PROBS_MAX_TOP], counts[kMaxPieces / 64], found[W];
    float threshold, bounds[W][2];
    int listed;
};

// The sums of the waves, in their order; every thread gets them.
template <int W>
__device__ void join_sums(Joined<W>& j, Sums& sums)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) j.m[wave] = sums.m;
    __syncthreads();
    float m = j.m[0];
    for (int w = 1; w < W; ++w) m = fmaxf(m, j.m[w]);
    if (lane == 0 && sums.m != m) sums.whole();
    const int equal = __popcll(__ballot(lane < W && j.m[lane & (W - 1)] == m));         // waves that go on without their maximum: one of them may
    sums.rescale(m);                                            // (one exponential a wave, not W in every one)
    const double R = wave_sum(sums.R), T = wave_sum(sums.T);
    if (lane == 0) {
        j.R[wave] = R;
        j.T[wave] = T;
    }
    __syncthreads();
    sums.R = sums.T = 0.0;
    for (int w = 0; w < W; ++w) {
        sums.R += j.R[w];
        sums.T += j.T[w];
    }
    if (m > kLowest) sums.R += static_cast<double>(equal - 1);
    asm volatile("" : "+v"(sums.R), "+v"(sums.T));              // added up here: 32 registers of summands would wait for the end
}

// Of the 64 keys of group `other` in LDS, those that go before key v of lane `lane` of group `group`: greater ones, and equal
// ones of lower places.
__device__ __forceinline__ int places_before(const int4* keys, int other, int32_t v, int group, int lane)
{
    int before = 0;
    if (other != group) {
        const int32_t least = other < group ? v - 1 : v;
#pragma unroll 2
        for (int q = 0; q < 16; ++q) {
            const int4 x = keys[other * 16 + q];
            before += (x.x > least ? 1 : 0) + (x.y > least ? 1 : 0) + (x.z > least ? 1 : 0) + (x.w > least ? 1 : 0);
        }
        return before;
    }
#pragma unroll 2
    for (int q = 0; q < 16; ++q) {
        const int4 x = keys[other * 16 + q];
        before += (x.x > (4 * q < lane ? v - 1 : v) ? 1 : 0) + (x.y > (4 * q + 1 < lane ? v - 1 : v) ? 1 : 0) +
                  (x.z > (4 * q + 2 < lane ? v - 1 : v) ? 1 : 0) + (x.w > (4 * q + 3 < lane ? v - 1 : v) ? 1 : 0);
    }
    return before;
}

// At most the n-th largest of the 64 lanes' values and less than 2^-5 below it, for two n: the upper 14 bits of its order key,
// one by one.
__device__ __forceinline__ float2 nth_largest(float value, int n0, int n1)
{
    const uint32_t key = static_cast<uint32_t>(order_key(value)) ^ 0x80000000u;
    uint32_t found0 = 0, found1 = 0;
#pragma unroll
    for (int bit = 31; bit > 17; --bit) {
        const uint32_t with0 = found0 | 1u << bit, with1 = found1 | 1u << bit;
        found0 = __popcll(__ballot(key >= with0)) >= n0 ? with0 : found0;
        found1 = __popcll(__ballot(key >= with1)) >= n1 ? with1 : found1;
    }
    // (keys below that of the least finite number are no numbers)
    return float2{found0 < 0x00800000u ? -INFINITY : order_value(static_cast<int32_t>(found0 ^ 0x80000000u)),
                  found1 < 0x00800000u ? -INFINITY : order_value(static_cast<int32_t>(found1 ^ 0x80000000u))};
}

// The `top` best logits of a row whose pieces' maxima are in LDS -> j.best, in their order.
template <int W>
__device__ void find_best(Joined<W>& j, const LogProbArgs& a, const float* x)
{
    constexpr int kRounds = (kMaxPieces + W * 64 - 1) / (W * 64), kList = W * NNHIP_LOG_PROBS_MAX_TOP;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), top = a.d.top, pieces = a.pieces;
    const int wanted = top < pieces ? top : pieces;
    const bool choose = top < pieces;
    if (tid == 0) j.listed = 0;
    if (choose) {
        // The place of every piece among all: groups of 64 pieces against groups of 64, spread over the waves.
        const int groups = (pieces + 63) / 64;
        for (int p = tid; p < groups * 64; p += W * 64) {
            j.before[p] = 0;
            if (p >= pieces) j.maxima[p] = INT32_MIN;
        }
        __syncthreads();
        for (int task = wave; task < groups * groups; task += W) {
            const int group = task % groups, p = group * 64 + lane;
            atomicAdd(&j.before[p], places_before(reinterpret_cast<const int4*>(j.maxima), task / groups, j.maxima[p], group, lane));
        }
        __syncthreads();
        bool chosen[kRounds];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int p = (r * W + wave) * 64 + lane;
            chosen[r] = p < pieces && j.before[p] < top;
            if (chosen[r] && j.before[p] == top - 1) j.threshold = order_value(j.maxima[p]);
            const uint64_t mask = __ballot(chosen[r]);
            if (lane == 0 && r * W + wave < kMaxPieces / 64) j.counts[r * W + wave] = __popcll(mask);
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {                         // in rising order
            const uint64_t mask = __ballot(chosen[r]);
            if (mask == 0) continue;
            int at = __popcll(mask & ((1ull << lane) - 1));
            for (int w = 0; w < r * W + wave; ++w) at += j.counts[w];
            if (chosen[r]) j.chosen[at] = (r * W + wave) * 64 + lane;
        }
        __syncthreads();
    } else {
        __syncthreads();
    }
    float threshold = choose ? j.threshold : -INFINITY;
    float now[kHand], next[kHand];
    int64_t at = 0, end = 0, next_at = 0, next_end = 0;
    auto fetch = [&](float (&to)[kHand], int64_t from, int64_t until) {
        const float* y = x + from;
        const int left = static_cast<int>(until - from < kHandLogits ? until - from : kHandLogits);
#pragma unroll
        for (int u = 0; u < kHand; ++u) to[u] = u * 64 + lane < left ? y[u * 64 + lane] : 0.0f;
    };
    auto open = [&](int c, int64_t& from, int64_t& until) {
        from = static_cast<int64_t>(choose ? __builtin_amdgcn_readfirstlane(j.chosen[c]) : c) * a.piece;
        until = from + a.piece < a.d.vocabulary ? from + a.piece : a.d.vocabulary;
    };
    int c = wave;
    if (c < wanted) {
        open(c, at, end);
        fetch(now, at, end);
    }
    if (!choose) {
        // No more pieces than alternatives: a threshold from the lanes of the waves' first pieces.  Where each of n waves has top / n
        // lanes no smaller, the row has `top` logits no smaller; so it has where one wave has `top` of them.
        const int waves = wanted < W ? wanted : W, each = (top + waves - 1) / waves;
        if (wave < waves) {
            const int left = static_cast<int>(end - at < kHandLogits ? end - at : kHandLogits);
            float most = -INFINITY;
#pragma unroll
            for (int u = 0; u < kHand; ++u) most = u * 64 + lane < left ? (now[u] != now[u] ? INFINITY : fmaxf(most, now[u])) : most;
            const float2 bounds = nth_largest(most, each, top);
            if (lane == 0) {
                j.bounds[wave][0] = bounds.x;
                j.bounds[wave][1] = bounds.y;
            }
        }
        __syncthreads();
        float least = INFINITY;
        for (int w = 0; w < waves; ++w) {
            least = fminf(least, j.bounds[w][0]);
            threshold = fmaxf(threshold, j.bounds[w][1]);
        }
        threshold = fmaxf(threshold, least);
    }
    // Piece by piece, 1024 logits at a time, the next ones on their way.  What is not below the threshold goes into one list (241
    // rows of 13507, 32 alternatives: 22 us; sorted lists in every wave from the start 32); where that is too short (many equal
    // logits, rows in rising order), once more with a sorted list of `top` in every wave: as many as the list has room for.
    int all = 0;
    for (bool listed = true;; listed = false) {
        Best best;
        best.clear();
        while (c < wanted) {
            const int left = static_cast<int>(end - at < kHandLogits ? end - at : kHandLogits);
            next_at = at + kHandLogits;
            next_end = end;
            if (next_at >= end) {
                c += W;
                if (c < wanted) open(c, next_at, next_end);
            }
            if (c < wanted) fetch(next, next_at, next_end);
            uint64_t mask[kHand];
            int count = 0;
#pragma unroll
            for (int u = 0; u < kHand; ++u) {
                mask[u] = __ballot(u * 64 + lane < left && !(now[u] < threshold));
                count += __popcll(mask[u]);
            }
            if (listed && count != 0) {
                int place = 0;
                if (lane == 0) place = atomicAdd(&j.listed, count);         // (the order in the list has no influence)
                place = __builtin_amdgcn_readfirstlane(place);
#pragma unroll
                for (int u = 0; u < kHand; ++u) {
                    if (mask[u] == 0) continue;
                    const int mine = place + __popcll(mask[u] & ((1ull << lane) - 1));
                    if ((mask[u] >> lane & 1) != 0 && mine < kList)
                        j.candidates[mine] = candidate_key(now[u] != now[u] ? INFINITY : now[u], static_cast<int32_t>(at) + u * 64 + lane);
                    place += __popcll(mask[u]);
                }
            } else if (!listed) {
                // (through LDS, so that the code that takes one in exists once)
#pragma unroll
                for (int u = 0; u < kHand; ++u) j.hand[wave][u * 64 + lane] = now[u];
                for (int u = 0; u < kHand; ++u) {
                    const float v = j.hand[wave][u * 64 + lane];
                    best.offer(__ballot(u * 64 + lane < left && !(v < threshold) && !(v <= best.last)), v, static_cast<int32_t>(at) + u * 64 + lane, top);
                }
            }
            at = next_at;
            end = next_end;
#pragma unroll
            for (int u = 0; u < kHand; ++u) now[u] = next[u];
        }
        if (!listed) {          // the waves' entries side by side
            const uint64_t held = __ballot(best.id >= 0);
            if (lane == 0) j.found[wave] = __popcll(held);
            __syncthreads();
            int place = 0;
            all = 0;
            for (int w = 0; w < W; ++w) {
                place += w < wave ? j.found[w] : 0;
                all += j.found[w];
            }
            if (best.id >= 0) j.candidates[place + lane] = candidate_key(best.value, best.id);          // (entries fill the lanes from 0 on)
            break;
        }
        __syncthreads();
        all = j.listed;
        if (all <= kList) break;
        c = wave;
        if (c < wanted) {
            open(c, at, end);
            fetch(now, at, end);
        }
    }
    __syncthreads();
    // every entry counts those that go before it, four threads a quarter each
    for (int e = tid >> 2; e < (all + 63 & ~63); e += W * 16) {
        const uint64_t key = e < all ? j.candidates[e] : 0;
        int before = 0;
#pragma unroll 4
        for (int k = tid & 3; k < all; k += 4) before += j.candidates[k] > key ? 1 : 0;
        before += __shfl_xor(before, 1);
        before += __shfl_xor(before, 2);
        if ((tid & 3) == 0 && e < all && before < top) j.best[before] = key;
    }
    __syncthreads();
}

// Results of one row from the sums over all of it and the best in LDS.
template <int W>
__device__ void write_row(const nnhip_log_probs_desc& d, int row, const Joined<W>& j, const Sums& sums)
{
    const int tid = threadIdx.x;
    // (a NaN among the logits makes R NaN; where all are -infinity nothing is left out and R is 0)
    const bool defined = (sums.m > kLowest || sums.R > 0.0) && sums.R < INFINITY && sums.m < INFINITY;
    const double rest = sums.m > kLowest ? sums.R : sums.R - 1.0, log_sum = log1p(rest), m = static_cast<double>(sums.m);
    if (tid < d.top) {
        const size_t at = static_cast<size_t>(row) * d.top + tid;
        const uint64_t key = j.best[tid];
        const float x = order_value(static_cast<int32_t>(static_cast<uint32_t>(key >> 32) ^ 0x80000000u));
        d.top_ids[at] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
        if (d.top_log_probs) d.top_log_probs[at] = defined ? static_cast<float>((static_cast<double>(x) - m) - log_sum) : no_number();
    }
    if (tid == 128 && d.entropy) d.entropy[row] = defined ? static_cast<float>(log_sum - sums.T / (1.0 + rest)) : no_number();
    if (tid == 64 && d.log_probs) {
        const int32_t t = d.targets[row];
        float lp = no_number();
        if (defined && t >= 0 && t < d.vocabulary)
            lp = static_cast<float>((static_cast<double>(d.logits[static_cast<int64_t>(row) * d.row_stride + t]) - m) - log_sum);
        d.log_probs[row] = lp;
    }
}

template <int W>
__global__ __launch_bounds__(W * 64) void log_probs_kernel(const LogProbArgs a)
{
    __shared__ Joined<W> joined;
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
    // wave w takes the pieces w, w + W, ... of the segment
    const int64_t step = static_cast<int64_t>(W - 1) * a.piece;
    int64_t at = first + static_cast<int64_t>(wave) * a.piece, piece_end = at + a.piece;
    float largest = -INFINITY;
    if (at < end) fetch(now, at);
    while (at < end) {
        const int64_t following = at + kHandLogits == piece_end ? piece_end + step : at + kHandLogits;
        if (following < end) fetch(next, following);
        float most = now[0];
#pragma unroll
        for (int u = 1; u < kHand; ++u) most = fmaxf(most, now[u]);
        const float of_lane = most;
        most = wave_max(most);
        // e^d = 2^a e^(d - a ln 2) with a = fl(d log2 e): the second factor makes up for the rounding of a and of log2 e, which
        // would cost 1.45 |d| 2^-24 of the term (512 rows of 262144: 100.8 us and 98.8 without).  The 16 products of T meet in FP32, which
        // costs T at most 2^-20 of itself and 6e-8 in those rows (in 64 bits 101.4 us, 32 such rows 20.8 instead of 20.3).
        float t = 0.0f;
        auto term = [&](float v) {
            const float all = v - sums.m, d = all < -200.0f ? -200.0f : all;            // (e is 0 long before; a NaN stays one)
            const float power = d * kLog2e, term_of_power = __builtin_amdgcn_exp2f(power);
            const float e = fmaf(term_of_power, fmaf(-power, kLn2Low, fmaf(-power, kLn2, d)), term_of_power);
            t = fmaf(d, e, t);
            return e;
        };
        if (most > sums.m) {
            // a new maximum: the lane that holds it leaves out its largest term
            const int owner = __builtin_ctzll(__ballot(of_lane == most));
            if (lane == 0) sums.whole();
            sums.rescale(most);
            float largest_term = 0.0f;
#pragma unroll
            for (int u = 0; u < kHand; ++u) {
                const float e = term(now[u]);
                sums.R += static_cast<double>(fminf(largest_term, e));
                largest_term = fmaxf(largest_term, e);
            }
            sums.R += static_cast<double>((t - t) + (lane == owner ? 0.0f : largest_term));         // (t - t: 0 or no number)
        } else {
#pragma unroll
            for (int u = 0; u < kHand; ++u) sums.R += static_cast<double>(term(now[u]));
        }
        sums.T += static_cast<double>(t);
        if (a.d.top > 0) {
            largest = __any(t != t) ? INFINITY : fmaxf(largest, most);          // a NaN counts as +infinity
            if (following != at + kHandLogits || following >= end) {
                const int piece = static_cast<int>((piece_end - 1) / a.piece);
                if (lane == 0) {
                    if (a.segments == 1)
                        joined.maxima[piece] = order_key(largest);
                    else
                        a.maxima[static_cast<size_t>(row) * a.pieces + piece] = order_key(largest);
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
        a.sums[2 * static_cast<size_t>(blockIdx.x)] = sums.R;
        a.sums[2 * static_cast<size_t>(blockIdx.x) + 1] = sums.T;
    }
}

// One row: the sums of its segments, and its best logits.
template <int W>
__global__ __launch_bounds__(W * 64) void log_probs_join_kernel(const LogProbArgs a)
{
    constexpr int kThreads = W * 64;
    __shared__ Joined<W> joined;
    const int tid = threadIdx.x;
    const size_t from = static_cast<size_t>(blockIdx.x) * a.segments;
    if (a.d.top > 0)
        for (int p = tid; p < a.pieces; p += kThreads) joined.maxima[p] = a.maxima[static_cast<size_t>(blockIdx.x) * a.pieces + p];
    Sums sums;
    sums.clear();
    // (at most 128 segments: a quarter of the pieces there can be)
    if (tid < a.segments) sums = Sums{a.tops[from + tid], a.sums[2 * (from + tid)], a.sums[2 * (from + tid) + 1]};
    const float m = wave_max(sums.m);
    const int equal = __popcll(__ballot(sums.m == m));          // lanes that go on without their maximum: one of them may
    if (sums.m != m) sums.whole();
    sums.rescale(m);
    if ((tid & 63) == 0 && m > kLowest) sums.R += static_cast<double>(equal - 1);
    join_sums(joined, sums);
    if (a.d.top > 0) find_best(joined, a, a.d.logits + static_cast<int64_t>(blockIdx.x) * a.d.row_stride);
    write_row(a.d, blockIdx.x, joined, sums);
}

}  // namespace

LogProbPlan plan_token_log_probs(const nnhip_log_probs_desc& d, int compute_units)
{
    LogProbPlan p{};
    const int64_t V = d.vocabulary, hands = (V + kHandLogits - 1) / kHandLogits;
    const int64_t piece = (hands + kMaxPieces - 1) / kMaxPieces, pieces = (hands + piece - 1) / piece;
    p.piece = static_cast<int>(piece * kHandLogits);
    p.pieces = static_cast<int>(pieces);
    // A few short rows are one workgroup's work each, sixteen waves in one launch: up to 16 pieces always (250 rows of 16000, five
    // alternatives: 11.9 us instead of 15.7), up to 32 where there is more to rank than to read (250 of 18000, five 12.6 and
    // 16.2, twenty 19.0 and 22.5; a row of 32000 and one alternative would take 11.7 instead of 10.5, of 48000 14.5 instead of 10.4).
    // 2100 rows of 5000 would take 81 us instead of 25.
    const bool one = pieces <= (d.top > kWaves ? 32 : 16) && d.rows <= compute_units;
    p.waves = one && pieces > kWaves ? 16 : kWaves;
    // Otherwise eight workgroups of four waves a compute unit (of which five fit at a time), none with less than a piece for each wave.
    int64_t segments = one ? 1 : 8 * static_cast<int64_t>(compute_units) / d.rows;
    if (segments > (pieces + kWaves - 1) / kWaves) segments = (pieces + kWaves - 1) / kWaves;
    if (segments < 1) segments = 1;
    const int64_t each = (pieces + segments - 1) / segments;
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
        a.maxima = reinterpret_cast<int32_t*>(a.tops + parts);
    }
    if (p.waves == 16)
        hipLaunchKernelGGL(log_probs_kernel<16>, dim3(static_cast<unsigned>(parts)), dim3(1024), 0, lane->stream, a);
    else
        hipLaunchKernelGGL(log_probs_kernel<kWaves>, dim3(static_cast<unsigned>(parts)), dim3(kThreads), 0, lane->stream, a);
    if (p.segments == 1) return hipGetLastError();
    // Pieces are ranked and looked at again wave by wave: sixteen waves a row where the device has room for them and there is
    // work for them (32 rows of 262144: twenty alternatives 12.7 us with four waves, 10.8 with sixteen, one 8.8 and 8.4; a row of
    // 32000 and one alternative: 6.1 and 7.5).
    if (d.rows <= lane->compute_units && d.top > 0 && (p.pieces > 64 || d.top > kWaves))
        hipLaunchKernelGGL(log_probs_join_kernel<16>, dim3(d.rows), dim3(1024), 0, lane->stream, a);
    else
        hipLaunchKernelGGL(log_probs_join_kernel<kWaves>, dim3(d.rows), dim3(kThreads), 0, lane->stream, a);
    return hipGetLastError();
}

}  // namespace nnhip
