// The 8-bit key/value cache: storing tokens (rotary positions, block quantisation), advancing the lengths, reading back.
//
// Definition (nnhip.h): scale = fl32(max |x| / 127) over a block, code = rint(x / scale) of the exact quotient.  With
// n = rint(fl(x * fl(1 / scale))), off by one at most, the remainder x - n scale is exact in one fused multiply-add (it is a
// multiple of half an ulp of scale and at most about half of scale), so comparing twice its magnitude with scale decides
// between n and its neighbour, ties to even.  The codes are then a function of the stored values alone.
//
// The rotation is done in 64 bits and rounded once, for positions where an FP32 angle has no correct digit of the turn left:
// angle = position * inv_freq, reduced by multiples of pi / 2 in two parts, and the Taylor polynomials of degree 17 and 16 on
// [-pi/4, pi/4], whose remainders are below 2^-58; in a block every sixteenth token's, the ones between by products.
//
// Bound by moving the bytes: a workgroup takes one block of one head, keys or values, through an FP32 tile in LDS from which
// the codes are read out in the order of the cache (16 bytes a store).  A single token rarely changes its block's scale: then
// it alone is quantised and its bytes alone are written; otherwise the block is quantised again from the FP32 values kept.
#include "kv_cache_layout.h"
#include "nnhip_internal.h"

namespace nnhip {

namespace {

constexpr int kThreads = 256;

typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kAlone = 8;       // new tokens that may go in without the rest of their block
constexpr int kMoreStored = 256;        // in a mark: the block has had more tokens than the buffer holds, and its scale is theirs too

struct StoreArgs {
    KvLayout cache;
    int tokens;
    const int32_t* counts;
    nnhip_rows k, v, q, q_out;
    const float* inv_freq;
    int rotary_width;
    uint32_t rotary_style;
    int heads;
    uint32_t pair_magic;    // 2^32 / (rotary_width / 2), rounded up: e / pairs is the high word of e * pair_magic for e < 2^16
    int slots;              // workgroups of each pair and kind, a block each
    unsigned kv_groups;     // workgroups of the cache part; the query part follows
    bool wide_k, wide_v;    // rows lie on 16-byte boundaries and head_width is a multiple of 4
    bool wide_q;            // so do those of q and q_out, and the rotary halves are multiples of 4
};

// cos and sin of position * inv_freq.
__device__ __forceinline__ double2 turn_of(int position, float inv_freq)
{
    const double angle = static_cast<double>(position) * static_cast<double>(inv_freq);
    double s, c;
    if (!(fabs(angle) < 0x1p40)) {
        sincos(angle, &s, &c);
        return double2{c, s};
    }
    const double n = rint(angle * 0.63661977236758134308);
    double r = fma(n, -1.57079632679489655800, angle);          // pi / 2 rounded to 64 bits,
    r = fma(n, -6.12323399573676603587e-17, r);                 // and what is left of it
    const double z = r * r;
    s = 2.8114572543455207632e-15;                              // 1 / 17!
    s = fma(s, z, -7.6471637318198164759e-13);
    s = fma(s, z, 1.6059043836821614599e-10);
    s = fma(s, z, -2.5052108385441718775e-08);
    s = fma(s, z, 2.7557319223985890653e-06);
    s = fma(s, z, -1.9841269841269841270e-04);
    s = fma(s, z, 8.3333333333333333333e-03);
    s = fma(s, z, -1.6666666666666666667e-01);
    s = fma(s * z, r, r);
    c = 4.7794773323873852974e-14;                              // 1 / 16!
    c = fma(c, z, -1.1470745597729724714e-11);
    c = fma(c, z, 2.0876756987868098979e-09);
    c = fma(c, z, -2.7557319223985890653e-07);
    c = fma(c, z, 2.4801587301587301587e-05);
    c = fma(c, z, -1.3888888888888888889e-03);
    c = fma(c, z, 4.1666666666666666667e-02);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const double quarter = n - 4.0 * floor(n * 0.25);           // 0 .. 3
    const double a = quarter == 1.0 || quarter == 3.0 ? s : c, b = quarter == 1.0 || quarter == 3.0 ? c : s;
    return double2{quarter == 1.0 || quarter == 2.0 ? -a : a, quarter >= 2.0 ? -b : b};
}

// The code of x, biased: see the top of this file.  inverse = 1 / scale; a scale so small that its inverse is no number takes
// the quotient in 64 bits; scale 0 or NaN gives code 0.
struct Quantizer {
    float scale, inverse;
    bool zero, tiny;

    __device__ __forceinline__ explicit Quantizer(float s) : scale(s), inverse(1.0f / s), zero(!(s > 0.0f)), tiny(s < 0x1p-120f) {}
    __device__ __forceinline__ uint32_t operator()(float x) const
    {
        if (zero) return 128u;
        float n;
        if (tiny) {
            n = static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(scale)));
        } else {
            n = rintf(x * inverse);
            const float rest = fmaf(-n, scale, x), twice = 2.0f * fabsf(rest);
            const bool odd = (static_cast<int>(n) & 1) != 0;
            if (twice > scale || (twice == scale && odd)) n += copysignf(1.0f, rest);
        }
        return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(n, -127.0f), 127.0f)) + 128);
    }
    // Sixteen at a time: where every remainder is less than half of scale, the first guesses are the codes (five instructions
    // a value); otherwise, at a tie or a guess off by one, one by one.
    __device__ __forceinline__ uint4 operator()(const float (&x)[16]) const
    {
        uint32_t word[4] = {0, 0, 0, 0};
        float worst = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float n = rintf(x[i] * inverse);
            worst = fmaxf(worst, fabsf(fmaf(-n, scale, x[i])));
            word[i / 4] = __builtin_amdgcn_cvt_pk_u8_f32(n + 128.0f, i % 4, word[i / 4]);
        }
        if (zero || tiny || !(2.0f * worst < scale)) {
            word[0] = word[1] = word[2] = word[3] = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) word[i / 4] |= (*this)(x[i]) << (8 * (i % 4));
        }
        return uint4{word[0], word[1], word[2], word[3]};
    }
};

// Components a, b of rotary pair j.
__device__ inline void rotary_pair(const StoreArgs& a, int j, int* first, int* second)
{
    const bool halves = a.rotary_style == NNHIP_ROTARY_HALVES;
    *first = halves ? j : 2 * j;
    *second = halves ? j + a.rotary_width / 2 : 2 * j + 1;
}

__device__ inline void turn(float* a, float* b, double c, double s)
{
    const double x = *a, y = *b;
    *a = static_cast<float>(x * c - y * s);
    *b = static_cast<float>(y * c + x * s);
}

// max |x| over the tile's tokens [from, to) as bits (the order of the numbers, infinity and NaN above all), for every thread.
template <int DP>
__device__ __forceinline__ uint32_t largest_of(const float* tile, int from, int to, uint32_t* exchange)
{
    constexpr int quads = DP / 4, pitch = DP + 4;
    const int tid = threadIdx.x;
    uint32_t top = 0;
#pragma unroll 4
    for (int e = tid; e < (to - from) * quads; e += kThreads) {
        const int t = from + e / quads;
        const float4 x = *reinterpret_cast<const float4*>(&tile[t * pitch + e % quads * 4]);
        top = max(top, max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu),
                           max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu)));
    }
    for (int y = 32; y > 0; y >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), y)));
    __syncthreads();
    if ((tid & 63) == 0) exchange[tid >> 6] = top;
    __syncthreads();
    return max(max(exchange[0], exchange[1]), max(exchange[2], exchange[3]));
}

__device__ __forceinline__ float scale_of(uint32_t largest)
{
    return largest < 0x7f800000u ? __uint_as_float(largest) / 127.0f : __uint_as_float(0x7fc00000u);
}

// New tokens [from, to) of a block into the tile, keys turned by their positions.
template <int DP>
__device__ __forceinline__ void load_new(const StoreArgs& a, float* tile, int which, int b, int head, int block, int start, int from, int to)
{
    constexpr int padded = DP, quads = DP / 4, pitch = DP + 4;
    const int tid = threadIdx.x, width = a.cache.head_width;
    const nnhip_rows& rows = which ? a.v : a.k;
    const float* data = rows.data + b * rows.sequence_stride + (static_cast<int64_t>(block) * kKvBlock - start) * rows.token_stride + head * width;
    if (which ? a.wide_v : a.wide_k) {
#pragma unroll 8
        for (int e = tid; e < (to - from) * quads; e += kThreads) {
            const int t = from + e / quads, d = e % quads * 4;
            float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (d < width) x = *reinterpret_cast<const float4*>(data + t * rows.token_stride + d);
            *reinterpret_cast<float4*>(&tile[t * pitch + d]) = x;
        }
    } else {
#pragma unroll 8
        for (int e = tid; e < (to - from) * padded; e += kThreads) {
            const int t = from + e / padded, d = e % padded;
            tile[t * pitch + d] = d < width ? data[t * rows.token_stride + d] : 0.0f;
        }
    }
    if (which || !a.inv_freq) return;
    __syncthreads();
    // A thread turns one pair of the new tokens among sixteen: every sixteenth position has its turn from its angle, each further
    // one is a step more (a product of complex numbers in 64 bits, 2^-49 off after sixteen).  The steps are taken from that position
    // whichever token is the call's first, so that a token's turn is the same number however the tokens arrive.
    constexpr int kRun = 16;
    const int pairs = a.rotary_width / 2, before = from / kRun, runs = (to + kRun - 1) / kRun - before;
    for (int e = tid; e < runs * pairs; e += kThreads) {
        const int run = pairs == 1 ? e : static_cast<int>(__umulhi(static_cast<uint32_t>(e), a.pair_magic)), j = e - run * pairs;
        int t = (before + run) * kRun, d0, d1;
        const int end = min(t + kRun, to);
        const float f = a.inv_freq[j];
        double2 r = turn_of(block * kKvBlock + t, f);
        const double2 step = t + 1 < end ? turn_of(1, f) : double2{1.0, 0.0};
        rotary_pair(a, j, &d0, &d1);
        auto next = [&] { r = double2{fma(r.x, step.x, -r.y * step.y), fma(r.x, step.y, r.y * step.x)}; };
#pragma unroll 1
        for (; t < from; ++t) next();
        for (; t < end; ++t) {
            turn(&tile[t * pitch + d0], &tile[t * pitch + d1], r.x, r.y);
            next();
        }
    }
}

// One block of one head, keys or values: tokens [from, to) of the block are new, those before `from` are there already.
// `first` is the block that the call begins in.
template <int DP>
__device__ __forceinline__ void store_block(const StoreArgs& a, float* tile, uint32_t* exchange, int which, int b, int head, int pair, int block, int first,
                                            int start, int from, int to, bool last)
{
    constexpr int padded = DP, pitch = DP + 4, quads = DP / 4;
    const KvLayout& kv = a.cache;
    const int tid = threadIdx.x;
    int32_t* marks = kv.marks(which, pair);
    uint8_t* codes = kv.codes(which, pair, block);
    float* scale_at = kv.scales(pair, block) + which;
    // The buffer of this block's FP32 values: the one that holds it, else one that does not hold the block the call begins in
    // (another workgroup may be reading that one; it looks for `first` alone, which this workgroup never writes over).
    const int2 mark0 = reinterpret_cast<const int2*>(marks)[0], mark1 = reinterpret_cast<const int2*>(marks)[1];
    const int buffer = mark0.x == block ? 0 : mark1.x == block ? 1 : mark0.x == first ? 1 : 0;
    const int held_block = buffer ? mark1.x : mark0.x, held_mark = buffer ? mark1.y : mark0.y, held_tokens = held_mark & (kMoreStored - 1);
    float* open = kv.open_values(which, pair, buffer);
    const float old_scale = from > 0 ? *scale_at : 0.0f;
    load_new<DP>(a, tile, which, b, head, block, start, from, to);
    __syncthreads();
    bool done = false;
    if (from > 0 && to - from <= kAlone && held_block == block && held_mark == from) {
        // no new value above the block's largest: the other tokens stay as they are
        const float scale = scale_of(largest_of<DP>(tile, from, to, exchange));
        if (scale <= old_scale) {
            const Quantizer quantize(old_scale);
            for (int e = tid; e < (to - from) * padded; e += kThreads) {
                const int t = from + e / padded, d = e % padded;
                codes[which ? kv_value_offset(t, d) : kv_key_offset(padded, t, d)] = static_cast<uint8_t>(quantize(tile[t * pitch + d]));
            }
            done = true;
        }
    }
    if (!done) {
        // the older tokens: from the FP32 values kept of them, or from their codes where another block has taken the place
        const bool held = held_block == block && held_tokens >= from;
        if (held) {
            // (the whole buffer, four loads on their way at a time; what lies behind `from` is not used)
            const floatx4* kept = reinterpret_cast<const floatx4*>(open) + tid;
#pragma unroll 1
            for (int e = tid; e < from * quads; e += 4 * kThreads, kept += 4 * kThreads) {
                floatx4 x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u] = e + u * kThreads < kKvBlock * quads ? kept[u * kThreads] : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int at = e + u * kThreads;
                    if (at < from * quads) *reinterpret_cast<floatx4*>(&tile[at / quads * pitch + at % quads * 4]) = x[u];
                }
            }
        } else {
            for (int e = tid; e < from * quads; e += kThreads) {
                const int t = e / quads, d = e % quads * 4;
                float y[4];
                for (int u = 0; u < 4; ++u) y[u] = old_scale * static_cast<float>(codes[which ? kv_value_offset(t, d + u) : kv_key_offset(padded, t, d + u)] - 128);
                const float4 x = {y[0], y[1], y[2], y[3]};
                if (last) *reinterpret_cast<float4*>(&open[t * padded + d]) = x;
                *reinterpret_cast<float4*>(&tile[t * pitch + d]) = x;
            }
        }
        for (int e = tid; e < (kKvBlock - to) * quads; e += kThreads)
            *reinterpret_cast<float4*>(&tile[(to + e / quads) * pitch + e % quads * 4]) = float4{0.0f, 0.0f, 0.0f, 0.0f};
        __syncthreads();
        const float scale = scale_of(largest_of<DP>(tile, 0, to, exchange));
        if (tid == 0) *scale_at = scale;
        const Quantizer quantize(scale);
        // sixteen codes a thread, in the order of the cache
        for (int unit = tid; unit < padded * kKvBlock / 16; unit += kThreads) {
            float x[16];
            if (which) {
                const int lane = unit & 63, d = (unit >> 6) * 16 + (lane & 15), g = lane >> 4;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = tile[(16 * (i / 4) + 4 * g + i % 4) * pitch + d];
            } else {
                int t[2], d[2];         // two runs of eight components
                if (unit < padded / 64 * 256) {
                    t[0] = t[1] = (unit >> 6 & 3) * 16 + (unit & 15);
                    d[0] = (unit >> 8) * 64 + (unit >> 4 & 3) * 16;
                    d[1] = d[0] + 8;
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int place = 2 * (unit - padded / 64 * 256) + u;
                        t[u] = (place >> 6) * 16 + (place & 15);
                        d[u] = padded / 64 * 64 + (place >> 4 & 3) * 8;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const floatx4 y = *reinterpret_cast<const floatx4*>(&tile[t[j / 2] * pitch + d[j / 2] + j % 2 * 4]);
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[4 * j + u] = y[u];
                }
            }
            reinterpret_cast<uint4*>(codes)[unit] = quantize(x);
        }
    }
    if (last) {
        for (int e = tid; e < (to - from) * quads; e += kThreads) {
            const int t = from + e / quads, d = e % quads * 4;
            *reinterpret_cast<float4*>(&open[t * padded + d]) = *reinterpret_cast<const float4*>(&tile[t * pitch + d]);
        }
        if (tid == 0) {
            marks[2 * buffer] = block;
            marks[2 * buffer + 1] = to;
            // the other buffer's block, where this call has written over all of it
            const int other = buffer ? mark0.x : mark1.x;
            if (other == block || (other > first && other < block)) marks[2 * (1 - buffer) + 1] = kMoreStored;
        }
    } else if (block == first && held_block == block && tid == 0) {
        marks[2 * buffer + 1] = kMoreStored | min(held_tokens, from);       // the tokens behind them are this call's
    }
}

template <int DP>
__global__ __launch_bounds__(kThreads) void kv_store_kernel(const StoreArgs a)
{
    __shared__ float4 shared[kKvBlock * (DP + 4) / 4];
    __shared__ uint32_t exchange[4];
    float* tile = reinterpret_cast<float*>(shared);
    const KvLayout& kv = a.cache;
    bool left_out;
    if (blockIdx.x < a.kv_groups) {
        unsigned at = blockIdx.x;
        const int slot = static_cast<int>(at % static_cast<unsigned>(a.slots));
        at /= static_cast<unsigned>(a.slots);
        const int which = static_cast<int>(at & 1u), pair = static_cast<int>(at >> 1);
        const int b = pair / kv.kv_heads, head = pair - b * kv.kv_heads;
        const int start = kv.lengths[b];
        const int n = kv_tokens_of(start, kv.capacity, a.tokens, a.counts, b, &left_out);
        if (left_out || n == 0) return;
        const int end = start + n, first = start / kKvBlock, final = (end - 1) / kKvBlock;
        const int block = first + slot;
        if (block > final) return;
        const int from = slot == 0 ? start - first * kKvBlock : 0, to = block == final ? end - final * kKvBlock : kKvBlock;
        store_block<DP>(a, tile, exchange, which, b, head, pair, block, first, start, from, to, block == final);
        return;
    }
    // the query heads of one token: its turns once, in LDS
    double2* turns = reinterpret_cast<double2*>(shared);
    const unsigned at = blockIdx.x - a.kv_groups;
    const int b = static_cast<int>(at / static_cast<unsigned>(a.tokens)), i = static_cast<int>(at % static_cast<unsigned>(a.tokens));
    const int start = kv.lengths[b];
    const int n = kv_tokens_of(start, kv.capacity, a.tokens, a.counts, b, &left_out);
    if (left_out || i >= n) return;
    const float* q = a.q.data + b * a.q.sequence_stride + i * a.q.token_stride;
    float* out = a.q_out.data + b * a.q_out.sequence_stride + i * a.q_out.token_stride;
    const int pairs = a.rotary_width / 2, width = kv.head_width, rest = width - a.rotary_width;
    for (int j = threadIdx.x; j < pairs; j += kThreads) turns[j] = turn_of(start + i, a.inv_freq[j]);
    __syncthreads();
    if (a.wide_q) {
        const int quads = pairs / 4;
#pragma unroll 4
        for (int e = threadIdx.x; e < a.heads * quads; e += kThreads) {
            const int h = e / quads, j = e % quads * 4;
            float4 x = *reinterpret_cast<const float4*>(q + h * width + j), y = *reinterpret_cast<const float4*>(q + h * width + pairs + j);
            turn(&x.x, &y.x, turns[j].x, turns[j].y);
            turn(&x.y, &y.y, turns[j + 1].x, turns[j + 1].y);
            turn(&x.z, &y.z, turns[j + 2].x, turns[j + 2].y);
            turn(&x.w, &y.w, turns[j + 3].x, turns[j + 3].y);
            *reinterpret_cast<float4*>(out + h * width + j) = x;
            *reinterpret_cast<float4*>(out + h * width + pairs + j) = y;
        }
    } else {
        for (int e = threadIdx.x; e < a.heads * pairs; e += kThreads) {
            const int h = e / pairs, j = e - h * pairs;
            int d0, d1;
            rotary_pair(a, j, &d0, &d1);
            float x = q[h * width + d0], y = q[h * width + d1];
            turn(&x, &y, turns[j].x, turns[j].y);
            out[h * width + d0] = x;
            out[h * width + d1] = y;
        }
    }
    for (int e = threadIdx.x; e < a.heads * rest; e += kThreads) {
        const int d = e / rest * width + a.rotary_width + e % rest;
        out[d] = q[d];
    }
}

__global__ void kv_advance_kernel(int32_t* lengths, const int32_t* counts, int sequences, int tokens, int capacity)
{
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b >= sequences) return;
    bool left_out;
    const int n = kv_tokens_of(lengths[b], capacity, tokens, counts, b, &left_out);
    if (!left_out) lengths[b] += n;
}

// The values of one block of one head, keys or values: codes through LDS, [token][component], so that a wave writes whole rows
// (32 sequences, 64 tokens of 16 heads of 128: 11.8 us; keys straight from the order of the codes, 16 bytes in each of 16
// rows a store: 25 us; values straight from it, four components of sixteen tokens a thread: 12.5 us).
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const KvLayout kv, const int32_t* first, int tokens, int slots, nnhip_rows k, nnhip_rows v,
                                                           bool wide_k, bool wide_v)
{
    __shared__ uint4 shared[kKvBlock * (kKvMaxWidth + 16) / 16];
    uint8_t* tile = reinterpret_cast<uint8_t*>(shared);
    const int tid = threadIdx.x, padded = kv.padded, pitch = padded + 16;
    unsigned at = blockIdx.x;
    const int slot = static_cast<int>(at % static_cast<unsigned>(slots));
    at /= static_cast<unsigned>(slots);
    const int which = static_cast<int>(at & 1u), pair = static_cast<int>(at >> 1);
    const int b = pair / kv.kv_heads, head = pair - b * kv.kv_heads;
    const nnhip_rows& rows = which ? v : k;
    if (!rows.data) return;
    const int64_t begin = first ? first[b] : 0, end = begin + tokens;
    const int64_t block = (begin >> 6) + slot, t0 = block * kKvBlock;
    static_assert(kKvBlock == 64, "block of a token by a shift");
    if (t0 >= end) return;
    const int from = static_cast<int>(begin > t0 ? begin - t0 : 0), to = static_cast<int>(end - t0 < kKvBlock ? end - t0 : kKvBlock);
    const bool inside = block >= 0 && block < kv.blocks;
    float scale = 0.0f;
    if (inside) {
        scale = kv.scales(pair, static_cast<int>(block))[which];
        const uint4* codes = reinterpret_cast<const uint4*>(kv.codes(which, pair, static_cast<int>(block)));
        for (int unit = tid; unit < padded * kKvBlock / 16; unit += kThreads) {
            const uint4 x = codes[unit];
            if (which) {
                const int lane = unit & 63, d = (unit >> 6) * 16 + (lane & 15), g = lane >> 4;
                const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) tile[(16 * j + 4 * g + i) * pitch + d] = static_cast<uint8_t>(word[j] >> (8 * i));
            } else if (unit < padded / 64 * 256) {
                *reinterpret_cast<uint4*>(&tile[((unit >> 6 & 3) * 16 + (unit & 15)) * pitch + (unit >> 8) * 64 + (unit >> 4 & 3) * 16]) = x;
            } else {
                const int place = 2 * (unit - padded / 64 * 256);           // two lanes of eight components
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    *reinterpret_cast<uint2*>(&tile[((place >> 6) * 16 + (place & 15) + u) * pitch + padded / 64 * 64 + (place >> 4 & 3) * 8]) =
                        u ? uint2{x.z, x.w} : uint2{x.x, x.y};
            }
        }
    }
    __syncthreads();
    float* out = rows.data + b * rows.sequence_stride + (t0 - begin) * rows.token_stride + head * kv.head_width;
    // tokens between the capacity and the end of its last block do not exist either
    const int64_t there = inside ? kv.capacity - t0 : 0;
    if (which ? wide_v : wide_k) {
        const int quads = kv.head_width / 4;
#pragma unroll 8
        for (int e = tid; e < (to - from) * quads; e += kThreads) {
            const int t = from + e / quads, d = e % quads * 4;
            float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
            if (t < there) {
                const uint32_t word = *reinterpret_cast<const uint32_t*>(&tile[t * pitch + d]);
                x.x = scale * static_cast<float>(static_cast<int>(word & 255u) - 128);
                x.y = scale * static_cast<float>(static_cast<int>(word >> 8 & 255u) - 128);
                x.z = scale * static_cast<float>(static_cast<int>(word >> 16 & 255u) - 128);
                x.w = scale * static_cast<float>(static_cast<int>(word >> 24) - 128);
            }
            *reinterpret_cast<float4*>(out + t * rows.token_stride + d) = x;
        }
    } else {
        for (int e = tid; e < (to - from) * kv.head_width; e += kThreads) {
            const int t = from + e / kv.head_width, d = e % kv.head_width;
            out[t * rows.token_stride + d] = t < there ? scale * static_cast<float>(tile[t * pitch + d] - 128) : 0.0f;
        }
    }
}

}  // namespace

static bool on_16_bytes(const nnhip_rows& r)
{
    return (reinterpret_cast<uintptr_t>(r.data) & 15u) == 0 && r.token_stride % 4 == 0 && r.sequence_stride % 4 == 0;
}

hipError_t launch_kv_store(Lane* lane, const KvLayout& cache, const nnhip_kv_store_desc& d)
{
    StoreArgs a{cache, d.tokens, d.counts, d.k, d.v, d.q, d.q_out, d.inv_freq, d.rotary_width, d.rotary_style, d.heads, 0, 0, 0, false, false, false};
    if (d.rotary_width > 0) {
        const uint64_t pairs = static_cast<uint64_t>(d.rotary_width) / 2;
        a.pair_magic = static_cast<uint32_t>(((1ull << 32) + pairs - 1) / pairs);       // (not used for one pair)
    }
    a.slots = static_cast<int>((static_cast<int64_t>(d.tokens) + kKvBlock - 2) / kKvBlock + 1);      // the blocks n tokens can touch
    a.kv_groups = static_cast<unsigned>(a.slots) * 2u * static_cast<unsigned>(cache.sequences * cache.kv_heads);
    a.wide_k = cache.head_width % 4 == 0 && on_16_bytes(d.k);
    a.wide_v = cache.head_width % 4 == 0 && on_16_bytes(d.v);
    a.wide_q = cache.head_width % 4 == 0 && d.rotary_width % 8 == 0 && d.rotary_style == NNHIP_ROTARY_HALVES && on_16_bytes(d.q) && on_16_bytes(d.q_out);
    const dim3 grid(a.kv_groups + (d.q.data ? static_cast<unsigned>(cache.sequences) * static_cast<unsigned>(d.tokens) : 0u)), block(kThreads);
    switch (cache.padded) {
    case 32: hipLaunchKernelGGL(kv_store_kernel<32>, grid, block, 0, lane->stream, a); break;
    case 64: hipLaunchKernelGGL(kv_store_kernel<64>, grid, block, 0, lane->stream, a); break;
    case 96: hipLaunchKernelGGL(kv_store_kernel<96>, grid, block, 0, lane->stream, a); break;
    case 128: hipLaunchKernelGGL(kv_store_kernel<128>, grid, block, 0, lane->stream, a); break;
    case 192: hipLaunchKernelGGL(kv_store_kernel<192>, grid, block, 0, lane->stream, a); break;
    default: hipLaunchKernelGGL(kv_store_kernel<256>, grid, block, 0, lane->stream, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_kv_advance(Lane* lane, const KvLayout& cache, int tokens, const int32_t* counts)
{
    hipLaunchKernelGGL(kv_advance_kernel, dim3((cache.sequences + 255) / 256), dim3(256), 0, lane->stream, cache.lengths, counts,
                       cache.sequences, tokens, cache.capacity);
    return hipGetLastError();
}

hipError_t launch_kv_read(Lane* lane, const KvLayout& cache, const int32_t* first, int tokens, const nnhip_rows& k, const nnhip_rows& v)
{
    const int slots = static_cast<int>((static_cast<int64_t>(tokens) + kKvBlock - 2) / kKvBlock + 1);
    const bool fours = cache.head_width % 4 == 0;
    hipLaunchKernelGGL(kv_read_kernel, dim3(static_cast<unsigned>(slots) * 2u * static_cast<unsigned>(cache.sequences * cache.kv_heads)), dim3(kThreads), 0,
                       lane->stream, cache, first, tokens, slots, k, v, fours && on_16_bytes(k), fours && on_16_bytes(v));
    return hipGetLastError();
}

}  // namespace nnhip
