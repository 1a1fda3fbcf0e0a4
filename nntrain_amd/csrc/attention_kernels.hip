// Attention over the 8-bit key/value cache (nnhip_cached_attention): causal, grouped query heads, optional sliding window
// with the first tokens kept visible.
//
// One pass over the keys with the running maximum m and sum l of the softmax, a block of 64 keys at a time:
//     s_t = scale q . K_t,   m' = max(m, max_t s_t),   l' = l e^(m - m') + sum_t e^(s_t - m'),   o' = o e^(m - m') + sum_t e^(s_t - m') V_t
// and o / l at the end.  All in powers of two: the factor log2(e) goes into the scale.
//
// The query rows that share a key/value head (tokens x heads of the group) are the columns of the matrix products, so a block
// of keys is read once for a tile of them: S^T = K Q^T, O^T = V^T P^T, on v_mfma_f32_16x16x32_f16 with 16 rows a column tile.
// Transposed this way a lane's accumulators hold 16 probabilities of one row, in the order in which the cache keeps the
// values' tokens (kv_cache_layout.h): they are the operand of the second product as they stand, and a row's maximum needs two
// exchanges between lanes.
//
// Precision: the codes are integers up to 127, exact in half precision.  Queries are scaled by a power of two to at most
// 2^14 and taken as hi + lo half-precision parts, so are the probabilities times (value scale / a running power of two above
// the value scales of the blocks a row has seen) times 2^14: 22 bits below the largest, nothing lost before 2^-38 of it.  Two products for each operand pair
// instead of one is what FP32 results cost; one rounding to half precision would leave 2^-12.
//
// All sums are FP32 and grow a block at a time: l and o of a row over n keys that one workgroup takes are off by up to (n / 16) 2^-23
// of themselves, seen where one key stands far above many (131000 keys, one 17 above the others, unsplit: 1.1e-4).
//
// Two kernels.  attend_few_kernel, up to 32 rows a key/value head (decode): bound by reading the cache, once for 32 rows of heads up
// to 128 and once for 16 of larger ones, so every wave walks over blocks of its own, codes go from memory to registers to half precision without LDS, and the keys are split over many
// workgroups.  attend_many_kernel (prompts): bound by the matrix cores and the softmax beside them, so the waves of a tile share
// each block, converted once into LDS; its keys are split where there are few tiles.  The parts are added up by
// attend_join_few_kernel (up to eight) or attend_join_kernel.
#include <algorithm>

#include "kv_cache_layout.h"
#include "nnhip_internal.h"

namespace nnhip {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kPartScale = 16384.0f;          // 2^14: probabilities enter the product as p * 2^14
constexpr float kSlack = 1.9f;                  // the running maximum may lag by this much: 2^1.9 * 2^14 is a half-precision number
constexpr float kLeastValueScale = 0x1p-100f;   // keeps kPartScale / (running value scale) finite

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

struct AttendArgs {
    KvLayout cache;
    int tokens;
    const int32_t* counts;
    nnhip_rows q, out;
    int heads, group;       // group: query heads of a key/value head
    int window, sinks;
    float scale;            // times log2(e)
    bool wide;              // rows of q and out lie on 16-byte boundaries and head_width is a multiple of 4
    int row_tiles;          // workgroups over the rows of a pair
    int splits;             // workgroups over the keys
    int least;              // fewest blocks a split takes
    int together;           // so many blocks are not split
    float* partial;         // [pair][row][split][padded] sums, then [pair][row][split][2] m, l
    float* stats;
};

// The blocks that the rows of one workgroup see: the first `sink_blocks`, then those from `window_block` on.
struct Span {
    int start, n;           // tokens before the call, tokens of the call
    int rows;               // n * group
    int first, last;        // positions of the first and the last row of the tile
    int sink_blocks, window_block, blocks;
    int begin, end;         // of this split
    bool left_out;
    __device__ int block(int index) const { return index < sink_blocks ? index : index - sink_blocks + window_block; }
};

__device__ __forceinline__ int blocks_of_split(const AttendArgs& a, int blocks)
{
    return blocks <= a.together ? a.together : max(a.least, (blocks + a.splits - 1) / a.splits);
}

// Rows [row0, row0 + rows_of_tile) of a pair, split `split`.  The number of splits in use follows from the blocks there are.
__device__ __forceinline__ Span span_of(const AttendArgs& a, int b, int row0, int rows_of_tile, int split)
{
    Span s;
    s.start = a.cache.lengths[b];
    s.n = kv_tokens_of(s.start, a.cache.capacity, a.tokens, a.counts, b, &s.left_out);
    s.rows = s.n * a.group;
    const int last_row = min(row0 + rows_of_tile, s.rows) - 1;
    s.first = s.start + row0 / a.group;
    s.last = s.start + max(last_row, 0) / a.group;
    const int low = a.window > 0 && s.first >= a.window ? s.first - a.window + 1 : 0;
    s.window_block = low / kKvBlock;
    s.sink_blocks = min((min(a.sinks, kKvBlock * s.window_block) + kKvBlock - 1) / kKvBlock, s.window_block);
    s.blocks = s.sink_blocks + s.last / kKvBlock + 1 - s.window_block;
    const int each = blocks_of_split(a, s.blocks);
    s.begin = static_cast<int>(min(static_cast<int64_t>(split) * each, static_cast<int64_t>(s.blocks)));
    s.end = min(s.begin + each, s.blocks);
    return s;
}

__device__ __forceinline__ int splits_used(const AttendArgs& a, const Span& s)
{
    const int each = blocks_of_split(a, s.blocks);
    return (s.blocks + each - 1) / each;
}

// Maximum / sum over the four lanes that share a column (lane % 16).
__device__ __forceinline__ float column_max(float x)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float column_sum(float x)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Eight biased codes to half precision: 0x6400 | byte is 1024 + byte, minus 1152 is the code.
__device__ __forceinline__ half8 halves(uint32_t a, uint32_t b)
{
    const half2v bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    half2v r[4];
    r[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + bias;
    r[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + bias;
    r[2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + bias;
    r[3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + bias;
    return __builtin_shufflevector(__builtin_shufflevector(r[0], r[1], 0, 1, 2, 3), __builtin_shufflevector(r[2], r[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// x[0..7] as hi + lo: the nearest half-precision numbers, then those nearest to what is left.  `minus` is -1 in a register: the
// difference is then one instruction that reads the half-precision number as it stands.
__device__ __forceinline__ void split_parts(const float* x, float minus, half8* hi, half8* lo)
{
    half2v h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const floatx2 v = {x[2 * i], x[2 * i + 1]};
        h[i] = __builtin_convertvector(v, half2v);
        const floatx2 r = {fmaf(static_cast<float>(h[i].x), minus, v.x), fmaf(static_cast<float>(h[i].y), minus, v.y)};
        l[i] = __builtin_convertvector(r, half2v);
    }
    *hi = __builtin_shufflevector(__builtin_shufflevector(h[0], h[1], 0, 1, 2, 3), __builtin_shufflevector(h[2], h[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
    *lo = __builtin_shufflevector(__builtin_shufflevector(l[0], l[1], 0, 1, 2, 3), __builtin_shufflevector(l[2], l[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ float minus_one()
{
    float x = -1.0f;
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ floatx4 mma(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Component at which the eight a lane holds of k-step `step` begin: the order of the key codes.
template <int DP>
__device__ __forceinline__ int component_of(int step, int g)
{
    return (step / 2 + 1) * 64 <= DP ? step / 2 * 64 + g * 16 + step % 2 * 8 : step / 2 * 64 + g * 8;
}

// One column tile: 16 query rows and their running softmax.  A lane belongs to row lane % 16.
template <int DP>
struct Rows16 {
    half8 hi[DP / 32], lo[DP / 32];
    floatx4 o[DP / 16];
    float c;                // what a product of the scaled query and codes is multiplied by, apart from the key scale
    float m, l;             // running maximum (in powers of two; it may lag by kSlack), this lane's part of the sum
    float running;          // the least power of two above the value scales of the blocks the row has seen: the sums o are scaled by it
    int position, low;      // of the row; first key of its window

    __device__ __forceinline__ void load(const AttendArgs& a, const Span& s, int b, int kv_head, int row)
    {
        const int lane = threadIdx.x & 63, g = lane >> 4, width = a.cache.head_width;
        const bool valid = row < s.rows;
        const int i = valid ? row / a.group : 0, h = valid ? row - i * a.group : 0;
        const float* q = a.q.data + b * a.q.sequence_stride + i * a.q.token_stride + (kv_head * a.group + h) * width;
        float x[DP / 32][8];
        uint32_t most = 0;
#pragma unroll
        for (int step = 0; step < DP / 32; ++step) {
            const int d = component_of<DP>(step, g);
            if (a.wide) {
#pragma unroll
                for (int u = 0; u < 8; u += 4) {
                    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (valid && d + u < width) v = *reinterpret_cast<const floatx4*>(q + d + u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[step][u + e] = v[e];
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) x[step][u] = valid && d + u < width ? q[d + u] : 0.0f;
            }
        }
#pragma unroll
        for (int step = 0; step < DP / 32; ++step)
#pragma unroll
            for (int u = 0; u < 8; ++u) most = max(most, __float_as_uint(x[step][u]) & 0x7fffffffu);
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
        most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
        // 2^shift brings the largest component into [2^13, 2^14)
        const int shift = min(13 - (static_cast<int>(most >> 23) - 127), 120);
        const float up = __uint_as_float(static_cast<uint32_t>(shift + 127) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
        for (int step = 0; step < DP / 32; ++step) {
#pragma unroll
            for (int u = 0; u < 8; ++u) x[step][u] *= up;
            split_parts(x[step], -1.0f, &hi[step], &lo[step]);
        }
        c = most < 0x7f800000u ? a.scale * down : 0.0f;
        m = -INFINITY;
        running = kLeastValueScale;
        l = most < 0x7f800000u ? 0.0f : __uint_as_float(0x7fc00000u);           // (a query that is not finite: its row is NaN)
        position = valid ? s.start + i : -1;        // a row that is not there sees nothing
        low = a.window > 0 && position >= a.window ? position - a.window + 1 : 0;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // Whether the row sees any token of the block that starts at t0, whether it sees token t.
    __device__ __forceinline__ bool sees_block(int t0, int sinks) const { return t0 <= position && (t0 + kKvBlock > low || t0 < sinks); }
    __device__ __forceinline__ bool sees(int t, int sinks) const { return t <= position && (t >= low || t < sinks); }
};

// The softmax step of one block for CT column tiles: scores (products of scaled queries and codes) -> parts of the
// probabilities for the second product; m, l, o and `running` of the rows move on.  A block that a row does not see leaves the
// row's `running` alone: values of any size there cost it no digits.
template <int DP, int CT>
__device__ __forceinline__ void softmax_step(Rows16<DP> (&r)[CT], floatx4 (&s)[CT][4], float2 scales, int t0, bool full, int sinks, float minus,
                                             half8 (&p_hi)[CT][2], half8 (&p_lo)[CT][2])
{
    const int g = (threadIdx.x & 63) >> 4;
    if (scales.x != scales.x || scales.y != scales.y) {         // rows that see some of the block become NaN, the others ignore it
#pragma unroll
        for (int t = 0; t < CT; ++t)
            if (r[t].sees_block(t0, sinks)) r[t].l = __uint_as_float(0x7fc00000u);
        scales = float2{0.0f, 0.0f};
    }
    if (!full) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!r[t].sees(t0 + 16 * j + 4 * g + i, sinks)) s[t][j][i] = -INFINITY;
    }
    const float above = __uint_as_float((__float_as_uint(scales.y) & 0x7f800000u) + 0x00800000u);
    float scale[CT], next[CT], base[CT], keep[CT], factor[CT];
    bool moved = false;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const bool sees = full || r[t].sees_block(t0, sinks);
        const float higher = sees ? fmaxf(r[t].running, above) : r[t].running;
        const float inverse = __uint_as_float(0x7f000000u - __float_as_uint(higher));         // (of a power of two, exact)
        keep[t] = r[t].running * inverse;
        factor[t] = sees ? scales.y * (kPartScale * inverse) : 0.0f;
        r[t].running = higher;
        // never 0: a hidden score stays at -infinity
        scale[t] = fmaxf(r[t].c * scales.x, 1e-37f);
        float top = s[t][0][0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][j][i]);
        next[t] = column_max(top) * scale[t];
        moved |= __any(next[t] > r[t].m + kSlack || keep[t] != 1.0f) != 0;
    }
    if (moved) {
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            next[t] = fmaxf(r[t].m, next[t]);
            const float shrink = __builtin_amdgcn_exp2f(r[t].m - (next[t] == -INFINITY ? 0.0f : next[t])), all = shrink * keep[t];
            r[t].l *= shrink;
            r[t].m = next[t];
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) r[t].o[d] *= all;
        }
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) base[t] = r[t].m == -INFINITY ? 0.0f : r[t].m;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[t][2 * h + u / 4][u % 4], scale[t], -base[t]));
                w[u] = p * factor[t];
                sum += p;
            }
            split_parts(w, minus, &p_hi[t][h], &p_lo[t][h]);
        }
        r[t].l += sum;
    }
}

// A block whose every token every row of [first, last] sees.
__device__ __forceinline__ bool sees_all(const AttendArgs& a, int t0, int first, int last)
{
    return t0 + kKvBlock - 1 <= first && (a.window == 0 || t0 > last - a.window || t0 + kKvBlock - 1 < a.sinks);
}

__device__ __forceinline__ void put(float* to, floatx4 v, int d, int width, bool wide)
{
    if (wide) {
        if (d < width) *reinterpret_cast<floatx4*>(to + d) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < width) to[d + e] = v[e];
    }
}

// Rows of sequences that are left out become NaN.
__device__ void refuse_rows(const AttendArgs& a, const Span& s, int b, int kv_head, int row0, int rows)
{
    for (int e = threadIdx.x; e < rows * a.cache.head_width; e += blockDim.x) {
        const int row = row0 + e / a.cache.head_width, d = e % a.cache.head_width;
        if (row >= s.rows) break;
        const int i = row / a.group, h = kv_head * a.group + row % a.group;
        a.out.data[b * a.out.sequence_stride + i * a.out.token_stride + h * a.cache.head_width + d] = __uint_as_float(0x7fc00000u);
    }
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Codes that one workgroup alone reads (two, where 17 to 32 rows of heads above 128 are two tiles): streamed past the caches.
__device__ __forceinline__ uint4 stream(const uint8_t* p)
{
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return uint4{x[0], x[1], x[2], x[3]};
}

template <int DP>
struct Codes {
    static constexpr int kWhole = DP / 64, kRest = DP % 64 ? 1 : 0;
    uint4 k[kWhole ? kWhole * 4 : 1], v[DP / 16];
    uint2 rest[4];
    float2 scales;

    __device__ __forceinline__ void load_keys(const KvLayout& kv, int pair, int block, int lane)
    {
        const uint8_t* at = kv.codes(0, pair, block);
#pragma unroll
        for (int u = 0; u < kWhole * 4; ++u) k[u] = stream(at + u * 1024 + lane * 16);
        if (kRest) {
#pragma unroll
            for (int j = 0; j < 4; ++j) rest[j] = *reinterpret_cast<const uint2*>(at + kWhole * 4096 + j * 512 + lane * 8);
        }
        scales = *reinterpret_cast<const float2*>(kv.scales(pair, block));
    }
    __device__ __forceinline__ void load_values(const KvLayout& kv, int pair, int block, int lane)
    {
        const uint8_t* at = kv.codes(1, pair, block);
#pragma unroll
        for (int u = 0; u < DP / 16; ++u) v[u] = stream(at + u * 1024 + lane * 16);
    }
    __device__ __forceinline__ half8 key(int step, int j) const
    {
        if (step / 2 < kWhole) {
            const uint4& x = k[step / 2 * 4 + j];
            return step % 2 ? halves(x.z, x.w) : halves(x.x, x.y);
        }
        return halves(rest[j].x, rest[j].y);
    }
    __device__ __forceinline__ half8 value(int t, int h) const { return h ? halves(v[t].z, v[t].w) : halves(v[t].x, v[t].y); }
};

template <int DP, int CT>
__global__ __launch_bounds__(kThreads, DP * CT <= 128 ? 2 : 1) void attend_few_kernel(const AttendArgs a)
{
    constexpr int kRows = CT * 16, kPitch = DP + 4;
    __shared__ float sums[2][kRows * kPitch];
    __shared__ float stats[kWaves][kRows][2];
    const KvLayout& kv = a.cache;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    unsigned at = blockIdx.x;
    const int split = static_cast<int>(at % static_cast<unsigned>(a.splits));
    at /= static_cast<unsigned>(a.splits);
    const int row0 = static_cast<int>(at % static_cast<unsigned>(a.row_tiles)) * kRows, pair = static_cast<int>(at / static_cast<unsigned>(a.row_tiles));
    const int b = pair / kv.kv_heads, kv_head = pair - b * kv.kv_heads;
    const Span s = span_of(a, b, row0, kRows, split);
    if (row0 >= s.rows) return;
    if (s.left_out) {
        if (split == 0) refuse_rows(a, s, b, kv_head, row0, kRows);
        return;
    }
    if (s.begin >= s.end) return;

    Rows16<DP> r[CT];
    Codes<DP> codes;
    int index = s.begin + wave;
    if (index < s.end) {
        codes.load_keys(kv, pair, s.block(index), lane);
        codes.load_values(kv, pair, s.block(index), lane);
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) r[t].load(a, s, b, kv_head, row0 + t * 16 + (lane & 15));
    const float minus = minus_one();
    while (index < s.end) {
        const int t0 = s.block(index) * kKvBlock;
        floatx4 scores[CT][4];
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) scores[t][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int step = 0; step < DP / 32; ++step) {
            half8 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = codes.key(step, j);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) scores[t][j] = mma(k[j], r[t].hi[step], scores[t][j]);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) scores[t][j] = mma(k[j], r[t].lo[step], scores[t][j]);
        }
        const float2 scales = codes.scales;
        index += kWaves;
        const int next = s.block(min(index, s.end - 1));
        if (index < s.end) codes.load_keys(kv, pair, next, lane);
        half8 p_hi[CT][2], p_lo[CT][2];
        softmax_step<DP, CT>(r, scores, scales, t0, sees_all(a, t0, s.first, s.last), a.sinks, minus, p_hi, p_lo);
#pragma unroll
        for (int d = 0; d < DP / 16; d += 2) {
            half8 v[2][2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) v[u][h] = codes.value(d + u, h);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int t = 0; t < CT; ++t) r[t].o[d + u] = mma(v[u][h], part ? p_lo[t][h] : p_hi[t][h], r[t].o[d + u]);
        }
        if (index < s.end) codes.load_values(kv, pair, next, lane);
    }
    // the four waves' sums, in a fixed order: 0 + 2 and 1 + 3 through LDS, then the two
    const int column = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        r[t].l = column_sum(r[t].l);
        if (g == 0) {
            stats[wave][t * 16 + column][0] = r[t].m;
            stats[wave][t * 16 + column][1] = r[t].l;
        }
    }
    __syncthreads();
    for (int round = 0; round < 2; ++round) {
        if (wave / 2 == round) {
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const int row = t * 16 + column;
                float m = stats[0][row][0];
                for (int w = 1; w < kWaves; ++w) m = fmaxf(m, stats[w][row][0]);
                const float factor = __builtin_amdgcn_exp2f(r[t].m - (m == -INFINITY ? 0.0f : m)) * (r[t].running * (1.0f / kPartScale));
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    floatx4* to = reinterpret_cast<floatx4*>(&sums[wave & 1][row * kPitch + d * 16 + g * 4]);
                    const floatx4 x = r[t].o[d] * factor;
                    *to = round ? *to + x : x;
                }
            }
        }
        __syncthreads();
    }
    const int used = splits_used(a, s);
    for (int e = threadIdx.x; e < kRows * (DP / 4); e += kThreads) {
        const int row = e / (DP / 4), d = e % (DP / 4) * 4;
        if (row0 + row >= s.rows) break;
        float m = stats[0][row][0], l = 0.0f;
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, stats[w][row][0]);
        const float base = m == -INFINITY ? 0.0f : m;
        for (int w = 0; w < kWaves; ++w) l += stats[w][row][1] * __builtin_amdgcn_exp2f(stats[w][row][0] - base);
        floatx4 x = *reinterpret_cast<const floatx4*>(&sums[0][row * kPitch + d]) + *reinterpret_cast<const floatx4*>(&sums[1][row * kPitch + d]);
        if (used == 1) {
            const int i = (row0 + row) / a.group, h = kv_head * a.group + (row0 + row) % a.group;
            x /= l;
            put(a.out.data + b * a.out.sequence_stride + i * a.out.token_stride + h * kv.head_width, x, d, kv.head_width, a.wide);
        } else {
            const size_t to = (static_cast<size_t>(pair) * a.tokens * a.group + row0 + row) * a.splits + split;
            *reinterpret_cast<floatx4*>(a.partial + to * DP + d) = x;
            if (d == 0) {
                a.stats[2 * to] = m;
                a.stats[2 * to + 1] = l;
            }
        }
    }
}

// CT * 16 rows a wave, W waves a team; G teams share the rows, take every G-th block and add up at the end.  Blocks are staged in
// LDS as half precision in operand order (every fragment 1 KB in lane order: no bank is asked twice), two buffers, one
// barrier a block; the next block's codes travel during the products.
template <int DP, int CT, int W, int G>
__global__ __launch_bounds__(G * W * 64, 2) void attend_many_kernel(const AttendArgs a)
{
    constexpr int kThreads = W * 64, kRows = CT * 16 * W, kUnits = DP * kKvBlock / 16, kPerThread = (kUnits + kThreads - 1) / kThreads;
    constexpr int kWhole = DP / 64, kFragments = DP * kKvBlock * 2 / 1024;       // KB of keys (or values) in half precision
    extern __shared__ uint4 staged_all[];                                        // [group][2][keys, values][fragment][64]
    const KvLayout& kv = a.cache;
    const int team = G == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kThreads), tid = threadIdx.x - team * kThreads;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    uint4* staged = staged_all + team * 2 * 2 * kFragments * 64;
    // the tiles with the longest spans first, the pairs side by side
    const int pairs = kv.sequences * kv.kv_heads;
    unsigned at = blockIdx.x;
    const int pair = static_cast<int>(at % static_cast<unsigned>(pairs));
    at /= static_cast<unsigned>(pairs);
    const int split = static_cast<int>(at % static_cast<unsigned>(a.splits)), row0 = (a.row_tiles - 1 - static_cast<int>(at / static_cast<unsigned>(a.splits))) * kRows;
    const int b = pair / kv.kv_heads, kv_head = pair - b * kv.kv_heads;
    const Span s = span_of(a, b, row0, kRows, split);
    if (row0 >= s.rows) return;
    if (s.left_out) {
        if (split == 0) refuse_rows(a, s, b, kv_head, row0, kRows);
        return;
    }
    if (s.begin >= s.end) return;

    uint4 keys[kPerThread], values[kPerThread];
    float2 scales = {0.0f, 0.0f}, scales_next;
    auto fetch = [&](int index) {
        const int block = s.block(index);
        const uint4* k = reinterpret_cast<const uint4*>(kv.codes(0, pair, block));
        const uint4* v = reinterpret_cast<const uint4*>(kv.codes(1, pair, block));
#pragma unroll
        for (int u = 0; u < kPerThread; ++u)
            if (kUnits % kThreads == 0 || tid + u * kThreads < kUnits) {
                keys[u] = k[tid + u * kThreads];
                values[u] = v[tid + u * kThreads];
            }
        scales_next = *reinterpret_cast<const float2*>(kv.scales(pair, block));
    };
    // 16 codes of a unit are two lanes' or two steps' fragments
    auto stage = [&](int buffer) {
        uint4* k = staged + buffer * 2 * kFragments * 64;
        uint4* v = k + kFragments * 64;
#pragma unroll
        for (int u = 0; u < kPerThread; ++u) {
            const int unit = tid + u * kThreads;
            if (kUnits % kThreads != 0 && unit >= kUnits) break;
            const uint4 x0 = __builtin_bit_cast(uint4, halves(keys[u].x, keys[u].y)), x1 = __builtin_bit_cast(uint4, halves(keys[u].z, keys[u].w));
            if (unit < kWhole * 256) {                              // [chunk][j][lane]: steps 2 chunk, 2 chunk + 1
                const int chunk = unit >> 8, j = unit >> 6 & 3, l = unit & 63;
                k[((2 * chunk) * 4 + j) * 64 + l] = x0;
                k[((2 * chunk + 1) * 4 + j) * 64 + l] = x1;
            } else {                                                // [j][lane pair]: the last step
                const int rest = unit - kWhole * 256;
                k[(2 * kWhole * 4) * 64 + 2 * rest] = x0;
                k[(2 * kWhole * 4) * 64 + 2 * rest + 1] = x1;
            }
            v[(unit >> 6) * 128 + (unit & 63)] = __builtin_bit_cast(uint4, halves(values[u].x, values[u].y));
            v[(unit >> 6) * 128 + 64 + (unit & 63)] = __builtin_bit_cast(uint4, halves(values[u].z, values[u].w));
        }
        scales = scales_next;
    };

    if (s.begin + team < s.end) fetch(s.begin + team);
    Rows16<DP> r[CT];
    const int row_of_wave = row0 + wave * CT * 16;
#pragma unroll
    for (int t = 0; t < CT; ++t) r[t].load(a, s, b, kv_head, row_of_wave + t * 16 + (lane & 15));
    // positions of this wave's rows, for what it may skip
    const int first = s.start + min(row_of_wave, s.rows - 1) / a.group, last = s.start + (min(row_of_wave + CT * 16, s.rows) - 1) / a.group;
    const int low = a.window > 0 && first >= a.window ? first - a.window + 1 : 0;
    const bool any_row = row_of_wave < s.rows;
    const float minus = minus_one();
    if (s.begin + team < s.end) stage(0);
    __syncthreads();
    for (int at_block = s.begin, buffer = 0; at_block < s.end; at_block += G, buffer ^= 1) {
        const int index = at_block + team, t0 = s.block(index) * kKvBlock;
        const float2 now = scales;
        if (index + G < s.end) fetch(index + G);
        if (index < s.end && any_row && t0 <= last && (t0 + kKvBlock > low || t0 < a.sinks)) {
            const uint4* k = staged + buffer * 2 * kFragments * 64 + lane;
            const uint4* v = k + kFragments * 64;
            floatx4 scores[CT][4];
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) scores[t][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int step = 0; step < DP / 32; ++step) {
                half8 x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = __builtin_bit_cast(half8, k[(step * 4 + j) * 64]);
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) scores[t][j] = mma(x[j], r[t].hi[step], scores[t][j]);
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) scores[t][j] = mma(x[j], r[t].lo[step], scores[t][j]);
            }
            half8 p_hi[CT][2], p_lo[CT][2];
            softmax_step<DP, CT>(r, scores, now, t0, sees_all(a, t0, first, last), a.sinks, minus, p_hi, p_lo);
#pragma unroll
            for (int d = 0; d < DP / 16; d += 2) {
                half8 x[2][2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) x[u][h] = __builtin_bit_cast(half8, v[((d + u) * 2 + h) * 64]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int t = 0; t < CT; ++t) r[t].o[d + u] = mma(x[u][h], part ? p_lo[t][h] : p_hi[t][h], r[t].o[d + u]);
            }
        }
        if (index + G < s.end) stage(buffer ^ 1);
        __syncthreads();
    }
    const int used = splits_used(a, s), g = lane >> 4;
    float part[CT];                 // what the sums are scaled by
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        r[t].l = column_sum(r[t].l);
        part[t] = r[t].running * (1.0f / kPartScale);
    }
    if constexpr (G == 2) {
        constexpr int kPitch = DP + 4;
        float* sums = reinterpret_cast<float*>(staged_all);
        float* stats = sums + kRows * kPitch;
        const int row_in = wave * CT * 16 + (lane & 15);
        if (team == 1) {
#pragma unroll
            for (int t = 0; t < CT; ++t) {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) *reinterpret_cast<floatx4*>(&sums[(row_in + t * 16) * kPitch + d * 16 + g * 4]) = r[t].o[d] * part[t];
                if (g == 0) {
                    stats[2 * (row_in + t * 16)] = r[t].m;
                    stats[2 * (row_in + t * 16) + 1] = r[t].l;
                }
            }
        }
        __syncthreads();
        if (team == 1) return;
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const float m1 = stats[2 * (row_in + t * 16)], l1 = stats[2 * (row_in + t * 16) + 1], m = fmaxf(r[t].m, m1), base = m == -INFINITY ? 0.0f : m;
            const float mine = __builtin_amdgcn_exp2f(r[t].m - base), other = __builtin_amdgcn_exp2f(m1 - base);
            r[t].l = r[t].l * mine + l1 * other;
            r[t].m = m;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
                r[t].o[d] = r[t].o[d] * (part[t] * mine) + *reinterpret_cast<const floatx4*>(&sums[(row_in + t * 16) * kPitch + d * 16 + g * 4]) * other;
            part[t] = 1.0f;
        }
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const float l = r[t].l;
        const int row = row_of_wave + t * 16 + (lane & 15);
        if (row >= s.rows) continue;
        if (used == 1) {
            const int i = row / a.group, h = kv_head * a.group + row % a.group;
            float* to = a.out.data + b * a.out.sequence_stride + i * a.out.token_stride + h * kv.head_width;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) put(to, r[t].o[d] * part[t] / l, d * 16 + g * 4, kv.head_width, a.wide);
        } else {
            const size_t to = (static_cast<size_t>(pair) * a.tokens * a.group + row) * a.splits + split;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
                *reinterpret_cast<floatx4*>(a.partial + to * DP + d * 16 + g * 4) = r[t].o[d] * part[t];
            if (g == 0) {
                a.stats[2 * to] = r[t].m;
                a.stats[2 * to + 1] = l;
            }
        }
    }
}

// Adds up to kFewSplits splits of rows, four components a thread, every load on its way before the first is used: what bounds
// it is reading the partial results (8000 rows of 256 in four splits: 9.2 us; a workgroup a row takes 49).
constexpr int kFewSplits = 8;
__global__ __launch_bounds__(kThreads) void attend_join_few_kernel(const AttendArgs a, int rows_of_tile, int rows_of_group, unsigned all)
{
    const KvLayout& kv = a.cache;
    const int quads = kv.padded / 4, row_in = static_cast<int>(threadIdx.x) / quads, d = (static_cast<int>(threadIdx.x) - row_in * quads) * 4;
    const unsigned at = blockIdx.x * static_cast<unsigned>(rows_of_group) + row_in;
    if (row_in >= rows_of_group || at >= all) return;
    const unsigned rows = static_cast<unsigned>(a.tokens) * static_cast<unsigned>(a.group);
    const int row = static_cast<int>(at % rows), pair = static_cast<int>(at / rows), b = pair / kv.kv_heads, kv_head = pair - b * kv.kv_heads;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + static_cast<size_t>(at) * a.splits;
    const float* partial = a.partial + static_cast<size_t>(at) * a.splits * kv.padded + d;
    floatx4 x[kFewSplits];
    float2 st[kFewSplits];
#pragma unroll
    for (int k = 0; k < kFewSplits; ++k) {
        const int from = min(k, a.splits - 1);
        x[k] = *reinterpret_cast<const floatx4*>(partial + from * kv.padded);
        st[k] = stats[from];
    }
    const Span s = span_of(a, b, row / rows_of_tile * rows_of_tile, rows_of_tile, 0);
    if (row >= s.rows || s.left_out) return;
    const int used = splits_used(a, s);
    if (used == 1) return;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int k = 0; k < kFewSplits; ++k) m = fmaxf(m, k < used ? st[k].x : -INFINITY);
    const float base = m == -INFINITY ? 0.0f : m;
    floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kFewSplits; ++k)
        if (k < used) {
            const float weight = __builtin_amdgcn_exp2f(st[k].x - base);
            l += st[k].y * weight;
            sum += x[k] * weight;
        }
    const int i = row / a.group, h = kv_head * a.group + row % a.group;
    put(a.out.data + b * a.out.sequence_stride + i * a.out.token_stride + h * kv.head_width, sum / l, d, kv.head_width, a.wide);
}

// Adds up the splits of one row: sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k.  32 lanes hold 128 components, eight groups of
// them take every eighth split; the groups meet in LDS in their order.  What bounds it is a chain of memory latencies, so
// the first 64 splits are asked for before it is known how many are in use (those that are not have no weight).
__global__ __launch_bounds__(kThreads) void attend_join_kernel(const AttendArgs a, int rows_of_tile)
{
    constexpr int kAhead = 8;
    __shared__ floatx4 sums[kThreads];
    __shared__ float totals[8];
    const KvLayout& kv = a.cache;
    const int tid = threadIdx.x, group = tid >> 5;
    const unsigned rows = static_cast<unsigned>(a.tokens) * static_cast<unsigned>(a.group);
    const int row = static_cast<int>(blockIdx.x % rows), pair = static_cast<int>(blockIdx.x / rows);
    const int b = pair / kv.kv_heads, kv_head = pair - b * kv.kv_heads;
    const size_t from = static_cast<size_t>(blockIdx.x) * a.splits;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + from;
    for (int d0 = 0; d0 < kv.padded; d0 += 128) {
        const int d = d0 + (tid & 31) * 4, d_in = min(d, kv.padded - 4);
        const float* partial = a.partial + from * kv.padded + d_in;
        floatx4 x[kAhead];
        float2 st[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = min(group + 8 * u, a.splits - 1);
            x[u] = *reinterpret_cast<const floatx4*>(partial + static_cast<size_t>(k) * kv.padded);
            st[u] = stats[k];
        }
        const Span s = span_of(a, b, row / rows_of_tile * rows_of_tile, rows_of_tile, 0);
        if (row >= s.rows || s.left_out) return;
        const int used = splits_used(a, s);
        if (used == 1) return;
        float m = -INFINITY;
        for (int k = tid & 31; k < used; k += 32) m = fmaxf(m, stats[k].x);
        for (int y = 16; y > 0; y >>= 1) m = fmaxf(m, __shfl_xor(m, y));        // (every half wave finds the same maximum)
        const float base = m == -INFINITY ? 0.0f : m;
        floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (group + 8 * u < used) {
                const float weight = __builtin_amdgcn_exp2f(st[u].x - base);
                l += st[u].y * weight;
                sum += x[u] * weight;
            }
        for (int k = group + 8 * kAhead; k < used; k += 8) {
            const float weight = __builtin_amdgcn_exp2f(stats[k].x - base);
            l += stats[k].y * weight;
            sum += *reinterpret_cast<const floatx4*>(partial + static_cast<size_t>(k) * kv.padded) * weight;
        }
        sums[tid] = sum;
        if ((tid & 31) == 0) totals[group] = l;
        __syncthreads();
        if (tid < 32 && d < kv.padded) {
            l = totals[0];
            for (int k = 1; k < 8; ++k) {
                sum += sums[tid + 32 * k];
                l += totals[k];
            }
            const int i = row / a.group, h = kv_head * a.group + row % a.group;
            put(a.out.data + b * a.out.sequence_stride + i * a.out.token_stride + h * kv.head_width, sum / l, d, kv.head_width, a.wide);
        }
        __syncthreads();
    }
}

template <int DP, int CT, int W, int G>
hipError_t launch_many(Lane* lane, const AttendArgs& a, unsigned groups)
{
    constexpr int kLds = G * 2 * 2 * DP * kKvBlock * 2;
    static LdsLimit limit;
    const hipError_t e = limit.ensure(lane->device, reinterpret_cast<const void*>(&attend_many_kernel<DP, CT, W, G>), kLds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attend_many_kernel<DP, CT, W, G>), dim3(groups), dim3(G * W * 64), kLds, lane->stream, a);
    return hipGetLastError();
}

template <int DP>
hipError_t launch(Lane* lane, const AttendArgs& a, const AttendPlan& p)
{
    const int tiles = p.rows_of_tile / 16;
    const unsigned groups = static_cast<unsigned>(a.cache.sequences) * static_cast<unsigned>(a.cache.kv_heads) * static_cast<unsigned>(a.row_tiles) * static_cast<unsigned>(a.splits);
    if (p.few) {
        if constexpr (DP <= 128) {
            if (tiles == 2) {
                hipLaunchKernelGGL((attend_few_kernel<DP, 2>), dim3(groups), dim3(kThreads), 0, lane->stream, a);
                return hipGetLastError();
            }
        }
        hipLaunchKernelGGL((attend_few_kernel<DP, 1>), dim3(groups), dim3(kThreads), 0, lane->stream, a);
        return hipGetLastError();
    }
    if constexpr (DP <= 128) {
        if (tiles == 8) return launch_many<DP, 2, 4, 1>(lane, a, groups);
        return p.teams == 2 ? launch_many<DP, 1, 4, 2>(lane, a, groups) : launch_many<DP, 1, 4, 1>(lane, a, groups);
    } else {
        return tiles == 8 ? launch_many<DP, 1, 8, 1>(lane, a, groups) : launch_many<DP, 1, 4, 1>(lane, a, groups);
    }
}

}  // namespace

// Splits of the keys and scratch floats for a call; the caller provides the scratch memory.
AttendPlan plan_cached_attention(const KvLayout& cache, const nnhip_attention_desc& d, int compute_units)
{
    AttendPlan p{};
    const int64_t rows = static_cast<int64_t>(d.tokens) * (d.heads / cache.kv_heads);
    p.few = rows <= 32;
    p.least = 4;
    const int64_t pairs = static_cast<int64_t>(cache.sequences) * cache.kv_heads;
    // the blocks that a tile of rows can see, the most splits they are worth
    auto blocks_of = [&](int rows_of_tile) {
        int64_t blocks = cache.blocks;
        if (d.window > 0) {
            const int64_t seen = (static_cast<int64_t>(d.window) + rows_of_tile / (d.heads / cache.kv_heads) + 1) / kKvBlock + 2 +
                                 (static_cast<int64_t>(d.sinks) + kKvBlock - 1) / kKvBlock;
            blocks = blocks < seen ? blocks : seen;
        }
        return blocks;
    };
    auto most_splits = [&](int64_t blocks) { return blocks <= p.together ? 1 : (blocks + p.least - 1) / p.least; };
    p.rows_of_tile = rows <= 16 || cache.padded > 128 ? 16 : 32;
    // Short spans are not split: for a single token 16 blocks, which its four waves go through in about the time of a second
    // launch (one token, 32 heads on 8 of 128: over 500 tokens 9 us whole and 11.4 split, over 1000 11.8 either way, over 2000 17.4
    // in two splits and 11.9 in eight), 8 where blocks are larger (8 heads of 256 over 600: 17.0 and 14.3) and for prompts
    // (8 heads on one, 1017 tokens: 26.4 with 16, 23.7 with 8; 4 on one, 390 tokens: 15.2 with 8, 16.8 with 4).
    p.together = p.few && cache.padded * p.rows_of_tile <= 128 * 16 ? 16 : 8;
    if (!p.few && cache.padded <= 128) {
        // 128 rows halve what a row costs in LDS reads and conversions, 64 fill the device twice as well: 1000 tokens of 40 heads
        // on 8 (320 tiles of 128 rows) take 55 us with 128 and 36 with 64, four sequences of 512 tokens behind
        // 3000, 32 heads on 16 (512 tiles), 94 and 101, 2000 tokens of the first 101 and 103, 4093 tokens 320 and 364.
        p.rows_of_tile = (rows + 127) / 128 * pairs >= 2 * compute_units ? 128 : 64;
    } else if (!p.few) {
        // A unit holds one workgroup here, of eight waves or four, whose steps of a block take about 15 and 8: the form whose
        // workgroups are through first (heads of 256, 128 and 64 rows: 4000 tokens of 16 on 4 231 and 340 us, 2357 of 4 on 2 64 and
        // 99, 600 of 8 behind 20000 185 and 276, 1376 of 4 42 and 45, 700 of 16 on 8 48 and 37, 60 of 8 on 2 behind 500 27 and 22).
        auto steps = [&](int rows_of_tile, int64_t step) {
            const int64_t tiles = (rows + rows_of_tile - 1) / rows_of_tile * pairs, blocks = blocks_of(rows_of_tile);
            const int64_t free = std::max<int64_t>(compute_units / tiles, 1), splits = std::min<int64_t>(free, most_splits(blocks));
            return static_cast<double>(std::max<int64_t>(compute_units, tiles * splits)) * static_cast<double>((blocks + splits - 1) / splits * step);
        };
        p.rows_of_tile = steps(128, 15) <= steps(64, 8) ? 128 : 64;
    }
    p.row_tiles = static_cast<int>((rows + p.rows_of_tile - 1) / p.rows_of_tile);
    const int64_t groups = pairs * p.row_tiles;
    // Workgroups to aim at, rounded down: one more than fit at a time and the units wait for it (17 sequences of 5 tokens behind
    // 4768, 10 heads on 2: 39 us with 272 workgroups, 25 with 238).  One a compute unit: every further split costs its prologue and a
    // partial result to add up (one token over 131000, 8 pairs: 48 us with one a unit, 50 with two, 54 with three), and prompts
    // have thousands of those (1500 tokens behind 500, 8 heads of 128: 45 us whole, 52 in two splits and one and a half
    // workgroups a unit; 400 tokens of 8 heads on one behind 16000: 77 and 105).  Two a unit for single tokens, where a unit holds two
    // (as DP * CT in attend_few_kernel), when blocks are small (four sequences of 30000 tokens, 16 heads of 64: 54 us with one, 46
    // with two) or one would leave a tenth of the units free (136 pairs over 8000, 5 heads each: 71 us with 136 workgroups, 64 with
    // 272, 54 with 408; 24 pairs over 30000: 47 with 264, 37 with 240 or 504).
    const int64_t full = groups * (compute_units / groups);
    const bool two = p.few && cache.padded * p.rows_of_tile <= 128 * 16 && (cache.padded <= 64 || full * 10 < compute_units * 9);
    int64_t splits = (two ? 2 : 1) * compute_units / groups;
    const int64_t most = most_splits(blocks_of(p.rows_of_tile));
    if (splits > most) splits = most;
    p.splits = static_cast<int>(splits < 1 ? 1 : splits);
    // Tiles that leave every compute unit at most one workgroup are taken by two teams: 2000 tokens of 8 heads on 8 take 47 us
    // instead of 58, 1000 of 8 on 2 27 instead of 32, 64 of 32 on 8 behind 8000 41 instead of 45; with more tiles than units the
    // two workgroups of a unit do the same (500 tokens of 40 on 8: 22 and 21).
    p.teams = !p.few && cache.padded <= 128 && p.rows_of_tile == 64 && groups * p.splits <= compute_units ? 2 : 1;
    if (p.splits > 1) {
        p.stats_at = static_cast<size_t>(cache.sequences) * cache.kv_heads * rows * p.splits * cache.padded;
        p.scratch_floats = p.stats_at + static_cast<size_t>(cache.sequences) * cache.kv_heads * rows * p.splits * 2;
    }
    return p;
}

hipError_t launch_cached_attention(Lane* lane, const KvLayout& cache, const nnhip_attention_desc& d, const AttendPlan& p, float* scratch)
{
    AttendArgs a{cache, d.tokens, d.counts, d.q, d.out, d.heads, d.heads / cache.kv_heads, d.window, d.sinks, d.scale * 1.44269504088896340736f, false, p.row_tiles,
                 p.splits, p.least, p.together, scratch, scratch ? scratch + p.stats_at : nullptr};
    auto aligned = [](const nnhip_rows& r) {
        return (reinterpret_cast<uintptr_t>(r.data) & 15u) == 0 && r.token_stride % 4 == 0 && r.sequence_stride % 4 == 0;
    };
    a.wide = cache.head_width % 4 == 0 && aligned(d.q) && aligned(d.out);
    hipError_t e;
    switch (cache.padded) {
    case 32: e = launch<32>(lane, a, p); break;
    case 64: e = launch<64>(lane, a, p); break;
    case 96: e = launch<96>(lane, a, p); break;
    case 128: e = launch<128>(lane, a, p); break;
    case 192: e = launch<192>(lane, a, p); break;
    default: e = launch<256>(lane, a, p); break;
    }
    if (e != hipSuccess || p.splits == 1) return e;
    const unsigned rows = static_cast<unsigned>(cache.sequences) * static_cast<unsigned>(d.tokens) * static_cast<unsigned>(d.heads);
    if (p.splits <= kFewSplits) {
        const int together = kThreads / (cache.padded / 4);
        hipLaunchKernelGGL(attend_join_few_kernel, dim3((rows + together - 1) / together), dim3(kThreads), 0, lane->stream, a, p.rows_of_tile, together, rows);
    } else {
        hipLaunchKernelGGL(attend_join_kernel, dim3(rows), dim3(kThreads), 0, lane->stream, a, p.rows_of_tile);
    }
    return hipGetLastError();
}

}  // namespace nnhip
