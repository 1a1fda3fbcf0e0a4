// The 8-bit key/value cache: storing tokens (rotary positions, block quantisation), advancing the lengths, reading back.
//
// Definition (nnhip.h): scale = fl32(max |x| / 127) over a block, code = rint(x / scale).  The quotient is taken in 64 bits:
// it is then never rounded onto a half-integer that the exact one misses (x / scale of two FP32 numbers is either a
// half-integer or at least 2^-27 away from it), so the codes are a function of the stored values alone.  The rotation is done
// in 64 bits and rounded once, for positions where an FP32 angle has no correct digit of the turn left.
#include "kv_cache_layout.h"
#include "nnhip_internal.h"

namespace nnhip {

namespace {

constexpr int kThreads = 256;

struct StoreArgs {
    KvLayout cache;
    int tokens;
    const int32_t* counts;
    nnhip_rows k, v, q, q_out;
    const float* inv_freq;
    int rotary_width;
    uint32_t rotary_style;
    int heads;
    int slots;              // workgroups of each pair and kind: slot 0 takes the first and the last block, the others one each
    unsigned kv_groups;     // workgroups of the cache part; the query part follows
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

// One block of one head, keys or values: tokens [from, to) of the block are new, those before `from` are there already.
__device__ void store_block(const StoreArgs& a, float* tile, uint32_t* largest, int which, int b, int head, int pair, int block,
                            int start, int from, int to, bool last)
{
    const KvLayout& kv = a.cache;
    const int tid = threadIdx.x, width = kv.head_width, padded = kv.padded, pitch = padded + 1;
    const nnhip_rows& rows = which ? a.v : a.k;
    float* open = kv.open_values(which, pair);
    int32_t* marks = kv.marks(which, pair);
    uint8_t* codes = kv.codes(which, pair, block);
    float* scale_at = kv.scales(pair, block) + which;
    const bool held = from == 0 || (marks[0] == block && marks[1] >= from);     // the older tokens' FP32 values are at hand
    const float old_scale = held ? 0.0f : *scale_at;
    if (tid == 0) *largest = 0;
    for (int e = tid; e < kKvBlock * padded; e += kThreads) {
        const int t = e / padded, d = e - t * padded;
        float x = 0.0f;
        if (d < width && t < to) {
            if (t >= from)
                x = rows.data[b * rows.sequence_stride +
                              (static_cast<int64_t>(block) * kKvBlock + t - start) * rows.token_stride + head * width + d];
            else if (held)
                x = open[t * padded + d];
            else
                x = old_scale * static_cast<float>(codes[which ? kv_value_offset(t, d) : kv_key_offset(padded, t, d)] - 128);
        }
        tile[t * pitch + d] = x;
    }
    __syncthreads();
    if (which == 0 && a.inv_freq) {
        const int pairs = a.rotary_width / 2;
        for (int e = tid; e < (to - from) * pairs; e += kThreads) {
            const int t = from + e / pairs, j = e % pairs;
            double s, c;
            sincos(static_cast<double>(block * kKvBlock + t) * static_cast<double>(a.inv_freq[j]), &s, &c);
            int d0, d1;
            rotary_pair(a, j, &d0, &d1);
            turn(&tile[t * pitch + d0], &tile[t * pitch + d1], c, s);
        }
        __syncthreads();
    }
    uint32_t top = 0;           // |x| as bits: the order of the numbers, infinity and NaN above all
    for (int e = tid; e < to * padded; e += kThreads) {
        const int t = e / padded, d = e - t * padded;
        const uint32_t bits = __float_as_uint(tile[t * pitch + d]) & 0x7fffffffu;
        top = bits > top ? bits : top;
    }
    atomicMax(largest, top);
    __syncthreads();
    const uint32_t most = *largest;
    const bool finite = most < 0x7f800000u;
    const float scale = finite ? __uint_as_float(most) / 127.0f : __uint_as_float(0x7fc00000u);
    if (tid == 0) *scale_at = scale;
    for (int e = tid; e < kKvBlock * padded; e += kThreads) {
        const int t = e / padded, d = e - t * padded;
        int code = 0;
        if (finite && scale > 0.0f) {
            const double r = rint(static_cast<double>(tile[t * pitch + d]) / static_cast<double>(scale));
            code = static_cast<int>(fmin(fmax(r, -127.0), 127.0));
        }
        codes[which ? kv_value_offset(t, d) : kv_key_offset(padded, t, d)] = static_cast<uint8_t>(code + 128);
        if (last && t < to && (t >= from || !held)) open[t * padded + d] = tile[t * pitch + d];
    }
    __syncthreads();
    if (last && tid == 0) {
        marks[0] = block;
        marks[1] = to;
    }
}

__global__ __launch_bounds__(kThreads) void kv_store_kernel(const StoreArgs a)
{
    extern __shared__ float tile[];
    __shared__ uint32_t largest;
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
        // The first and the last block go through one workgroup, in this order: the first reads the FP32 values kept of the
        // open block, the last replaces them.
        for (int pass = 0; pass < 2; ++pass) {
            int block;
            if (slot == 0)
                block = pass == 0 ? first : final;
            else
                block = first + slot;
            if (pass == 1 && (slot != 0 || final == first)) break;
            if (slot != 0 && block >= final) break;
            const int from = block == first ? start - first * kKvBlock : 0;
            const int to = block == final ? end - final * kKvBlock : kKvBlock;
            store_block(a, tile, &largest, which, b, head, pair, block, start, from, to, block == final);
            __syncthreads();
        }
        return;
    }
    const unsigned at = blockIdx.x - a.kv_groups;
    const int b = static_cast<int>(at / static_cast<unsigned>(a.tokens)), i = static_cast<int>(at % static_cast<unsigned>(a.tokens));
    const int start = kv.lengths[b];
    const int n = kv_tokens_of(start, kv.capacity, a.tokens, a.counts, b, &left_out);
    if (left_out || i >= n) return;
    const float* q = a.q.data + b * a.q.sequence_stride + i * a.q.token_stride;
    float* out = a.q_out.data + b * a.q_out.sequence_stride + i * a.q_out.token_stride;
    const int pairs = a.rotary_width / 2, width = kv.head_width, rest = width - a.rotary_width;
    for (int e = threadIdx.x; e < a.heads * pairs; e += kThreads) {
        const int h = e / pairs, j = e - h * pairs;
        double s, c;
        sincos(static_cast<double>(start + i) * static_cast<double>(a.inv_freq[j]), &s, &c);
        int d0, d1;
        rotary_pair(a, j, &d0, &d1);
        float x = q[h * width + d0], y = q[h * width + d1];
        turn(&x, &y, c, s);
        out[h * width + d0] = x;
        out[h * width + d1] = y;
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

__global__ __launch_bounds__(kThreads) void kv_read_kernel(const KvLayout kv, const int32_t* first, int tokens, nnhip_rows k, nnhip_rows v)
{
    const int i = static_cast<int>(blockIdx.x % static_cast<unsigned>(tokens)), b = static_cast<int>(blockIdx.x / static_cast<unsigned>(tokens));
    const int64_t t = static_cast<int64_t>(first ? first[b] : 0) + i;
    const bool inside = t >= 0 && t < kv.capacity;
    const int block = inside ? static_cast<int>(t / kKvBlock) : 0, at = inside ? static_cast<int>(t % kKvBlock) : 0;
    for (int e = threadIdx.x; e < 2 * kv.kv_heads * kv.head_width; e += kThreads) {
        const int which = e / (kv.kv_heads * kv.head_width), c = e % (kv.kv_heads * kv.head_width);
        const nnhip_rows& rows = which ? v : k;
        if (!rows.data) continue;
        const int head = c / kv.head_width, d = c % kv.head_width, pair = b * kv.kv_heads + head;
        float x = 0.0f;
        if (inside)
            x = kv.scales(pair, block)[which] *
                static_cast<float>(kv.codes(which, pair, block)[which ? kv_value_offset(at, d) : kv_key_offset(kv.padded, at, d)] - 128);
        rows.data[b * rows.sequence_stride + i * rows.token_stride + c] = x;
    }
}

}  // namespace

hipError_t launch_kv_store(Lane* lane, const KvLayout& cache, const nnhip_kv_store_desc& d)
{
    StoreArgs a{cache, d.tokens, d.counts, d.k, d.v, d.q, d.q_out, d.inv_freq, d.rotary_width, d.rotary_style, d.heads, 0, 0};
    // n tokens touch at most (n + 62) / 64 + 1 blocks, of which the first and the last share a workgroup
    a.slots = static_cast<int>((static_cast<int64_t>(d.tokens) + kKvBlock - 2) / kKvBlock);
    if (a.slots < 1) a.slots = 1;
    a.kv_groups = static_cast<unsigned>(a.slots) * 2u * static_cast<unsigned>(cache.sequences * cache.kv_heads);
    const unsigned q_groups = d.q.data ? static_cast<unsigned>(cache.sequences) * static_cast<unsigned>(d.tokens) : 0u;
    const size_t lds = static_cast<size_t>(kKvBlock) * (cache.padded + 1) * sizeof(float);
    static LdsLimit big;
    const hipError_t e = big.ensure(lane->device, reinterpret_cast<const void*>(&kv_store_kernel), kKvBlock * (kKvMaxWidth + 1) * 4);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kv_store_kernel, dim3(a.kv_groups + q_groups), dim3(kThreads), lds, lane->stream, a);
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
    hipLaunchKernelGGL(kv_read_kernel, dim3(static_cast<unsigned>(cache.sequences) * static_cast<unsigned>(tokens)), dim3(kThreads), 0,
                       lane->stream, cache, first, tokens, k, v);
    return hipGetLastError();
}

}  // namespace nnhip
