// Attention over the 8-bit key/value cache (nnhip_cached_attention): causal, grouped query heads, optional sliding window
// with the first tokens kept visible.
//
// One wave takes one query row and walks over the blocks of 64 keys with the running maximum m and sum l of the softmax:
//     s_t = scale q . K_t,   m' = max(m, max_t s_t),   l' = l e^(m - m') + sum_t e^(s_t - m'),   o' = o e^(m - m') + sum_t e^(s_t - m') V_t
// and writes o / l.  A lane holds the score of one token, then the components d, d + 64, ... of o.
#include "kv_cache_layout.h"
#include "nnhip_internal.h"

namespace nnhip {

namespace {

struct AttendArgs {
    KvLayout cache;
    int tokens;
    const int32_t* counts;
    nnhip_rows q, out;
    int heads, window, sinks;
    float scale;
};

__global__ __launch_bounds__(64) void attend_row_kernel(const AttendArgs a)
{
    __shared__ float query[kKvMaxWidth];
    __shared__ float prob[kKvBlock];
    const KvLayout& kv = a.cache;
    const int lane = threadIdx.x, width = kv.head_width;
    const unsigned row = blockIdx.x;
    const int h = static_cast<int>(row % static_cast<unsigned>(a.heads));
    const int i = static_cast<int>(row / static_cast<unsigned>(a.heads) % static_cast<unsigned>(a.tokens));
    const int b = static_cast<int>(row / static_cast<unsigned>(a.heads) / static_cast<unsigned>(a.tokens));
    const int start = kv.lengths[b];
    bool left_out;
    const int n = kv_tokens_of(start, kv.capacity, a.tokens, a.counts, b, &left_out);
    if (i >= n) return;
    const float* q = a.q.data + b * a.q.sequence_stride + i * a.q.token_stride + h * width;
    float* out = a.out.data + b * a.out.sequence_stride + i * a.out.token_stride + h * width;
    if (left_out) {
        for (int d = lane; d < width; d += 64) out[d] = __uint_as_float(0x7fc00000u);
        return;
    }
    const int pair = b * kv.kv_heads + h / (a.heads / kv.kv_heads), p = start + i;
    const int low = a.window > 0 && p >= a.window ? p - a.window + 1 : 0;       // first key of the window
    for (int d = lane; d < width; d += 64) query[d] = q[d];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[kKvMaxWidth / 64] = {};
    for (int block = 0; block * kKvBlock <= p; ++block) {
        if (block * kKvBlock + kKvBlock <= low && block * kKvBlock >= a.sinks) {
            block = low / kKvBlock - 1;
            continue;
        }
        const int t = block * kKvBlock + lane;
        const bool seen = t <= p && (t >= low || t < a.sinks);
        const float* scales = kv.scales(pair, block);
        const uint8_t* k = kv.codes(0, pair, block);
        float s = 0.0f;
        for (int d = 0; d < width; ++d) s = fmaf(query[d], static_cast<float>(k[kv_key_offset(kv.padded, lane, d)] - 128), s);
        s = s * scales[0] * a.scale;
        float top = seen ? s : -INFINITY;
        for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float next = fmaxf(m, top), base = next == -INFINITY ? 0.0f : next;
        const float keep = expf(m - base), e = seen ? expf(s - base) : 0.0f;
        m = next;
        prob[lane] = seen ? e * scales[1] : 0.0f;
        __syncthreads();
        l = l * keep + e;
        const uint8_t* v = kv.codes(1, pair, block);
        for (int c = 0; c * 64 < width; ++c) {
            o[c] *= keep;
            const int d = c * 64 + lane;
            if (d >= width) continue;
            for (int u = 0; u < kKvBlock; ++u)
                if (prob[u] != 0.0f) o[c] = fmaf(prob[u], static_cast<float>(v[kv_value_offset(u, d)] - 128), o[c]);
        }
        __syncthreads();
    }
    for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
    for (int c = 0; c * 64 < width; ++c)
        if (c * 64 + lane < width) out[c * 64 + lane] = o[c] / l;
}

}  // namespace

hipError_t launch_cached_attention(Lane* lane, const KvLayout& cache, const nnhip_attention_desc& d)
{
    const AttendArgs a{cache, d.tokens, d.counts, d.q, d.out, d.heads, d.window, d.sinks, d.scale};
    hipLaunchKernelGGL(attend_row_kernel, dim3(static_cast<unsigned>(cache.sequences) * static_cast<unsigned>(d.tokens) * static_cast<unsigned>(d.heads)),
                       dim3(64), 0, lane->stream, a);
    return hipGetLastError();
}

}  // namespace nnhip
