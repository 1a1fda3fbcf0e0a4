// Log probabilities of given tokens, entropy and top alternatives of rows of logits (nnhip_token_log_probs).
//
// With m = max x, S = sum e^(x - m), T = sum (x - m) e^(x - m):
//     ln p[t] = (x_t - m) - ln S,    entropy = ln S - T / S.
// S and T are sums in 64 bits: the largest logit adds exactly 1 to S, so S - 1 keeps the digits that the entropy and the log
// probability of a peaked row consist of.
#include "nnhip_internal.h"

namespace nnhip {

namespace {

constexpr int kThreads = 256;

__device__ inline float order_value(float x) { return x != x ? INFINITY : x; }

__global__ __launch_bounds__(kThreads) void log_probs_kernel(const nnhip_log_probs_desc a)
{
    __shared__ double sums[2][kThreads];
    __shared__ float values[kThreads];
    __shared__ int ids[kThreads];
    const int tid = threadIdx.x, V = a.vocabulary;
    const float* x = a.logits + static_cast<int64_t>(blockIdx.x) * a.row_stride;
    float m = -INFINITY;
    bool nan = false;
    for (int i = tid; i < V; i += kThreads) {
        nan |= x[i] != x[i];
        m = fmaxf(m, x[i]);
    }
    values[tid] = nan ? INFINITY : m;
    __syncthreads();
    for (int s = kThreads / 2; s > 0; s >>= 1) {
        if (tid < s) values[tid] = fmaxf(values[tid], values[tid + s]);
        __syncthreads();
    }
    m = values[0];
    const bool defined = m > -INFINITY && m < INFINITY;
    double S = 0.0, T = 0.0;
    for (int i = tid; i < V && defined; i += kThreads) {
        const float d = fmaxf(x[i] - m, -200.0f), e = expf(d);
        S += e;
        T += d * e;
    }
    sums[0][tid] = S;
    sums[1][tid] = T;
    __syncthreads();
    for (int s = kThreads / 2; s > 0; s >>= 1) {
        if (tid < s) {
            sums[0][tid] += sums[0][tid + s];
            sums[1][tid] += sums[1][tid + s];
        }
        __syncthreads();
    }
    const float none = __uint_as_float(0x7fc00000u);
    const double log_sum = log1p(sums[0][0] - 1.0);
    if (tid == 0) {
        if (a.log_probs && a.targets) {
            const int t = a.targets[blockIdx.x];
            a.log_probs[blockIdx.x] = defined && t >= 0 && t < V ? static_cast<float>((static_cast<double>(x[t]) - m) - log_sum) : none;
        }
        if (a.entropy) a.entropy[blockIdx.x] = defined ? static_cast<float>(log_sum - sums[1][0] / sums[0][0]) : none;
    }
    float last = INFINITY;
    int last_id = -1;
    for (int k = 0; k < a.top; ++k) {       // the largest one behind the last one taken
        float best = 0.0f;
        int best_id = -1;
        for (int i = tid; i < V; i += kThreads) {
            const float v = order_value(x[i]);
            if ((v < last || (v == last && i > last_id)) && (best_id < 0 || v > best)) {
                best = v;
                best_id = i;
            }
        }
        __syncthreads();
        values[tid] = best;
        ids[tid] = best_id;
        __syncthreads();
        for (int s = kThreads / 2; s > 0; s >>= 1) {
            if (tid < s && ids[tid + s] >= 0 &&
                (ids[tid] < 0 || values[tid + s] > values[tid] || (values[tid + s] == values[tid] && ids[tid + s] < ids[tid]))) {
                values[tid] = values[tid + s];
                ids[tid] = ids[tid + s];
            }
            __syncthreads();
        }
        last = values[0];
        last_id = ids[0];
        if (tid == 0) {
            const size_t at = static_cast<size_t>(blockIdx.x) * a.top + k;
            a.top_ids[at] = last_id;
            if (a.top_log_probs) a.top_log_probs[at] = defined ? static_cast<float>((static_cast<double>(last) - m) - log_sum) : none;
        }
    }
}

}  // namespace

hipError_t launch_token_log_probs(Lane* lane, const nnhip_log_probs_desc& d)
{
    hipLaunchKernelGGL(log_probs_kernel, dim3(d.rows), dim3(kThreads), 0, lane->stream, d);
    return hipGetLastError();
}

}  // namespace nnhip
