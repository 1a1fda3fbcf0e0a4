// Memory layout of the 8-bit key/value cache (nnhip_kv_cache), shared by the kernels that write and read it.
//
// A block is 64 consecutive tokens of one key/value head; its codes are stored biased (byte = code + 128), so that one byte
// permutation and one packed subtraction turn two of them into half-precision numbers.  Both orders below are the operand
// order of v_mfma_f32_16x16x32_f16, so that a wave reads whole kilobytes in lane order and shuffles nothing:
//   keys    [64-wide chunk c][16 tokens j][lane][16 bytes]: lane = g * 16 + token % 16, bytes = components 64c + 16g ..+15
//           (a last chunk of 32 components: [j][lane][8 bytes], components 64c + 8g ..+7);
//   values  [16 components dt][lane][16 bytes]: lane = g * 16 + component % 16, byte 4j + i = token 16j + 4g + i: the
//           tokens whose probabilities the accumulators of the key product leave in the lanes of group g.
// head_width is padded to the next of 32, 64, 96, 128, 192, 256; padded components hold code 0.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nnhip.h"

namespace nnhip {

constexpr int kKvBlock = NNHIP_KV_BLOCK_TOKENS;
constexpr int kKvMaxWidth = 256;

__host__ __device__ inline int kv_padded_width(int head_width)
{
    if (head_width <= 128) return (head_width + 31) & ~31;
    return (head_width + 63) & ~63;
}

// Byte of the key code of token t (0..63), component d inside a block.
__host__ __device__ inline int kv_key_offset(int padded, int t, int d)
{
    const int c = d >> 6, j = t >> 4;
    if ((c + 1) * 64 <= padded) {
        const int g = (d >> 4) & 3;
        return c * 4096 + j * 1024 + (g * 16 + (t & 15)) * 16 + (d & 15);
    }
    const int g = (d >> 3) & 3;
    return c * 4096 + j * 512 + (g * 16 + (t & 15)) * 8 + (d & 7);
}

// Byte of the value code of token t, component d inside a block.
__host__ __device__ inline int kv_value_offset(int t, int d)
{
    const int j = t >> 4, g = (t >> 2) & 3, i = t & 3;
    return (d >> 4) * 1024 + (g * 16 + (d & 15)) * 16 + 4 * j + i;
}

// Where the parts of one cache lie.  "pair" = one sequence and key/value head: sequence * kv_heads + head.
struct KvLayout {
    uint8_t* base;
    int32_t* lengths;
    int sequences, kv_heads, head_width, capacity;
    int padded;             // components stored for each token
    int blocks;             // blocks of each pair
    size_t code_bytes;      // bytes of all key codes (the value codes follow, as many)
    size_t scales_at, open_at, marks_at;

    __host__ __device__ size_t block_bytes() const { return static_cast<size_t>(kKvBlock) * padded; }
    // codes of a block; which: 0 keys, 1 values
    __host__ __device__ uint8_t* codes(int which, int pair, int block) const
    {
        return base + which * code_bytes + (static_cast<size_t>(pair) * blocks + block) * block_bytes();
    }
    // [2]: key scale, value scale
    __host__ __device__ float* scales(int pair, int block) const
    {
        return reinterpret_cast<float*>(base + scales_at) + (static_cast<size_t>(pair) * blocks + block) * 2;
    }
    // FP32 values of the tokens of the last block stored, [64][padded] (keys turned by their positions): two buffers, so that a
    // call may fill up one block and open another in workgroups that do not wait for each other
    __host__ __device__ float* open_values(int which, int pair, int buffer) const
    {
        return reinterpret_cast<float*>(base + open_at) + ((static_cast<size_t>(pair) * 2 + which) * 2 + buffer) * kKvBlock * padded;
    }
    // [2 buffers][2]: the index of the block held, the number of its tokens (those whose values in the buffer still are the
    // block's, plus a flag where the block went on without the buffer)
    __host__ __device__ int32_t* marks(int which, int pair) const
    {
        return reinterpret_cast<int32_t*>(base + marks_at) + (static_cast<size_t>(pair) * 2 + which) * 4;
    }
};

// Whole size in *bytes; false when it does not fit 63 bits.  Sizes are positive, head_width at most kKvMaxWidth.
inline bool kv_layout(int sequences, int kv_heads, int head_width, int capacity, KvLayout* out, uint64_t* bytes)
{
    KvLayout k{};
    k.sequences = sequences;
    k.kv_heads = kv_heads;
    k.head_width = head_width;
    k.capacity = capacity;
    k.padded = kv_padded_width(head_width);
    k.blocks = static_cast<int>((static_cast<int64_t>(capacity) + kKvBlock - 1) / kKvBlock);
    const unsigned __int128 pairs = static_cast<unsigned __int128>(sequences) * kv_heads;
    const unsigned __int128 code = pairs * k.blocks * kKvBlock * k.padded;
    const unsigned __int128 scale = (pairs * k.blocks * 8 + 255) / 256 * 256;
    const unsigned __int128 open = pairs * 4 * kKvBlock * k.padded * 4;
    const unsigned __int128 total = 2 * code + scale + open + pairs * 32;
    // (positions stay a block away from the largest integer)
    if (capacity > 0x40000000 || pairs > 0x7fffffff || total >> 62) return false;
    k.code_bytes = static_cast<size_t>(code);
    k.scales_at = static_cast<size_t>(2 * code);
    k.open_at = static_cast<size_t>(2 * code + scale);
    k.marks_at = static_cast<size_t>(2 * code + scale + open);
    *out = k;
    *bytes = static_cast<uint64_t>(total);
    return true;
}

// Tokens of sequence b in this call (0 for one that is left out), and whether it is left out.
__device__ inline int kv_tokens_of(int start, int capacity, int tokens, const int32_t* counts, int b, bool* left_out)
{
    int n = counts ? counts[b] : tokens;
    n = n < 0 ? 0 : (n > tokens ? tokens : n);
    *left_out = start < 0 || static_cast<int64_t>(start) + n > capacity;
    return n;
}

}  // namespace nnhip
