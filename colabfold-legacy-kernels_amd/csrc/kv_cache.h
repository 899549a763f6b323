// The key-value cache's layout on the device, shared by the kernels that write and read it (heads.hip) and attention
// (paged_attn.hip).
//
// Keys and values are [pages, heads, page, D], D a multiple of 32 and page a multiple of 16. Within a page's head, blocks of
// 16 tokens lie one after another, each in the order in which v_mfma_f32_16x16x32 takes its A operand, so
// attention loads an operand as one contiguous kilobyte, into registers, with no transposition and no LDS:
//   keys    [D / W][16 tokens][W channels], 16 bytes a lane: W = 8 values of 16 bits or 16 of 8 bits
//   values  [D / (16 C)][4 g][16 i][C e][4 j]: token 4 g + j, channel 16 (C b + e) + i: four tokens of a channel side by
//           side, which is what a lane of the scores' result holds of a block, for C channels: 16 bytes a lane,
//           C = 2 for 16 bits and 4 for 8 bits (2, and 8 bytes, where D is no multiple of 64)
// An 8-bit cache has a scale a token and head beside them, [pages, heads, page] fp32, as 8-bit rows have.
#pragma once

#include "clk_common.h"

namespace clk {

constexpr int kCacheBlock = 16;  // tokens

__host__ __device__ constexpr int key_width(bool q8) { return q8 ? 16 : 8; }
__host__ __device__ constexpr int value_group(bool q8, int D) { return q8 && D % 64 == 0 ? 4 : 2; }

// Where channel c of token t (of 16) lies in a block of keys, and of values
__device__ __forceinline__ int key_place(bool q8, int t, int c) {
    return q8 ? (c >> 4) * 256 + t * 16 + (c & 15) : (c >> 3) * 128 + t * 8 + (c & 7);
}
__device__ __forceinline__ int value_place(int group, int t, int c) {  // group: 2 or 4
    const int b = c >> 4, shift = group == 4 ? 2 : 1;
    return (b >> shift) * (256 << shift) + (((t >> 2) * 16 + (c & 15)) << (shift + 2)) + (b & (group - 1)) * 4 + (t & 3);
}

struct CacheShape {
    int64_t pages = 0, heads = 0, page = 0, D = 0;
    bool q8 = false;
};

// The checks of a cache that the entry points share. 16-bit caches hold the activations' type.
int check_cache(const char* what, const clk_buffer* k, const clk_buffer* v, const clk_buffer* ks, const clk_buffer* vs, int act,
                CacheShape& shape);

}  // namespace clk
