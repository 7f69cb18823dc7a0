// What a launcher is told of rows, of a packed weight and of groups of rows: laid out once by whoever holds them, and not argument by argument
// at every call.
#pragma once
#include <stdint.h>

// Rows of activations: bfloat16 (scale null), or e4m3 with a float32 scale for each 128 values of a row.
struct BlockRows {
    const void* data;
    const float* scale;
    long long stride;            // bytes from row to row
    int rows, cols, scale_ld;
};
// A packed weight of `groups` matrices [rows, cols]: the tiles, and of e4m3 the scales of every eight rows and 128 k.
struct BlockWeight {
    const void* data;
    const float* scale;
    int groups, rows, cols, k_blocks, scale_ld, glu;
};
// The pairs (row, choice) in the order of their groups: group g's are order[offsets[g]] .. order[offsets[g + 1] - 1]; place is the way back.
struct RowGroupsView {
    int *offsets, *order, *place, *counts;      // counts: room for up to GROUP_BLOCKS blocks' pairs by group (of more than 2,048 pairs)
    int rows, top, groups;
};
constexpr int GROUP_BLOCKS = 128;
// The kernels count rows, pairs and values in 32 bits and step past the end by up to a block's 8,192 values.
constexpr int BLOCK_MOST = 0x7fffffff - 8191;

#ifdef __CUDACC__
#define JLLM_HERE __host__ __device__ __forceinline__
#else
#define JLLM_HERE inline
#endif
struct alignas(8) Bytes8 {
    uint32_t lo, hi;
};
// Eight neighbouring bytes that begin at a multiple of 8, of which `left` exist: one load where all do, else none behind the last (the end of a row may be the
// end of its memory).
JLLM_HERE Bytes8 bytes_of(const uint8_t* p, int left) {
    if (left >= 8) return *reinterpret_cast<const Bytes8*>(p);
    Bytes8 b = {0, 0};
#pragma unroll
    for (int j = 0; j < 7; ++j)
        if (j < left) (j < 4 ? b.lo : b.hi) |= (uint32_t)p[j] << 8 * (j & 3);
    return b;
}
