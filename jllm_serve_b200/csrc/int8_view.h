// What a launcher is told of a matrix in 8-bit integers: laid out once by whoever holds it, and not argument by argument at every call.
#pragma once
#include <stdint.h>

struct Int8View {
    const int8_t* data;
    const float* scale;
    int rows, cols, stride;      // stride: bytes from row to row, or, of a packed weight, its k blocks
};
// The kernels count rows and values in 32 bits and step past the end by up to a block's 8,192 values.
constexpr int INT8_MOST = 0x7fffffff - 8191;
