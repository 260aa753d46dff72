// What the kernels of a product with 8-bit weights share: y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k].
#pragma once

#include <cuda_runtime.h>

namespace linear8 {

// Up to FEW_ROWS rows of x the weights are streamed through mma.sync, up to twice as many where the weights are FEW_BYTES at most.
constexpr int FEW_ROWS = 8;
constexpr long long FEW_BYTES = 20 << 20;

struct Operands {
    const unsigned char* x;  // [M, K] e4m3
    const float* sx;         // row m's scale of block b at m * sx_row + b * sx_block: warps read those of many rows at once, which lie side by
    int sx_row, sx_block;    // side where they were made for this, [kblocks, M]; a caller's are [M, kblocks]
    const unsigned char* w;  // [N, K] e4m3
    const float* sw;         // [ceil(N / 128), kblocks]
    void* out;               // [M, N], row stride ldo
    int M, N, K, kblocks, ldo, out_dtype;
};

// The rows of x [M, K] (float32 or bfloat16, row stride ldx) in 8 bits; scales [kblocks, M].
int quantize_rows(const void* x, int dtype, long long ldx, unsigned char* values, float* scales, int M, int K, cudaStream_t stream);
// `early`: w and sw may be read while the kernel in front still runs.
int few(const Operands& p, bool early, cudaStream_t stream);
int some(const Operands& p, bool early, int* error_flag, cudaStream_t stream);
// The same for scales that are powers of two, x's and the weights'.
int some_scaled(const Operands& p, bool early, int* error_flag, cudaStream_t stream);
int many_scaled(const Operands& p, int split, bool early, int* error_flag, cudaStream_t stream);
int many(const Operands& p, bool early, int* error_flag, cudaStream_t stream);

}  // namespace linear8
