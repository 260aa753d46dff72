// What the kernels of a product with 8-bit weights share: y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k].
#pragma once

#include <cuda_runtime.h>

namespace linear8 {

constexpr int FEW_ROWS = 64;  // up to this many rows of x the weights are streamed through mma.sync; more go to tcgen05

struct Operands {
    const unsigned char* x;  // [M, K] e4m3
    const float* sx;         // [M, kblocks]
    const unsigned char* w;  // [N, K] e4m3
    const float* sw;         // [ceil(N / 128), kblocks]
    void* out;               // [M, N], row stride ldo
    int M, N, K, kblocks, ldo, out_dtype;
};

// `early`: w and sw may be read while the kernel in front still runs.
int few(const Operands& p, bool early, cudaStream_t stream);
int many(const Operands& p, int* error_flag, cudaStream_t stream);

}  // namespace linear8
