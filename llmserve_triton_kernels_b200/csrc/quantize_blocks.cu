// values[m, k] = e4m3(x[m, k] / s), s a power of two for every block of 128 columns of one row (activations) or of 128 rows
// (weights); see fp8.cuh for the scale.  One pass: a block's values stay in registers between its maximum and its rounding, so
// every input byte is read once and every output byte written once.  The bytes bound it: a weight of 4,096 x 14,336 in 32 bits takes
// 43.7 us, 6.7 TB/s (a copy reaches 6.57 on this chip); with 256 threads a block of 128 x 128 instead of 512 it took 75.  A decode step's
// rows (8 x 5,632) take 2 us, which is a launch.
#include "fp8.cuh"
#include "linear8.h"

namespace {

constexpr int THREADS = 256, TILE_THREADS = 512, BLOCK = 128;

using fp8::load8;

__device__ __forceinline__ unsigned top_of(const float (&v)[8]) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, fp8::finite_bits(v[i]));
    return top;
}

__device__ __forceinline__ void store8(unsigned char* p, const float (&v)[8], float inv) {
    *reinterpret_cast<uint2*>(p) = make_uint2(fp8::pack4(v[0], v[1], v[2], v[3], inv), fp8::pack4(v[4], v[5], v[6], v[7], inv));
}

// Rows on their own, K a multiple of 8 and rows on 16 bytes: half a warp a block, eight values a lane.  UNROLL blocks a
// half warp are on their way at once.  `across`: the scales are laid down block by block, [blocks][M], as products read them.
template <typename T, int UNROLL>
__global__ void __launch_bounds__(THREADS)
quantize_rows_kernel(const T* __restrict__ x, long long ldx, unsigned char* __restrict__ values, float* __restrict__ scales, int M, int K, int across) {
    pdl_wait();
    pdl_trigger();  // after the wait: whoever starts behind this kernel starts when everything in front of it has ended
    const int kblocks = (K + BLOCK - 1) / BLOCK, lane = threadIdx.x & 15;
    const unsigned mask = (threadIdx.x & 16) ? 0xffff0000u : 0x0000ffffu;
    const long long blocks = (long long)M * kblocks, step = (long long)gridDim.x * (THREADS / 16);
    for (long long b0 = (long long)blockIdx.x * (THREADS / 16) + (threadIdx.x >> 4); b0 < blocks; b0 += step * UNROLL) {
        float v[UNROLL][8];
        long long row[UNROLL];
        int col[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long long b = b0 + u * step;
            row[u] = b / kblocks;
            col[u] = (int)(b - row[u] * kblocks) * BLOCK + lane * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
            if (b < blocks && col[u] < K) load8(x + row[u] * ldx + col[u], v[u]);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const unsigned e = fp8::scale_exponent(__reduce_max_sync(mask, top_of(v[u])));
            const long long b = b0 + u * step;
            if (b >= blocks) continue;
            if (col[u] < K) store8(values + row[u] * K + col[u], v[u], fp8::inverse(e));
            if (lane == 0) scales[across ? (b - row[u] * kblocks) * M + row[u] : b] = fp8::power(e);
        }
    }
}

// ... any K, any layout: a warp a block.
template <typename T>
__global__ void __launch_bounds__(THREADS)
quantize_rows_any_kernel(const T* __restrict__ x, long long ldx, unsigned char* __restrict__ values, float* __restrict__ scales, int M, int K, int across) {
    pdl_wait();
    pdl_trigger();
    const int kblocks = (K + BLOCK - 1) / BLOCK, lane = threadIdx.x & 31;
    const long long blocks = (long long)M * kblocks, step = (long long)gridDim.x * (THREADS / 32);
    for (long long b = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); b < blocks; b += step) {
        const long long row = b / kblocks;
        const int k0 = (int)(b - row * kblocks) * BLOCK + lane;
        float v[4];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = k0 + 32 * i < K ? to_float(x[row * ldx + k0 + 32 * i]) : 0.f;
            top = max(top, fp8::finite_bits(v[i]));
        }
        const unsigned e = fp8::scale_exponent(__reduce_max_sync(0xffffffffu, top));
        const float inv = fp8::inverse(e);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k0 + 32 * i < K) values[row * K + k0 + 32 * i] = (unsigned char)fp8::pack2(v[i], 0.f, inv);
        if (lane == 0) scales[across ? (b - row * kblocks) * M + row : b] = fp8::power(e);
    }
}

// Blocks of 128 x 128, one a CTA: 32 values a thread.  VECTOR: K a multiple of 8 and rows on 16 bytes.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(TILE_THREADS, 2)
quantize_tiles_kernel(const T* __restrict__ x, long long ldx, unsigned char* __restrict__ values, float* __restrict__ scales, int M, int K) {
    constexpr int PER = BLOCK / (TILE_THREADS / 16);  // rows a thread
    __shared__ unsigned tops[TILE_THREADS / 32];
    pdl_wait();
    pdl_trigger();
    const int kblocks = (K + BLOCK - 1) / BLOCK;
    const int tile_row = blockIdx.x / kblocks, tile_col = blockIdx.x - tile_row * kblocks;
    const int r0 = tile_row * BLOCK + (threadIdx.x >> 4), c0 = tile_col * BLOCK + (threadIdx.x & 15) * 8;
    float v[PER][8];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = r0 + (TILE_THREADS / 16) * i;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (r < M && c0 < K) {
            if (VECTOR) {
                load8(x + (long long)r * ldx + c0, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c0 + j < K) v[i][j] = to_float(x[(long long)r * ldx + c0 + j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) top = max(top, top_of(v[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TILE_THREADS / 32; ++w) top = max(top, tops[w]);
    const unsigned e = fp8::scale_exponent(top);
    const float inv = fp8::inverse(e);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int r = r0 + (TILE_THREADS / 16) * i;
        if (r >= M || c0 >= K) continue;
        if (VECTOR) {
            store8(values + (long long)r * K + c0, v[i], inv);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < K) values[(long long)r * K + c0 + j] = (unsigned char)fp8::pack2(v[i][j], 0.f, inv);
        }
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = fp8::power(e);
}

template <typename T>
int launch(const void* x, long long ldx, unsigned char* values, float* scales, int M, int K, int rows, int across, cudaStream_t stream) {
    const T* p = (const T*)x;
    const long long kblocks = (K + BLOCK - 1) / BLOCK;
    const bool vector = K % 8 == 0 && ((uintptr_t)x & 15) == 0 && (ldx * sizeof(T)) % 16 == 0 && ((uintptr_t)values & 7) == 0;
    if (rows == BLOCK) {
        const long long tiles = (long long)((M + BLOCK - 1) / BLOCK) * kblocks;
        if (tiles > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
        return vector ? launch_pdl(quantize_tiles_kernel<T, true>, dim3((unsigned)tiles), dim3(TILE_THREADS), 0, stream, p, ldx, values, scales, M, K)
                      : launch_pdl(quantize_tiles_kernel<T, false>, dim3((unsigned)tiles), dim3(TILE_THREADS), 0, stream, p, ldx, values, scales, M, K);
    }
    const long long blocks = (long long)M * kblocks, most = (long long)device_sms() * 8;
    const long long per = vector ? THREADS / 16 : THREADS / 32;
    const long long want = (blocks + per - 1) / per;
    const unsigned grid = (unsigned)(want < most ? want : most);
    if (!vector) return launch_pdl(quantize_rows_any_kernel<T>, dim3(grid), dim3(THREADS), 0, stream, p, ldx, values, scales, M, K, across);
    return launch_pdl(quantize_rows_kernel<T, 2>, dim3(grid), dim3(THREADS), 0, stream, p, ldx, values, scales, M, K, across);
}

}  // namespace

// x [M, K] (row stride ldx elements, unit inner stride; float32 or bfloat16) -> values [M, K] e4m3, contiguous, and scales float32
// [M, ceil(K / 128)] (rows 1) or [ceil(M / 128), ceil(K / 128)] (rows 128).
LLM_EXPORT int llm_quantize_blocks(const void* x, int dtype, long long ldx, unsigned char* values, float* scales, int M, int K, int rows,
                                   cudaStream_t stream) {
    if (M <= 0 || K <= 0) return 0;
    if (rows != 1 && rows != BLOCK) return LLM_ERR_BAD_ARGUMENT;
    if (dtype == LLM_F32) return launch<float>(x, ldx, values, scales, M, K, rows, 0, stream);
    if (dtype == LLM_BF16) return launch<__nv_bfloat16>(x, ldx, values, scales, M, K, rows, 0, stream);
    return LLM_ERR_BAD_ARGUMENT;
}

int linear8::quantize_rows(const void* x, int dtype, long long ldx, unsigned char* values, float* scales, int M, int K, cudaStream_t stream) {
    if (dtype == LLM_F32) return launch<float>(x, ldx, values, scales, M, K, 1, 1, stream);
    if (dtype == LLM_BF16) return launch<__nv_bfloat16>(x, ldx, values, scales, M, K, 1, 1, stream);
    return LLM_ERR_BAD_ARGUMENT;
}
