// How the products on tcgen05 write their results, and are launched.
#pragma once

#include "common.cuh"
#include "linear8.h"

#include <cooperative_groups.h>

namespace linear8 {

// 32 rows (the warp's lanes) x 32 columns of sums, turned round in shared memory so that lanes side by side write 16 bytes each of one row:
// a thread's own row would be a sector of each of 32 rows a store, which the way to memory takes several times as long for.
template <typename TO>
constexpr int PIECE_PITCH = 32 * sizeof(TO) + 16;
template <typename TO>
constexpr int PIECE_BYTES = 32 * PIECE_PITCH<TO>;
template <typename TO>
__device__ __forceinline__ void store_piece(const Operands& p, unsigned char* piece, const unsigned long long* sums, int m0, int n0, int lane) {
    constexpr int EACH = 16 / sizeof(TO), LANES = 32 / EACH;  // columns of 16 bytes; lanes of a row
    unsigned char* mine = piece + lane * PIECE_PITCH<TO>;
#pragma unroll
    for (int j = 0; j < 32; j += EACH) {
        if constexpr (sizeof(TO) == 4) {
            *reinterpret_cast<ulonglong2*>(mine + j * 4) = make_ulonglong2(sums[j / 2], sums[j / 2 + 1]);
        } else {
            unsigned u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(__uint_as_float((unsigned)sums[j / 2 + i]), __uint_as_float((unsigned)(sums[j / 2 + i] >> 32)));
                u[i] = *reinterpret_cast<const unsigned*>(&a);
            }
            *reinterpret_cast<uint4*>(mine + j * 2) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
    __syncwarp();
    if (((uintptr_t)p.out & 15) != 0 || (p.ldo * sizeof(TO)) % 16 != 0) {
        // rows that start anywhere: lanes side by side write one element each of one row (8 elements a lane took 20 us more of 537 x 9,593 x 7,056)
        for (int row = 0; row < 32; ++row)
            if (m0 + row < p.M && n0 + lane < p.N)
                reinterpret_cast<TO*>(p.out)[(size_t)(m0 + row) * p.ldo + n0 + lane] = *reinterpret_cast<const TO*>(piece + row * PIECE_PITCH<TO> + lane * sizeof(TO));
        __syncwarp();  // the piece is written again
        return;
    }
    const int c = (lane % LANES) * EACH, valid = p.N - n0 - c;
    TO* out = reinterpret_cast<TO*>(p.out) + n0 + c;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 32 / LANES) {
        const int row = r0 + lane / LANES, m = m0 + row;
        if (m >= p.M) continue;
        const unsigned char* from = piece + row * PIECE_PITCH<TO> + c * sizeof(TO);
        if (valid >= EACH) {
            *reinterpret_cast<uint4*>(out + (size_t)m * p.ldo) = *reinterpret_cast<const uint4*>(from);
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                if (i < valid) out[(size_t)m * p.ldo + i] = reinterpret_cast<const TO*>(from)[i];
        }
    }
    __syncwarp();  // the piece is written again
}

// Some CTAs of a cluster have summed some of a tile's k-blocks each, [ROWS rows of x][WIDTH rows of w + 4] floats in shared memory: `split`
// of them, from rank `first` on every `step`-th, of which this is number `index`.  Each adds up some rows of x, the partial sums in
// the order of the k-blocks (the cluster has met since they were written); a thread asks for BATCH times four sums of every CTA at once, which take some 700 cycles.
template <int ROWS, int WIDTH, int THREADS, int MAX_SPLIT, int BATCH, typename TO>
__device__ __forceinline__ void join_cluster(const Operands& p, const float* sums, int split, int index, int first, int step, int m0, int n0) {
    constexpr int PITCH = WIDTH + 4, PARTS = WIDTH / 4;
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int rows = min(ROWS, p.M - m0), total = ((rows - index + split - 1) / split) * PARTS;  // this CTA's: rows index, index + split, ..
    for (int i0 = threadIdx.x; i0 < total; i0 += THREADS * BATCH) {
        float4 v[BATCH][MAX_SPLIT];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int i = min(i0 + b * THREADS, total - 1), m = (i / PARTS) * split + index, c = (i % PARTS) * 4;
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r)
                if (r < split) v[b][r] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(sums + m * PITCH + c, first + step * r));
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int i = i0 + b * THREADS, m = (i / PARTS) * split + index, n = n0 + (i % PARTS) * 4;
            if (i >= total || n >= p.N) continue;
            float y[4] = {v[b][0].x, v[b][0].y, v[b][0].z, v[b][0].w};
#pragma unroll
            for (int r = 1; r < MAX_SPLIT; ++r)
                if (r < split) {
                    y[0] += v[b][r].x;
                    y[1] += v[b][r].y;
                    y[2] += v[b][r].z;
                    y[3] += v[b][r].w;
                }
            TO* out = reinterpret_cast<TO*>(p.out) + (size_t)(m0 + m) * p.ldo + n;
            if (n + 4 <= p.N && ((uintptr_t)out & (4 * sizeof(TO) - 1)) == 0) {
                store4(out, y);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < p.N) out[j] = from_float<TO>(y[j]);
            }
        }
    }
    // nobody leaves while its sums are read (which has been done: nothing has to be made visible)
    asm volatile("barrier.cluster.arrive.relaxed;\nbarrier.cluster.wait;\n" ::: "memory");
}

// In clusters of `size` CTAs, behind the kernel in front as launch_pdl does it.
template <typename... Params, typename... Args>
inline int launch_clusters(void (*kernel)(Params...), unsigned blocks, unsigned threads, size_t smem, unsigned size, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace linear8
