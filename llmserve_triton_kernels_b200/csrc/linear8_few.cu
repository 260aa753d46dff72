// y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k] for up to 16 rows: x and w in e4m3, a scale for every 128 k.
//
// The weights are read from HBM once, 16 bytes a lane straight into tensor-core fragments; the rows of x ride along as the
// narrow side (the 16 rows of an mma.sync m16n8k32 tile are 16 output features, its 8 columns are 8 rows of x).  A lane takes
// 32 consecutive bytes of a weight row's 128-byte block: the k of the four products of a block are permuted the same way on
// both sides, which a sum over k does not notice, so that no shuffle and no shared memory stands between the load and the product.
// The eight warps of a CTA share a tile's k-blocks and meet once a tile.
//
// A block's four products start from zero and enter the 32-bit sums times both scales.  (The e4m3 product of mma.sync adds
// its 32 terms without loss on this chip: 2,048 terms came out within 1.6e-7 of the 64-bit sum.)
//
// The weights' bytes bound it, and where they are few what comes before the first of them: 8 rows by 28,672 features of 4,096 take 25.2
// us, 4.7 TB/s (26 with x quantised in front), 1 row by 2,560 of 2,048 some 5.  9 to 16 rows take it twice the products, which
// tell for large weights: 16 rows by 28,672 are left to linear8_mid.cu, by 4,096 not (8.8 us against 10).
#include "common.cuh"
#include "linear8.h"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, BLOCK = 128, GROUP = 2;  // GROUP: k-blocks that a warp asks for at once

__device__ __forceinline__ void mma_e4m3(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// weights are used once by this kernel: past L1
__device__ __forceinline__ uint4 load_weights(const unsigned char* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// GROUP k-blocks of 16 weight rows: rows g and g + 8, 32 bytes of each.
struct Weights {
    uint4 v[GROUP][4];
};

template <int NT, typename TO>
__global__ void __launch_bounds__(THREADS)
linear8_few_kernel(const linear8::Operands p, const int early) {
    extern __shared__ __align__(16) float red[];  // [2][WARPS][NT * 4][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tiles = (p.N + 15) / 16;
    const int groups = (p.kblocks + WARPS * GROUP - 1) / (WARPS * GROUP);  // of every warp and tile

    auto fetch = [&](Weights& w, int tile, int group) {
        const unsigned char* r0 = p.w + (size_t)min(tile * 16 + g, p.N - 1) * p.K;
        const unsigned char* r1 = p.w + (size_t)min(tile * 16 + g + 8, p.N - 1) * p.K;
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const int k = ((group * GROUP + u) * WARPS + warp) * BLOCK + 32 * t;
            const uint4 none = make_uint4(0u, 0u, 0u, 0u);
            w.v[u][0] = k < p.K ? load_weights(r0 + k) : none;
            w.v[u][1] = k < p.K ? load_weights(r1 + k) : none;
            w.v[u][2] = k + 16 < p.K ? load_weights(r0 + k + 16) : none;
            w.v[u][3] = k + 16 < p.K ? load_weights(r1 + k + 16) : none;
        }
    };

    Weights now, next;
    int tile = blockIdx.x, group = 0, turn = 0;
    if (early) fetch(now, tile, 0);
    pdl_wait();
    pdl_trigger();
    if (!early) fetch(now, tile, 0);

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

    while (tile < tiles) {
        const bool last = group == groups - 1;
        const int next_tile = last ? tile + gridDim.x : tile, next_group = last ? 0 : group + 1;
        if (next_tile < tiles) fetch(next, next_tile, next_group);
#pragma unroll
        for (int u = 0; u < GROUP; ++u) {
            const int kb = (group * GROUP + u) * WARPS + warp;
            if (kb >= p.kblocks) break;
            const int k = kb * BLOCK + 32 * t;
            const float sw = p.sw[(size_t)(tile >> 3) * p.kblocks + kb];
            const uint4 a0 = now.v[u][0], a1 = now.v[u][1], a2 = now.v[u][2], a3 = now.v[u][3];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const unsigned char* xr = p.x + (size_t)min(8 * i + g, p.M - 1) * p.K + k;
                const uint4 none = make_uint4(0u, 0u, 0u, 0u);
                const uint4 b0 = k < p.K ? *reinterpret_cast<const uint4*>(xr) : none;
                const uint4 b1 = k + 16 < p.K ? *reinterpret_cast<const uint4*>(xr + 16) : none;
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                mma_e4m3(c, a0.x, a1.x, a0.y, a1.y, b0.x, b0.y);
                mma_e4m3(c, a0.z, a1.z, a0.w, a1.w, b0.z, b0.w);
                mma_e4m3(c, a2.x, a3.x, a2.y, a3.y, b1.x, b1.y);
                mma_e4m3(c, a2.z, a3.z, a2.w, a3.w, b1.z, b1.w);
                const float s0 = sw * p.sx[(size_t)min(8 * i + 2 * t, p.M - 1) * p.sx_row + (size_t)kb * p.sx_block];
                const float s1 = sw * p.sx[(size_t)min(8 * i + 2 * t + 1, p.M - 1) * p.sx_row + (size_t)kb * p.sx_block];
                acc[i][0] = fmaf(c[0], s0, acc[i][0]);
                acc[i][1] = fmaf(c[1], s1, acc[i][1]);
                acc[i][2] = fmaf(c[2], s0, acc[i][2]);
                acc[i][3] = fmaf(c[3], s1, acc[i][3]);
            }
        }
        if (last) {
            // the warps' sums meet in shared memory (two copies in turn: one meeting a tile) and are added in the warps' order
            float* here = red + (size_t)(turn & 1) * WARPS * NT * 128;
            ++turn;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    here[(warp * NT * 4 + i * 4 + j) * 32 + lane] = acc[i][j];
                    acc[i][j] = 0.f;
                }
            __syncthreads();
            for (int e = threadIdx.x; e < 16 * 8 * NT; e += THREADS) {
                const int r = e & 15, m = e >> 4, n = tile * 16 + r;
                if (m >= p.M || n >= p.N) continue;
                // feature r, row m of the tile: accumulator j of lane (r & 7, (m & 7) / 2)
                const int from = ((m >> 3) * 4 + (r >> 3) * 2 + (m & 1)) * 32 + (r & 7) * 4 + ((m & 7) >> 1);
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += here[w * NT * 128 + from];
                reinterpret_cast<TO*>(p.out)[(size_t)m * p.ldo + n] = from_float<TO>(sum);
            }
        }
        now = next;
        tile = next_tile;
        group = next_group;
    }
}

template <int NT, typename TO>
int launch(const linear8::Operands& p, int early, cudaStream_t stream) {
    const int tiles = (p.N + 15) / 16, most = device_sms() * 2;
    return launch_pdl(linear8_few_kernel<NT, TO>, dim3(tiles < most ? tiles : most), dim3(THREADS), 2 * WARPS * NT * 128 * sizeof(float), stream, p, early);
}

}  // namespace

int linear8::few(const Operands& p, bool early, cudaStream_t stream) {
    if (p.out_dtype == LLM_F32) return p.M <= 8 ? launch<1, float>(p, early, stream) : launch<2, float>(p, early, stream);
    return p.M <= 8 ? launch<1, __nv_bfloat16>(p, early, stream) : launch<2, __nv_bfloat16>(p, early, stream);
}
