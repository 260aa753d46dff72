// y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k] for scales that are powers of two (as quantize_blocks makes
// them): tcgen05 takes them as they are, a byte of exponent for 32 k of a row (kind::mxf8f6f4), and sums over all of K in tensor memory.
//
// With scales of any value the sums leave tensor memory every 128 k (linear8_mid.cu, gemm8_tcgen05.cu), which takes an SM longer than
// the products.  Here nothing is done between the products but to write the scales into tensor memory: four warps, one for each
// quarter of the lanes, bring four k-blocks' at a time (a scale of 128 k is that of four times 32: the byte is repeated).  Roles, by warp:
//   warps 0, 1 : TMA producers, every other slot of a ring each; a slot is one k-block of both operands;
//   warp 2     : issues the products;
//   warps 4-7  : the scales, into a ring of GROUPS groups of four k-blocks;
//   warps 8 on : take the finished sums out of tensor memory.
// Every wait is bounded; one that gives up sets *error_flag and the roles run to their ends.
//
// The tensor cores' 32-bit sums truncate: 4,096 terms came out within 2.4e-6 of the terms' sizes, where
// sums in registers come within 2e-7; both are far below the 2^-4 of the numbers themselves.
//
// Some rows: the weights are the tall operand, 128 rows by up to 64 or 128 rows of x, and where there are few tiles a cluster of
// CTAs shares one's k-blocks and adds up in one another's shared memory.  Many rows: a pair of CTAs on tiles of 256 x 256.
// What it measured with x quantised in front: 4,096 x 28,672 x 4,096 357 us, 2,695 TFLOP/s, 0.43 us a k-block of a pair's tile, which
// takes the products 0.27 at the highest clock; 2,048 x 4,096 x 14,336 112 us; 256 x 4,096 x 4,096 15 us, of which some 7 are launches, first
// copies and the cluster's meeting.
#include "common.cuh"
#include "linear8.h"
#include "linear8_store.cuh"
#include "linear8_waits.cuh"
#include "tma.cuh"
#include "umma.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr int BM = 128, BK = 128, UMMA_K = 32, ISSUER = 2, FIRST_SCALES = 4, FIRST_EPI = 8;
constexpr int GROUP = 4, GROUPS = 4;     // k-blocks of a group of scales; groups in tensor memory
constexpr int SCALES_AT = 256;           // column of the first; the sums lie in front
constexpr int MAX_SPLIT = 4;

// A power of two's biased exponent, four times.
__device__ __forceinline__ unsigned exponents_of(float scale) { return (__float_as_uint(scale) >> 23 & 0xffu) * 0x01010101u; }

template <int BN, int STAGES, typename TO>
__global__ void __launch_bounds__(512, 1)
linear8_scaled_kernel(const linear8::Operands p, int split, int early, int* error_flag, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    constexpr int THREADS = 512, EPI_WARPS = THREADS / 32 - FIRST_EPI, COLS = BN / (EPI_WARPS / 4), PITCH = BM + 4;
    constexpr int A_BYTES = BM * BK, SLOT_BYTES = A_BYTES + BN * BK, NBUF = 2, XCOLS = BN / 32;
    constexpr int KB_COLS = 8;  // of a k-block's scales: 4 of the weights' rows, XCOLS of x's
    static_assert(GROUP * KB_COLS == 32, "a group is one store");
    static_assert(NBUF * BN <= SCALES_AT, "the sums lie in front of the scales");
    static_assert((size_t)BN * PITCH * 4 <= (size_t)STAGES * SLOT_BYTES, "the sums of a split tile lie where the ring was");
    constexpr unsigned IDESC = umma::idesc_e4m3_scaled(BM, BN);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full[NBUF], acc_empty[NBUF], drained;
    __shared__ __align__(8) unsigned long long scales_full[GROUPS], scales_empty[GROUPS];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up, asked[2];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = blockIdx.x % split, first_tile = blockIdx.x / split, tile_step = gridDim.x / split;
    const int col_tiles = (p.N + BM - 1) / BM, tiles = col_tiles * ((p.M + BN - 1) / BN);
    const int k_lo = p.kblocks * rank / split, k_hi = p.kblocks * (rank + 1) / split;

    if (threadIdx.x == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
            tma::mbar_init(&full[s], 1);
            tma::mbar_init(&empty[s], 1);
        }
#pragma unroll
        for (int b = 0; b < NBUF; ++b) {
            tma::mbar_init(&acc_full[b], 1);
            tma::mbar_init(&acc_empty[b], EPI_WARPS);
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            tma::mbar_init(&scales_full[g], 4);
            tma::mbar_init(&scales_empty[g], 1);
        }
        tma::mbar_init(&drained, 1);
        gave_up = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&xmap);
        tma::prefetch_map(&wmap);
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(&tmem_base)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if (warp >= ISSUER) {  // x and its scales come from the kernel before; the producers ask for weights first
        pdl_wait();
        pdl_trigger();
    }
    const linear8::Waits waits = {&gave_up, 0, error_flag};

    if (warp < ISSUER) {
        // ---- producers ----
        int it = 0, s = 0, turn = 0;
        bool ok = true;
        const int ahead = early ? min(STAGES, k_hi - k_lo) : 0;  // slots whose weights are asked for while x is still made
        if (umma::elect_one()) {
            for (int i = warp; i < ahead; i += 2) {
                tma::mbar_expect_tx(&full[i], SLOT_BYTES);
                tma::load_2d(ring + (size_t)i * SLOT_BYTES, &wmap, (k_lo + i) * BK, (first_tile % col_tiles) * BM, &full[i]);
            }
        }
        __syncwarp();
        pdl_wait();
        pdl_trigger();
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                if ((it & 1) == warp) {
                    if (it >= STAGES) ok = waits.there_untold(&empty[s], (turn - 1) & 1);
                    if (!ok) break;
                    unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                    if (umma::elect_one()) {
                        if (it >= ahead) {
                            tma::mbar_expect_tx(&full[s], SLOT_BYTES);
                            tma::load_2d(slot, &wmap, kb * BK, (tile % col_tiles) * BM, &full[s]);
                        }
                        tma::load_2d(slot + A_BYTES, &xmap, kb * BK, (tile / col_tiles) * BN, &full[s]);
                    }
                    __syncwarp();
                }
                if (++s == STAGES) s = 0, ++turn;
            }
        }
        if (lane == 0) asked[warp] = it;
    } else if (warp == ISSUER) {
        // ---- tensor-core issuer ----
        int s = 0, turn = 0, group = 0, round = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step, ++round) {
            const int buf = round % NBUF;
            if (round >= NBUF) ok = waits.there(&acc_empty[buf], (round / NBUF - 1) & 1);
            for (int kb = k_lo; kb < k_hi && ok; ++kb) {
                const int j = (kb - k_lo) % GROUP, g = group % GROUPS;
                const bool last = kb == k_hi - 1;
                ok = (j != 0 || waits.there(&scales_full[g], (group / GROUPS) & 1)) && waits.there(&full[s], turn & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                const unsigned long long a = umma::desc_sw128(slot), b = umma::desc_sw128(slot + A_BYTES);
                const unsigned d = tmem_base + buf * BN, scales = tmem_base + SCALES_AT + (g * GROUP + j) * KB_COLS;
                if (umma::elect_one()) {
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)  // 32 k = 32 bytes further along the rows: two 16-byte units
                        umma::mma_e4m3_scaled(d, a + 2 * k, b + 2 * k, IDESC, scales, scales + 4, kb != k_lo || k != 0);
                    umma::commit(&empty[s]);
                    if (j == GROUP - 1 || last) umma::commit(&scales_empty[g]);
                    if (last) umma::commit(&acc_full[buf]);
                }
                __syncwarp();
                if (j == GROUP - 1 || last) ++group;
                if (++s == STAGES) s = 0, ++turn;
            }
        }
        if (!ok) {  // nor for the products
            if (umma::elect_one()) umma::commit(&drained);
            (void)tma::mbar_wait(&drained, 0);
        }
    } else if (warp >= FIRST_SCALES && warp < FIRST_EPI) {
        // ---- scales: this warp's quarter of the lanes gets what the other quarters get ----
        const unsigned at = tmem_base + SCALES_AT + ((unsigned)((warp & 3) * 32) << 16);
        int group = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
            const float* sw = p.sw + (size_t)(tile % col_tiles) * p.kblocks;
            const float* sx[XCOLS];
#pragma unroll
            for (int c = 0; c < XCOLS; ++c) sx[c] = p.sx + (size_t)min((tile / col_tiles) * BN + 32 * c + lane, p.M - 1) * p.sx_row;
            float w[GROUP], x[GROUP][XCOLS];
            auto ask = [&](int k0) {
#pragma unroll
                for (int i = 0; i < GROUP; ++i) {
                    const int k = min(k0 + i, p.kblocks - 1);
                    w[i] = sw[k];
#pragma unroll
                    for (int c = 0; c < XCOLS; ++c) x[i][c] = sx[c][(size_t)k * p.sx_block];
                }
            };
            ask(k_lo);
            for (int k0 = k_lo; k0 < k_hi; k0 += GROUP, ++group) {
                unsigned r[GROUP * KB_COLS];
#pragma unroll
                for (int i = 0; i < GROUP; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        r[i * KB_COLS + c] = exponents_of(w[i]);
                        r[i * KB_COLS + 4 + c] = c < XCOLS ? exponents_of(x[i][c < XCOLS ? c : 0]) : 0u;
                    }
                if (k0 + GROUP < k_hi) ask(k0 + GROUP);
                const int g = group % GROUPS;
                ok = !waits.failed() && (group < GROUPS || waits.there(&scales_empty[g], (group / GROUPS - 1) & 1));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                umma::tmem_st32(at + g * GROUP * KB_COLS, r);
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) tma::mbar_arrive(&scales_full[g]);
            }
        }
    } else if (warp >= FIRST_EPI) {
        // ---- sums: rows (warp % 4) * 32 + lane of w, COLS rows of x from part * COLS on ----
        const int quarter = warp & 3, part = (warp - FIRST_EPI) >> 2;
        int round = 0;
        for (int tile = first_tile; tile < tiles; tile += tile_step, ++round) {
            const int n = (tile % col_tiles) * BM + quarter * 32 + lane, m_first = (tile / col_tiles) * BN + part * COLS, buf = round % NBUF;
            if (!waits.there(&acc_full[buf], (round / NBUF) & 1)) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            unsigned v[COLS / 32][32];
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) umma::tmem_ask32(tmem_base + buf * BN + part * COLS + 32 * c + ((unsigned)(quarter * 32) << 16), v[c]);
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) umma::tmem_have32(v[c]);
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&acc_empty[buf]);
            if (split == 1) {
                TO* out = reinterpret_cast<TO*>(p.out) + n;
#pragma unroll
                for (int j = 0; j < COLS; ++j)
                    if (n < p.N && m_first + j < p.M) out[(size_t)(m_first + j) * p.ldo] = from_float<TO>(__uint_as_float(v[j / 32][j % 32]));
            } else {
                // The ring's slots have all been read by the products (they were waited for); their memory takes the sums.
                float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int j = 0; j < COLS; ++j) sums[(part * COLS + j) * PITCH + quarter * 32 + lane] = __uint_as_float(v[j / 32][j % 32]);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    if (split > 1) cooperative_groups::this_cluster().sync(); else __syncthreads();
    if (warp < ISSUER && waits.failed()) {  // nobody waits for the copies on their way any more
        for (int i = max(0, asked[warp] - STAGES); i < asked[warp]; ++i)
            if ((i & 1) == warp) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(512) : "memory");
    }
    if (split > 1)
        linear8::join_cluster<BN, BM, THREADS, MAX_SPLIT, 2, TO>(p, reinterpret_cast<const float*>(ring), split, rank, 0, 1, (first_tile / col_tiles) * BN,
                                                                 (first_tile % col_tiles) * BM);
}

template <int BN, int STAGES, typename TO>
int launch(const linear8::Operands& p, int early, int* error_flag, cudaStream_t stream) {
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK + 1024;
    auto kernel = linear8_scaled_kernel<BN, STAGES, TO>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap xmap, wmap;
    if (!tma::make_map_2d_u8(&xmap, p.x, p.M, p.K, p.K, BN, BK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tma::make_map_2d_u8(&wmap, p.w, p.N, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B))
        return LLM_ERR_UNSUPPORTED;
    const long long tiles = (long long)((p.N + BM - 1) / BM) * ((p.M + BN - 1) / BN);
    if (tiles > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    const int sms = device_sms();
    int split = 1;  // doubled while all CTAs still run at once and none has fewer than four k-blocks
    while (split < MAX_SPLIT && tiles * split * 2 <= sms && p.kblocks >= 8 * split) split *= 2;
    return linear8::launch_clusters(kernel, (unsigned)(split > 1 ? tiles * split : tiles < sms ? tiles : sms), 512, smem, split, stream, p, split, early, error_flag, xmap, wmap);
}

// Many rows: a pair of CTAs (a cluster of two) on tiles of 256 rows of x by 256 of the weights.  Each CTA loads and keeps its 128 rows of x,
// half the tile's weights and its 128 rows of the result; the first CTA issues the products for both.  The sums take half of tensor
// memory and the scales the rest, so the next tile waits until the sums are in registers (some 300 cycles of a tile's 16,000).  Two pairs may
// share a tile's k-blocks; four did not pay (clusters of eight CTAs do not find room at once).
constexpr int PAIR_EPI_WARPS = 16, PAIR_THREADS = (FIRST_EPI + PAIR_EPI_WARPS) * 32;

template <int STAGES, typename TO>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
linear8_scaled_pair_kernel(const linear8::Operands p, int split, int early, int* error_flag, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    constexpr int BN = 256, A_BYTES = BM * BK, SLOT_BYTES = A_BYTES + BN / 2 * BK;  // of one CTA
    constexpr int COLS = BN / (PAIR_EPI_WARPS / 4);  // of an epilogue warp
    constexpr int KB_COLS = 16;                      // of a k-block's scales: 4 of the CTA's rows of x, 8 of the weights' rows, 4 unused
    constexpr int PITCH = BN + 4;
    static_assert((size_t)BM * PITCH * 4 <= (size_t)STAGES * SLOT_BYTES + PAIR_EPI_WARPS * linear8::PIECE_BYTES<TO>,
                  "a split tile's sums lie where ring and staging were");
    static_assert(BN <= SCALES_AT && SCALES_AT + GROUPS * GROUP * KB_COLS <= 512, "tensor memory");
    constexpr unsigned IDESC = umma::idesc_e4m3_scaled(2 * BM, BN);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* staging = ring + (size_t)STAGES * SLOT_BYTES;  // [PAIR_EPI_WARPS] pieces of the result
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full, acc_empty, scales_full[GROUPS], scales_empty[GROUPS], drained;
    __shared__ unsigned tmem_base;
    __shared__ int gave_up, asked[2];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // `split` pairs (1 or 2, a cluster) share a tile's k-blocks; the pair's first CTA has rank `leader` in the cluster
    const int place = blockIdx.x & 1, index = (blockIdx.x >> 1) % split, pair = (blockIdx.x >> 1) / split, pairs = (gridDim.x >> 1) / split;
    const unsigned leader = 2 * index;
    const int k_lo = p.kblocks * index / split, k_hi = p.kblocks * (index + 1) / split;
    const int row_tiles = (p.M + 2 * BM - 1) / (2 * BM), tiles = row_tiles * ((p.N + BN - 1) / BN);

    if (threadIdx.x == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
            tma::mbar_init(&full[s], 1);
            tma::mbar_init(&empty[s], 1);
        }
        tma::mbar_init(&acc_full, 1);
        tma::mbar_init(&acc_empty, 2 * PAIR_EPI_WARPS);  // the first CTA's is waited for, by both CTAs' warps
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            tma::mbar_init(&scales_full[g], 2 * 4);  // likewise
            tma::mbar_init(&scales_empty[g], 1);
        }
        tma::mbar_init(&drained, 1);
        gave_up = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&xmap);
        tma::prefetch_map(&wmap);
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(&tmem_base)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    cg::this_cluster().sync();  // both CTAs' barriers and tensor memory are there
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if (warp >= ISSUER) {  // x and its scales come from the kernel before; the producers ask for weights first
        pdl_wait();
        pdl_trigger();
    }
    const linear8::Waits waits = {&gave_up, 2 * split, error_flag};

    if (warp < ISSUER) {
        // ---- producers ----
        int it = 0, s = 0, turn = 0;
        bool ok = true;
        const int ahead = early ? min(STAGES, k_hi - k_lo) : 0;  // slots whose weights are asked for while x is still made
        if (umma::elect_one()) {
            for (int i = warp; i < ahead; i += 2) {
                if (place == 0) tma::mbar_expect_tx(&full[i], 2 * SLOT_BYTES);  // both CTAs' bytes
                tma::load_2d_pair(ring + (size_t)i * SLOT_BYTES + A_BYTES, &wmap, (k_lo + i) * BK, (pair / row_tiles) * BN + place * (BN / 2), &full[i]);
            }
        }
        __syncwarp();
        pdl_wait();
        pdl_trigger();
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int m0 = (tile % row_tiles) * 2 * BM + place * BM, n0 = (tile / row_tiles) * BN + place * (BN / 2);
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                if ((it & 1) == warp) {
                    if (it >= STAGES) ok = waits.there_untold(&empty[s], (turn - 1) & 1);
                    if (!ok) break;
                    unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                    if (umma::elect_one()) {
                        if (it >= ahead) {
                            if (place == 0) tma::mbar_expect_tx(&full[s], 2 * SLOT_BYTES);
                            tma::load_2d_pair(slot + A_BYTES, &wmap, kb * BK, n0, &full[s]);
                        }
                        tma::load_2d_pair(slot, &xmap, kb * BK, m0, &full[s]);
                    }
                    __syncwarp();
                }
                if (++s == STAGES) s = 0, ++turn;
            }
        }
        if (lane == 0) asked[warp] = it;
    } else if (warp == ISSUER) {
        // ---- tensor-core issuer, for both CTAs ----
        if (place == 0) {
            int s = 0, turn = 0, group = 0, round = 0;
            bool ok = true;
            for (int tile = pair; tile < tiles && ok; tile += pairs, ++round) {
                if (round > 0) ok = waits.there(&acc_empty, (round - 1) & 1);
                for (int kb = k_lo; kb < k_hi && ok; ++kb) {
                    const int j = (kb - k_lo) % GROUP, g = group % GROUPS;
                    const bool last = kb == k_hi - 1;
                    ok = (j != 0 || waits.there(&scales_full[g], (group / GROUPS) & 1)) && waits.there(&full[s], turn & 1);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                    const unsigned long long a = umma::desc_sw128(slot), b = umma::desc_sw128(slot + A_BYTES);
                    const unsigned scales = tmem_base + SCALES_AT + (g * GROUP + j) * KB_COLS;
                    if (umma::elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)  // 32 k = 32 bytes further along the rows: two 16-byte units
                            umma::mma_e4m3_scaled_pair(tmem_base, a + 2 * k, b + 2 * k, IDESC, scales, scales + 4, kb != k_lo || k != 0);
                        umma::commit_pair(&empty[s], leader);
                        if (j == GROUP - 1 || last) umma::commit_pair(&scales_empty[g], leader);
                        if (last) umma::commit_pair(&acc_full, leader);
                    }
                    __syncwarp();
                    if (j == GROUP - 1 || last) ++group;
                    if (++s == STAGES) s = 0, ++turn;
                }
            }
            if (!ok) {  // nor for the products
                if (umma::elect_one()) umma::commit_pair(&drained, leader);
                (void)tma::mbar_wait(&drained, 0);
            }
        }
    } else if (warp >= FIRST_SCALES && warp < FIRST_EPI) {
        // ---- scales: this warp's quarter of the lanes gets what the other quarters get ----
        const unsigned at = tmem_base + SCALES_AT + ((unsigned)((warp & 3) * 32) << 16);
        const int last_block = (p.N + 127) / 128 - 1;
        int group = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int block = (tile / row_tiles) * (BN / 128);
            const float *sw0 = p.sw + (size_t)block * p.kblocks, *sw1 = p.sw + (size_t)min(block + 1, last_block) * p.kblocks;
            const float* sx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) sx[c] = p.sx + (size_t)min((tile % row_tiles) * 2 * BM + place * BM + 32 * c + lane, p.M - 1) * p.sx_row;
            float w[GROUP][2], x[GROUP][4];
            auto ask = [&](int k0) {
#pragma unroll
                for (int i = 0; i < GROUP; ++i) {
                    const int k = min(k0 + i, p.kblocks - 1);
                    w[i][0] = sw0[k], w[i][1] = sw1[k];
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[i][c] = sx[c][(size_t)k * p.sx_block];
                }
            };
            ask(k_lo);
            for (int k0 = k_lo; k0 < k_hi; k0 += GROUP, ++group) {
                const int g = group % GROUPS;
                ok = !waits.failed() && (group < GROUPS || waits.there(&scales_empty[g], (group / GROUPS - 1) & 1));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    unsigned r[2 * KB_COLS];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            r[i * KB_COLS + c] = exponents_of(x[2 * half + i][c]);
                            r[i * KB_COLS + 4 + c] = exponents_of(w[2 * half + i][0]);
                            r[i * KB_COLS + 8 + c] = exponents_of(w[2 * half + i][1]);
                            r[i * KB_COLS + 12 + c] = 0u;
                        }
                    umma::tmem_st32(at + (g * GROUP + 2 * half) * KB_COLS, r);
                }
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) tma::mbar_arrive_at(&scales_full[g], leader);
                if (k0 + GROUP < k_hi) ask(k0 + GROUP);
            }
        }
    } else if (warp >= FIRST_EPI) {
        // ---- sums: rows (warp % 4) * 32 + lane of x, COLS columns ----
        const int quarter = warp & 3, part = (warp - FIRST_EPI) >> 2;
        int round = 0;
        for (int tile = pair; tile < tiles; tile += pairs, ++round) {
            const int m0 = (tile % row_tiles) * 2 * BM + place * BM, n0 = (tile / row_tiles) * BN + part * COLS;
            if (!waits.there(&acc_full, round & 1)) break;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            unsigned v[COLS / 32][32];
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) umma::tmem_ask32(tmem_base + part * COLS + 32 * c + ((unsigned)(quarter * 32) << 16), v[c]);
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) umma::tmem_have32(v[c]);
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tma::mbar_arrive_at(&acc_empty, leader);
            if (split > 1) {
                // The ring's slots have all been read by the products (they were waited for); its memory takes the sums.
                float* sums = reinterpret_cast<float*>(ring) + (quarter * 32 + lane) * PITCH + part * COLS;
#pragma unroll
                for (int j = 0; j < COLS; j += 4)
                    *reinterpret_cast<uint4*>(sums + j) = make_uint4(v[j / 32][j % 32], v[j / 32][j % 32 + 1], v[j / 32][j % 32 + 2], v[j / 32][j % 32 + 3]);
                continue;
            }
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
                unsigned long long sums[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[j] = umma::pair_of(v[c][2 * j], v[c][2 * j + 1]);
                if (n0 + 32 * c < p.N) linear8::store_piece<TO>(p, staging + (size_t)(warp - FIRST_EPI) * linear8::PIECE_BYTES<TO>, sums, m0 + quarter * 32, n0 + 32 * c, lane);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    cg::this_cluster().sync();  // neither leaves while the other reads its memory or arrives at its barriers
    if (waits.failed()) {  // (the whole cluster knows.)  Nobody waits for the copies on their way any more, which are counted at the first CTA
        if (place == 0 && warp < ISSUER) {
            for (int i = max(0, asked[warp] - STAGES); i < asked[warp]; ++i)
                if ((i & 1) == warp) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
        }
        cg::this_cluster().sync();
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(512) : "memory");
    }
    if (split > 1)
        linear8::join_cluster<BM, BN, PAIR_THREADS, 2, 3, TO>(p, reinterpret_cast<const float*>(ring), split, index, place, 2, (pair % row_tiles) * 2 * BM + place * BM,
                                                                      (pair / row_tiles) * BN);
}

template <typename TO>
int launch_pair(const linear8::Operands& p, int split, int early, int* error_flag, cudaStream_t stream) {
    constexpr int STAGES = sizeof(TO) == 4 ? 4 : 5;
    constexpr size_t smem = (size_t)STAGES * 2 * BM * BK + 1024 + PAIR_EPI_WARPS * linear8::PIECE_BYTES<TO>;
    auto kernel = linear8_scaled_pair_kernel<STAGES, TO>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap xmap, wmap;
    if (!tma::make_map_2d_u8(&xmap, p.x, p.M, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tma::make_map_2d_u8(&wmap, p.w, p.N, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B))
        return LLM_ERR_UNSUPPORTED;
    const long long tiles = (long long)((p.N + 255) / 256) * ((p.M + 255) / 256);
    if (tiles > 0x3fffffffLL) return LLM_ERR_UNSUPPORTED;
    const int pairs = device_sms() / 2;
    return linear8::launch_clusters(kernel, (unsigned)(split > 1 ? tiles * split : tiles < pairs ? tiles : pairs) * 2, PAIR_THREADS, smem, 2 * split, stream, p, split, early,
                                    error_flag, xmap, wmap);
}

}  // namespace

int linear8::some_scaled(const Operands& p, bool early, int* error_flag, cudaStream_t stream) {
    if (p.out_dtype == LLM_F32) return p.M <= 64 ? launch<64, 7, float>(p, early, error_flag, stream) : launch<128, 6, float>(p, early, error_flag, stream);
    return p.M <= 64 ? launch<64, 7, __nv_bfloat16>(p, early, error_flag, stream) : launch<128, 6, __nv_bfloat16>(p, early, error_flag, stream);
}

int linear8::many_scaled(const Operands& p, int split, bool early, int* error_flag, cudaStream_t stream) {
    return p.out_dtype == LLM_F32 ? launch_pair<float>(p, split, early, error_flag, stream) : launch_pair<__nv_bfloat16>(p, split, early, error_flag, stream);
}
