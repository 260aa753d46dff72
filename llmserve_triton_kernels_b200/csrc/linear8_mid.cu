// y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k] for some rows of x, on tcgen05 with the weights as the tall
// operand: a tile is 128 rows of w by up to 64 or 128 rows of x, so that no tile is mostly padding.
//
// Roles, rings and accumulators are those of gemm8_tcgen05.cu (a slot is one 128-byte k-block of both operands, its four products
// start from zero, the sums live in registers).  What differs: a thread of the sums holds one row of w and 32 of x's rows, whose
// scales differ from column to column; they come through a few bytes of shared memory of the warp's own, 16 bytes a read for everyone.
// Where there are fewer tiles than SMs, `split` CTAs (a cluster) share a tile's k-blocks and add up in one another's shared memory.
//
// What bounds it: a k-block of 64 rows takes the sums' warps some 600 cycles (16 KB of weights in 0.33 us, 7.5 TB/s over all SMs), of 128
// 850; and around them some 6 us of a launch, of first copies, and of the cluster's meeting and adding.  With x quantised in front 33 rows by
// 32,000 features of 2,048 take 20 us (250 tiles, two rounds), 32 rows by 4,096 of 14,336 16.9, by 4,096 of 4,096 9.8.
#include "common.cuh"
#include "linear8.h"
#include "linear8_store.cuh"
#include "linear8_waits.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace {

constexpr int BM = 128, BK = 128, UMMA_K = 32, FIRST_EPI = 4, FIRST_ISSUER = 2, NBUF = 4, MAX_SPLIT = 4;

template <int BN, int STAGES, int EPI_WARPS, typename TO>
__global__ void __launch_bounds__((FIRST_EPI + EPI_WARPS) * 32, 1)
linear8_mid_kernel(const linear8::Operands p, int split, int early, int* error_flag, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    constexpr int A_BYTES = BM * BK, SLOT_BYTES = A_BYTES + BN * BK, COLS = BN / (EPI_WARPS / 4), PITCH = BM + 4;
    constexpr int TMEM_COLS = NBUF * BN, THREADS = (FIRST_EPI + EPI_WARPS) * 32;
    static_assert(TMEM_COLS == 256 || TMEM_COLS == 512, "columns of tensor memory come in powers of two");
    static_assert((size_t)BN * PITCH * 4 <= (size_t)STAGES * SLOT_BYTES, "the sums of a split tile lie where the ring was");
    constexpr unsigned IDESC = umma::idesc_e4m3(BM, BN);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full[NBUF], acc_empty[NBUF], drained[2];
    __shared__ __align__(16) float scales[EPI_WARPS][2][COLS];
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
        tma::mbar_init(&drained[0], 1);
        tma::mbar_init(&drained[1], 1);
        gave_up = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&xmap);
        tma::prefetch_map(&wmap);
    }
    if (warp == FIRST_ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(&tmem_base)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if (warp >= FIRST_ISSUER) {  // x and its scales come from the kernel before; the producers ask for weights first
        pdl_wait();
        pdl_trigger();
    }

    const linear8::Waits waits = {&gave_up, 0, error_flag};

    const int which = warp & 1;  // of the two producers or issuers: its k-blocks are every other one
    if (warp < FIRST_ISSUER) {
        // ---- producers ----
        int it = 0, s = 0, turn = 0;
        bool ok = true;
        const int ahead = early ? min(STAGES, k_hi - k_lo) : 0;  // slots whose weights are asked for while x is still made
        if (umma::elect_one()) {
            for (int i = which; i < ahead; i += 2) {
                tma::mbar_expect_tx(&full[i], SLOT_BYTES);
                tma::load_2d(ring + (size_t)i * SLOT_BYTES, &wmap, (k_lo + i) * BK, (first_tile % col_tiles) * BM, &full[i]);
            }
        }
        __syncwarp();
        pdl_wait();
        pdl_trigger();
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                if ((it & 1) == which) {
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
        if (lane == 0) asked[which] = it;
    } else if (warp < FIRST_EPI) {
        // ---- tensor-core issuers ----
        int it = 0, s = 0, turn = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
            for (int kb = k_lo; kb < k_hi; ++kb, ++it) {
                if ((it & 1) == which) {
                    const int buf = it % NBUF;
                    ok = waits.there(&full[s], turn & 1) && (it < NBUF || waits.there(&acc_empty[buf], ((it / NBUF) - 1) & 1));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                    const unsigned long long a = umma::desc_sw128(slot), b = umma::desc_sw128(slot + A_BYTES);
                    const unsigned d = tmem_base + buf * BN;
                    if (umma::elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k) umma::mma_e4m3(d, a + 2 * k, b + 2 * k, IDESC, k != 0);
                        umma::commit(&empty[s]);
                        umma::commit(&acc_full[buf]);
                    }
                    __syncwarp();
                }
                if (++s == STAGES) s = 0, ++turn;
            }
        }
        if (!ok) {  // nor for the products
            if (umma::elect_one()) umma::commit(&drained[which]);
            (void)tma::mbar_wait(&drained[which], 0);
        }
    } else if (warp >= FIRST_EPI) {
        // ---- sums: rows (warp % 4) * 32 + lane of w, COLS rows of x from part * COLS on ----
        const int quarter = warp & 3, part = (warp - FIRST_EPI) >> 2;
        float(&mine)[2][COLS] = scales[warp - FIRST_EPI];
        int it = 0;
        bool ok = true;
        for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
            const int n = (tile % col_tiles) * BM + quarter * 32 + lane, m_first = (tile / col_tiles) * BN + part * COLS;
            const float* sw = p.sw + (size_t)(tile % col_tiles) * p.kblocks;
            unsigned long long acc[COLS / 2];
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
            // this lane's columns' scales, four k-blocks ahead
            const float* sx[COLS / 32];
#pragma unroll
            for (int u = 0; u < COLS / 32; ++u) sx[u] = p.sx + (size_t)min(m_first + 32 * u + lane, p.M - 1) * p.sx_row;
            float ahead[4][COLS / 32];
            auto ask = [&](int i, int kb) {
                const int k = min(kb, p.kblocks - 1);
                const float w = sw[k];
#pragma unroll
                for (int u = 0; u < COLS / 32; ++u) ahead[i][u] = sx[u][(size_t)k * p.sx_block] * w;
            };
#pragma unroll
            for (int i = 0; i < 4; ++i) ask(i, k_lo + i);
            for (int k0 = k_lo; k0 < k_hi && ok; k0 += 4) {
                float now[4][COLS / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int u = 0; u < COLS / 32; ++u) now[i][u] = ahead[i][u];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) ask(i, k0 + 4 + i);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (k0 + i >= k_hi) break;
                    const int buf = it % NBUF;
#pragma unroll
                    for (int u = 0; u < COLS / 32; ++u) mine[i & 1][32 * u + lane] = now[i][u];
                    ok = waits.there_untold(&acc_full[buf], (it / NBUF) & 1);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const unsigned base = tmem_base + buf * BN + part * COLS + ((unsigned)(quarter * 32) << 16);
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        unsigned v[32];
                        umma::tmem_ask32(base + c, v);
                        umma::tmem_have32(v);
                        if (c + 32 == COLS) {  // this warp has read its part: the accumulator may be filled again
                            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                            __syncwarp();
                            if (lane == 0) tma::mbar_arrive(&acc_empty[buf]);
                        }
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&mine[i & 1][c + j]);
                            asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(acc[(c + j) / 2]) : "l"(umma::pair_of(v[j], v[j + 1])), "l"(s.x));
                            asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(acc[(c + j) / 2 + 1]) : "l"(umma::pair_of(v[j + 2], v[j + 3])), "l"(s.y));
                        }
                    }
                    ++it;
                }
            }
            if (split == 1) {
                if (ok && n < p.N) {
                    TO* out = reinterpret_cast<TO*>(p.out) + n;
#pragma unroll
                    for (int j = 0; j < COLS; ++j) {
                        const float y = __uint_as_float((unsigned)(acc[j / 2] >> (32 * (j & 1))));
                        if (m_first + j < p.M) out[(size_t)(m_first + j) * p.ldo] = from_float<TO>(y);
                    }
                }
            } else {
                // The ring's slots have all been read by the products (they were waited for); their memory takes the sums.
                float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int j = 0; j < COLS; ++j) sums[(part * COLS + j) * PITCH + quarter * 32 + lane] = __uint_as_float((unsigned)(acc[j / 2] >> (32 * (j & 1))));
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    if (split > 1) cooperative_groups::this_cluster().sync(); else __syncthreads();
    if (warp < FIRST_ISSUER && waits.failed()) {  // nobody waits for the copies on their way any more
        for (int i = max(0, asked[warp] - STAGES); i < asked[warp]; ++i)
            if ((i & 1) == warp) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
    }
    if (warp == FIRST_ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
    if (split > 1)
        linear8::join_cluster<BN, BM, THREADS, MAX_SPLIT, 2, TO>(p, reinterpret_cast<const float*>(ring), split, rank, 0, 1, (first_tile / col_tiles) * BN,
                                                                 (first_tile % col_tiles) * BM);
}

template <int BN, int STAGES, int EPI_WARPS, typename TO>
int launch(const linear8::Operands& p, int early, int* error_flag, cudaStream_t stream) {
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK + 1024;
    auto kernel = linear8_mid_kernel<BN, STAGES, EPI_WARPS, TO>;
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
    return linear8::launch_clusters(kernel, (unsigned)(split > 1 ? tiles * split : tiles < sms ? tiles : sms), (FIRST_EPI + EPI_WARPS) * 32, smem,
                                    split, stream, p, split, early, error_flag, xmap, wmap);
}

}  // namespace

int linear8::some(const Operands& p, bool early, int* error_flag, cudaStream_t stream) {
    if (p.out_dtype == LLM_F32) return p.M <= 64 ? launch<64, 7, 8, float>(p, early, error_flag, stream) : launch<128, 6, 16, float>(p, early, error_flag, stream);
    return p.M <= 64 ? launch<64, 7, 8, __nv_bfloat16>(p, early, error_flag, stream) : launch<128, 6, 16, __nv_bfloat16>(p, early, error_flag, stream);
}
