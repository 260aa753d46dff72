// y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k] for many rows: x and w in e4m3, a scale for every 128 k,
// on tcgen05 (kind::f8f6f4) with TMA-fed tiles.
//
// A k-block is a block of the scales: 128 bytes of a row, which is also the swizzle's width, so a slot of the ring holds one
// k-block of both operands.  Its four products (K = 32 each) start from zero in tensor memory and leave it at once: the epilogue
// warps add them to 32-bit sums in registers, times sx of their row and sw of their columns.  Scales of any value are allowed
// that way, and no sum is longer than 128 terms before it is rounded to 32 bits.  Roles, by warp:
//   warps 0, 1 : TMA producers, every other slot of a ring of STAGES each;
//   warps 2, 3 : issue the products, every other k-block each, into one of NBUF accumulators of tensor memory, in turn;
//   warps 4-19 : the sums.  A warp owns its 32 rows (lanes) and a quarter of the tile's columns, two columns to an instruction
//                (fma.rn.f32x2).  The sums and 32 columns on their way need more registers than 640 threads are launched with: the
//                first four warps give theirs up.
// The sums are what bounds it: what a warp does for a k-block of 32 columns (wait, read tensor memory, 16 instructions of sums, give
// the accumulator back) takes it some 500 cycles beside three others on its quarter of the SM, the products 512 for a 256 x 256 tile of
// a pair.  The roles that issue were the bound before they were two warps each: a k-block's waits, products and commits take one
// warp 600 cycles (533 us for 4,096 x 28,672 x 4,096 with one, 459 with two: 2,096 TFLOP/s with x quantised in front).  Scales are read
// where rows lie side by side (linear8.h): from [rows, blocks] the same product took 100 us more.
// One CTA per SM walks 128 x 128 tiles, or a pair of CTAs 256 x 256, column tiles outermost, so that CTAs that run at the same time share
// their weights.  What lies beyond the matrices arrives as zeros and is masked at the store.  Every wait is bounded; one that gives up
// sets *error_flag and the roles run to their ends.
#include "common.cuh"
#include "linear8.h"
#include "linear8_store.cuh"
#include "linear8_waits.cuh"
#include "tma.cuh"
#include "umma.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr int BM = 128, BK = 128, UMMA_K = 32, EPI_WARPS = 16, FIRST_EPI = 4, FIRST_ISSUER = 2;
constexpr int THREADS = (FIRST_EPI + EPI_WARPS) * 32;
// 640 threads are launched with 96 registers each: 5 x 96 = 32 + 4 x 112
constexpr int FEW_REGISTERS = 32, MANY_REGISTERS = 112;

// sums += columns * scale, 32 columns as 16 pairs.
__device__ __forceinline__ void add_columns(unsigned long long* sums, const unsigned (&v)[32], unsigned long long scale) {
#pragma unroll
    for (int j = 0; j < 16; ++j) asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(sums[j]) : "l"(umma::pair_of(v[2 * j], v[2 * j + 1])), "l"(scale));
}

template <int STAGES, typename TO>
__global__ void __launch_bounds__(THREADS, 1)
gemm8_tcgen05_kernel(const linear8::Operands p, int early, int* error_flag, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    constexpr int BN = 128, A_BYTES = BM * BK, SLOT_BYTES = A_BYTES + BN * BK;
    constexpr int NBUF = 4, TMEM_COLS = NBUF * BN;
    static_assert(TMEM_COLS == 512, "all columns of tensor memory");
    constexpr int COLS = BN / (EPI_WARPS / 4);  // of an epilogue warp
    constexpr unsigned IDESC = umma::idesc_e4m3(BM, BN);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* staging = ring + (size_t)STAGES * SLOT_BYTES;  // [EPI_WARPS] pieces of the result
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full[NBUF], acc_empty[NBUF], drained[2];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up, asked[2];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int kblocks = p.kblocks;
    const int row_tiles = (p.M + BM - 1) / BM, col_tiles = (p.N + BN - 1) / BN, tiles = row_tiles * col_tiles;

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

    // (each role's share of the registers is set where the role begins: what follows a smaller share is compiled for it)
    if (warp >= FIRST_EPI) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(MANY_REGISTERS));
        // ---- sums: warp w may touch the 32 lanes (warp % 4) * 32 .. of tensor memory ----
        const int quarter = warp & 3, part = (warp - FIRST_EPI) >> 2;
        int it = 0;
        bool ok = true;
        auto release = [&](int buf) {  // this warp has read its part: the accumulator may be filled again
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&acc_empty[buf]);
        };
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            const int m0 = (tile % row_tiles) * BM, n0 = (tile / row_tiles) * BN + part * COLS;
            const float* sx = p.sx + (size_t)min(m0 + quarter * 32 + lane, p.M - 1) * p.sx_row;
            const float* sw = p.sw + (size_t)(min(n0, p.N - 1) >> 7) * kblocks;  // the warp's columns lie in one block of 128
            unsigned long long acc[COLS / 2];  // two 32-bit sums each
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
            // the scales of four k-blocks are asked for four k-blocks ahead
            float sx_now[4], sw_now[4], sx_next[4], sw_next[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sx_next[i] = sx[(size_t)min(i, kblocks - 1) * p.sx_block], sw_next[i] = sw[min(i, kblocks - 1)];
            for (int k0 = 0; k0 < kblocks && ok; k0 += 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sx_now[i] = sx_next[i], sw_now[i] = sw_next[i];
                    sx_next[i] = sx[(size_t)min(k0 + 4 + i, kblocks - 1) * p.sx_block], sw_next[i] = sw[min(k0 + 4 + i, kblocks - 1)];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (k0 + i >= kblocks) break;
                    const int buf = it % NBUF;
                    const float scale = sx_now[i] * sw_now[i];
                    ok = waits.there_untold(&acc_full[buf], (it / NBUF) & 1);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const unsigned base = tmem_base + buf * BN + part * COLS + ((unsigned)(quarter * 32) << 16);
                    const unsigned long long both = umma::pair_of(__float_as_uint(scale), __float_as_uint(scale));
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        unsigned v[32];
                        umma::tmem_ask32(base + c, v);
                        umma::tmem_have32(v);
                        if (c + 32 == COLS) release(buf);
                        add_columns(acc + c / 2, v, both);
                    }
                    ++it;
                }
            }
            if (ok) {
#pragma unroll
                for (int c = 0; c < COLS; c += 32) {
                    if (n0 + c < p.N) linear8::store_piece<TO>(p, staging + (size_t)(warp - FIRST_EPI) * linear8::PIECE_BYTES<TO>, acc + c / 2, m0 + quarter * 32, n0 + c, lane);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(FEW_REGISTERS));
        const int which = warp & 1;  // of the two producers or issuers: its k-blocks are every other one
        if (warp < FIRST_ISSUER) {
            // ---- producers ----
            int it = 0, s = 0, turn = 0;
            bool ok = true;
            const int ahead = early ? min(STAGES, kblocks) : 0;  // slots whose weights are asked for while x is still made
            if (umma::elect_one()) {
                for (int i = which; i < ahead; i += 2) {
                    tma::mbar_expect_tx(&full[i], SLOT_BYTES);
                    tma::load_2d(ring + (size_t)i * SLOT_BYTES + A_BYTES, &wmap, i * BK, ((int)blockIdx.x / row_tiles) * BN, &full[i]);
                }
            }
            __syncwarp();
            pdl_wait();
            pdl_trigger();
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int m0 = (tile % row_tiles) * BM, n0 = (tile / row_tiles) * BN;
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
                    if ((it & 1) == which) {
                        if (it >= STAGES) ok = waits.there_untold(&empty[s], (turn - 1) & 1);
                        if (!ok) break;
                        unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                        if (umma::elect_one()) {
                            if (it >= ahead) {
                                tma::mbar_expect_tx(&full[s], SLOT_BYTES);
                                tma::load_2d(slot + A_BYTES, &wmap, kb * BK, n0, &full[s]);
                            }
                            tma::load_2d(slot, &xmap, kb * BK, m0, &full[s]);
                        }
                        __syncwarp();
                    }
                    if (++s == STAGES) s = 0, ++turn;
                }
            }
            if (lane == 0) asked[which] = it;
        } else {
            // ---- tensor-core issuers ----
            int it = 0, s = 0, turn = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
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
                            for (int k = 0; k < BK / UMMA_K; ++k)  // 32 k = 32 bytes further along the rows: two 16-byte units
                                umma::mma_e4m3(d, a + 2 * k, b + 2 * k, IDESC, k != 0);
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
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp < FIRST_ISSUER && waits.failed()) {  // nobody waits for the copies on their way any more
        for (int i = max(0, asked[warp] - STAGES); i < asked[warp]; ++i)
            if ((i & 1) == warp) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
    }
    if (warp == FIRST_ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
}

// The same by a pair of CTAs (a cluster of two) on tiles of 256 x 256: each CTA loads and keeps its 128 rows of x, half the tile's rows of w and
// its 128 rows of the result; the first CTA issues the products for both.  A single CTA's 128 x 256 tile needs 48 KB a k-block, which
// the way from L2 to an SM does not bring in the products' time; a pair's needs 32 KB an SM.
template <int STAGES, typename TO>
__global__ void __launch_bounds__(THREADS, 1)
gemm8_pair_kernel(const linear8::Operands p, int early, int* error_flag, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    constexpr int BN = 256, A_BYTES = BM * BK, SLOT_BYTES = A_BYTES + BN / 2 * BK;  // of one CTA
    constexpr int NBUF = 2, TMEM_COLS = NBUF * BN;
    constexpr int COLS = BN / (EPI_WARPS / 4);  // of an epilogue warp
    constexpr unsigned IDESC = umma::idesc_e4m3(2 * BM, BN);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* staging = ring + (size_t)STAGES * SLOT_BYTES;  // [EPI_WARPS] pieces of the result
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full[NBUF], acc_empty[NBUF], drained[2];
    __shared__ unsigned tmem_base;
    __shared__ int gave_up, asked[2];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int kblocks = p.kblocks;
    const int place = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int row_tiles = (p.M + 2 * BM - 1) / (2 * BM), col_tiles = (p.N + BN - 1) / BN, tiles = row_tiles * col_tiles;

    if (threadIdx.x == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
            tma::mbar_init(&full[s], 1);
            tma::mbar_init(&empty[s], 1);
        }
#pragma unroll
        for (int b = 0; b < NBUF; ++b) {
            tma::mbar_init(&acc_full[b], 1);
            tma::mbar_init(&acc_empty[b], 2 * EPI_WARPS);  // the first CTA's is waited for, by both CTAs' warps
        }
        tma::mbar_init(&drained[0], 1);
        tma::mbar_init(&drained[1], 1);
        gave_up = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&xmap);
        tma::prefetch_map(&wmap);
    }
    if (warp == FIRST_ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(&tmem_base)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    cg::this_cluster().sync();  // both CTAs' barriers and tensor memory are there
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if (warp >= FIRST_ISSUER) {  // x and its scales come from the kernel before; the producers ask for weights first
        pdl_wait();
        pdl_trigger();
    }

    const linear8::Waits waits = {&gave_up, 2, error_flag};

    // (each role's share of the registers is set where the role begins: what follows a smaller share is compiled for it)
    if (warp >= FIRST_EPI) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(MANY_REGISTERS));
        // ---- sums: warp w may touch the 32 lanes (warp % 4) * 32 .. of tensor memory ----
        const int quarter = warp & 3, part = (warp - FIRST_EPI) >> 2;
        int it = 0;
        bool ok = true;
        auto release = [&](int buf) {  // this warp has read its part: the accumulator may be filled again
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tma::mbar_arrive_at(&acc_empty[buf], 0);
        };
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            const int m0 = (tile % row_tiles) * 2 * BM + place * BM, n0 = (tile / row_tiles) * BN + part * COLS;
            const float* sx = p.sx + (size_t)min(m0 + quarter * 32 + lane, p.M - 1) * p.sx_row;
            const float* sw = p.sw + (size_t)(min(n0, p.N - 1) >> 7) * kblocks;  // the warp's columns lie in one block of 128
            unsigned long long acc[COLS / 2];  // two 32-bit sums each
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
            // the scales of four k-blocks are asked for four k-blocks ahead
            float sx_now[4], sw_now[4], sx_next[4], sw_next[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sx_next[i] = sx[(size_t)min(i, kblocks - 1) * p.sx_block], sw_next[i] = sw[min(i, kblocks - 1)];
            for (int k0 = 0; k0 < kblocks && ok; k0 += 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sx_now[i] = sx_next[i], sw_now[i] = sw_next[i];
                    sx_next[i] = sx[(size_t)min(k0 + 4 + i, kblocks - 1) * p.sx_block], sw_next[i] = sw[min(k0 + 4 + i, kblocks - 1)];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (k0 + i >= kblocks) break;
                    const int buf = it % NBUF;
                    const float scale = sx_now[i] * sw_now[i];
                    // (waits.there_untold here and in the producers takes 4,096 x 28,672 x 4,096 from 461 us to 492: fail() in the middle of the loop)
                    ok = __all_sync(0xffffffffu, !waits.flag() && tma::mbar_wait(&acc_full[buf], (it / NBUF) & 1));
                    if (!ok) {
                        if (lane == 0) waits.fail();
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const unsigned base = tmem_base + buf * BN + part * COLS + ((unsigned)(quarter * 32) << 16);
                    const unsigned long long both = umma::pair_of(__float_as_uint(scale), __float_as_uint(scale));
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        unsigned v[32];
                        umma::tmem_ask32(base + c, v);
                        umma::tmem_have32(v);
                        if (c + 32 == COLS) release(buf);
                        add_columns(acc + c / 2, v, both);
                    }
                    ++it;
                }
            }
            if (ok) {
#pragma unroll
                for (int c = 0; c < COLS; c += 32) {
                    if (n0 + c < p.N) linear8::store_piece<TO>(p, staging + (size_t)(warp - FIRST_EPI) * linear8::PIECE_BYTES<TO>, acc + c / 2, m0 + quarter * 32, n0 + c, lane);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(FEW_REGISTERS));
        const int which = warp & 1;  // of the two producers or issuers: its k-blocks are every other one
        if (warp < FIRST_ISSUER) {
            // ---- producers ----
            int it = 0, s = 0, turn = 0;
            bool ok = true;
            const int ahead = early ? min(STAGES, kblocks) : 0;  // slots whose weights are asked for while x is still made
            if (umma::elect_one()) {
                for (int i = which; i < ahead; i += 2) {
                    if (place == 0) tma::mbar_expect_tx(&full[i], 2 * SLOT_BYTES);  // both CTAs' bytes
                    tma::load_2d_pair(ring + (size_t)i * SLOT_BYTES + A_BYTES, &wmap, i * BK, (pair / row_tiles) * BN + place * (BN / 2), &full[i]);
                }
            }
            __syncwarp();
            pdl_wait();
            pdl_trigger();
            for (int tile = pair; tile < tiles && ok; tile += pairs) {
                const int m0 = (tile % row_tiles) * 2 * BM + place * BM, n0 = (tile / row_tiles) * BN + place * (BN / 2);
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
                    if ((it & 1) == which) {
                        if (it >= STAGES) ok = waits.there(&empty[s], (turn - 1) & 1) && !waits.failed();
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
            if (lane == 0) asked[which] = it;
        } else if (place == 0) {
            // ---- tensor-core issuers, for both CTAs ----
            int it = 0, s = 0, turn = 0;
            bool ok = true;
            for (int tile = pair; tile < tiles && ok; tile += pairs) {
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
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
                            for (int k = 0; k < BK / UMMA_K; ++k)  // 32 k = 32 bytes further along the rows: two 16-byte units
                                umma::mma_e4m3_pair(d, a + 2 * k, b + 2 * k, IDESC, k != 0);
                            umma::commit_pair(&empty[s]);
                            umma::commit_pair(&acc_full[buf]);
                        }
                        __syncwarp();
                    }
                    if (++s == STAGES) s = 0, ++turn;
                }
            }
            if (!ok) {  // nor for the products
                if (umma::elect_one()) umma::commit_pair(&drained[which]);
                (void)tma::mbar_wait(&drained[which], 0);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    cg::this_cluster().sync();  // neither leaves while the other reads its memory or arrives at its barriers
    if (waits.failed()) {  // (both CTAs know.)  Nobody waits for the copies on their way any more, which are counted at the first CTA
        if (place == 0 && warp < FIRST_ISSUER) {
            for (int i = max(0, asked[warp] - STAGES); i < asked[warp]; ++i)
                if ((i & 1) == warp) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
        }
        cg::this_cluster().sync();
    }
    if (warp == FIRST_ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
}

template <typename TO>
int launch(const linear8::Operands& p, int early, int* error_flag, cudaStream_t stream) {
    constexpr int BN = 128, STAGES = 4;
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK + 1024 + EPI_WARPS * linear8::PIECE_BYTES<TO>;
    auto kernel = gemm8_tcgen05_kernel<STAGES, TO>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap xmap, wmap;
    if (!tma::make_map_2d_u8(&xmap, p.x, p.M, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tma::make_map_2d_u8(&wmap, p.w, p.N, p.K, p.K, BN, BK, CU_TENSOR_MAP_SWIZZLE_128B))
        return LLM_ERR_UNSUPPORTED;
    const long long tiles = (long long)((p.N + BN - 1) / BN) * ((p.M + BM - 1) / BM);
    if (tiles > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    const int sms = device_sms();
    return launch_pdl(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(THREADS), smem, stream, p, early, error_flag, xmap, wmap);
}

template <typename TO>
int launch_pair(const linear8::Operands& p, int early, int* error_flag, cudaStream_t stream) {
    constexpr int STAGES = 4;
    constexpr size_t smem = (size_t)STAGES * 2 * BM * BK + 1024 + EPI_WARPS * linear8::PIECE_BYTES<TO>;
    auto kernel = gemm8_pair_kernel<STAGES, TO>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap xmap, wmap;
    if (!tma::make_map_2d_u8(&xmap, p.x, p.M, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tma::make_map_2d_u8(&wmap, p.w, p.N, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B))
        return LLM_ERR_UNSUPPORTED;
    const long long tiles = (long long)((p.N + 255) / 256) * ((p.M + 255) / 256);
    if (tiles > 0x3fffffffLL) return LLM_ERR_UNSUPPORTED;
    const int pairs = device_sms() / 2;
    return linear8::launch_clusters(kernel, (unsigned)(tiles < pairs ? tiles : pairs) * 2, THREADS, smem, 2, stream, p, early, error_flag, xmap, wmap);
}

// A pair's tile of 256 x 256 takes 0.57 us a k-block, a CTA's of 128 x 128 0.39: pairs are faster (4,096 x 28,672 x 4,096: 459 us) but
// where their tiles leave most of them without work (512 x 4,096 x 4,096, 32 tiles for 74 pairs: 18.5 us by single CTAs).
template <typename TO>
int by_shape(const linear8::Operands& p, int early, int* error_flag, cudaStream_t stream) {
    const long long sms = device_sms(), pairs = sms / 2;
    auto rounds = [&](long long side, long long at_once) { return (((p.M + side - 1) / side) * ((p.N + side - 1) / side) + at_once - 1) / at_once; };
    if (rounds(256, pairs) * 57 <= rounds(128, sms) * 39) return launch_pair<TO>(p, early, error_flag, stream);
    return launch<TO>(p, early, error_flag, stream);
}

}  // namespace

int linear8::many(const Operands& p, bool early, int* error_flag, cudaStream_t stream) {
    return p.out_dtype == LLM_F32 ? by_shape<float>(p, early, error_flag, stream) : by_shape<__nv_bfloat16>(p, early, error_flag, stream);
}
