// y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k] for many rows: x and w in e4m3, a scale for every 128 k,
// on tcgen05 (kind::f8f6f4) with TMA-fed tiles.
//
// A k-block is a block of the scales: 128 bytes of a row, which is also the swizzle's width, so a slot of the ring holds one
// k-block of both operands.  Its four products (K = 32 each) start from zero in tensor memory and leave it at once: the epilogue
// warps add them to 32-bit sums in registers, times sx of their row and sw of their columns.  Scales of any value are allowed
// that way, and no sum is longer than 128 terms before it is rounded to 32 bits.  Roles, by warp:
//   warp 0     : TMA producer, a ring of STAGES slots;
//   warp 1     : issues the products into one of NBUF accumulators of tensor memory, in turn;
//   warps 4-11 : the sums.  A warp owns its 32 rows (lanes) and half of the tile's columns, two columns to an instruction
//                (fma.rn.f32x2); it asks for 32 columns of tensor memory while it adds the 32 before.  128 sums and two times
//                32 columns need more registers than a third of the SM has: the first four warps give theirs up.
// One CTA per SM walks 128 x BN tiles, column tiles outermost, so that CTAs that run at the same time share their weights.  What lies beyond
// the matrices arrives as zeros and is masked at the store.  Every wait is bounded; one that gives up sets *error_flag and the
// roles run to their ends.
#include "common.cuh"
#include "linear8.h"
#include "tma.cuh"
#include "umma.cuh"

namespace {

constexpr int BM = 128, BK = 128, UMMA_K = 32, EPI_WARPS = 8, FIRST_EPI = 4;
constexpr int THREADS = (FIRST_EPI + EPI_WARPS) * 32;
// 384 threads are launched with 168 registers each: 3 x 168 = 40 + 2 x 232
constexpr int FEW_REGISTERS = 40, MANY_REGISTERS = 232;

__device__ __forceinline__ unsigned long long pair_of(unsigned lo, unsigned hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}

// sums += columns * scale, 32 columns as 16 pairs.
__device__ __forceinline__ void add_columns(unsigned long long* sums, const unsigned (&v)[32], unsigned long long scale) {
#pragma unroll
    for (int j = 0; j < 16; ++j) asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(sums[j]) : "l"(pair_of(v[2 * j], v[2 * j + 1])), "l"(scale));
}

template <typename TO>
__device__ __forceinline__ void store_row(TO* dst, const float* v, int valid);
template <>
__device__ __forceinline__ void store_row<float>(float* dst, const float* v, int valid) {
    if (valid >= 32 && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < valid) dst[i] = v[i];
    }
}
template <>
__device__ __forceinline__ void store_row<__nv_bfloat16>(__nv_bfloat16* dst, const float* v, int valid) {
    if (valid >= 32 && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            unsigned u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(v[i + 2 * j], v[i + 2 * j + 1]);
                u[j] = *reinterpret_cast<const unsigned*>(&a);
            }
            *reinterpret_cast<uint4*>(dst + i) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < valid) dst[i] = __float2bfloat16_rn(v[i]);
    }
}

template <int BN, int STAGES, typename TO>
__global__ void __launch_bounds__(THREADS, 1)
gemm8_tcgen05_kernel(const linear8::Operands p, int* error_flag, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
    constexpr int A_BYTES = BM * BK, SLOT_BYTES = A_BYTES + BN * BK;
    constexpr int NBUF = BN == 256 ? 2 : 4, TMEM_COLS = NBUF * BN;
    static_assert(TMEM_COLS == 512 || TMEM_COLS == 256, "columns of tensor memory come in powers of two");
    constexpr int COLS = BN / 2;  // of an epilogue warp
    constexpr unsigned IDESC = umma::idesc_e4m3(BM, BN);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) unsigned long long full[STAGES], empty[STAGES], acc_full[NBUF], acc_empty[NBUF], drained;
    __shared__ unsigned tmem_base;
    __shared__ int gave_up;

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
        tma::mbar_init(&drained, 1);
        gave_up = 0;
        tma::mbar_fence_init();
        tma::prefetch_map(&xmap);
        tma::prefetch_map(&wmap);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tma::smem_addr(&tmem_base)), "n"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    pdl_wait();  // x comes from the kernel before
    pdl_trigger();

    auto fail = [&]() {
        *(volatile int*)&gave_up = 1;
        if (error_flag) atomicExch(error_flag, 1);
    };
    auto failed = [&]() { return *(volatile int*)&gave_up != 0; };

    // (each role's share of the registers is set where the role begins: what follows a smaller share is compiled for it)
    if (warp >= FIRST_EPI) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(MANY_REGISTERS));
        // ---- sums: warp w may touch the 32 lanes (warp % 4) * 32 .. of tensor memory ----
        const int quarter = warp & 3, half = (warp - FIRST_EPI) >> 2;
        int it = 0;
        bool ok = true;
        auto release = [&](int buf) {  // this warp has read its part: the accumulator may be filled again
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) tma::mbar_arrive(&acc_empty[buf]);
        };
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            const int m0 = (tile % row_tiles) * BM, n0 = (tile / row_tiles) * BN + half * COLS;
            const int row = m0 + quarter * 32 + lane;
            const float* sx = p.sx + (size_t)min(row, p.M - 1) * kblocks;
            const float* sw = p.sw + (size_t)(min(n0, p.N - 1) >> 7) * kblocks;  // the warp's columns lie in one block of 128
            unsigned long long acc[COLS / 2];  // two 32-bit sums each
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
            // the scales of four k-blocks are asked for four k-blocks ahead
            float sx_now[4], sw_now[4], sx_next[4], sw_next[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sx_next[i] = sx[min(i, kblocks - 1)], sw_next[i] = sw[min(i, kblocks - 1)];
            for (int k0 = 0; k0 < kblocks && ok; k0 += 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sx_now[i] = sx_next[i], sw_now[i] = sw_next[i];
                sx_next[i] = sx[min(k0 + 4 + i, kblocks - 1)], sw_next[i] = sw[min(k0 + 4 + i, kblocks - 1)];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (k0 + i >= kblocks) break;
                const int buf = it % NBUF;
                const float scale = sx_now[i] * sw_now[i];
                ok = __all_sync(0xffffffffu, !failed() && tma::mbar_wait(&acc_full[buf], (it / NBUF) & 1));
                if (!ok) {
                    if (lane == 0) fail();
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const unsigned base = tmem_base + buf * BN + half * COLS + ((unsigned)(quarter * 32) << 16);
                const unsigned long long both = pair_of(__float_as_uint(scale), __float_as_uint(scale));
                unsigned v0[32], v1[32];
                umma::tmem_ask32(base, v0);
#pragma unroll
                for (int c = 0; c < COLS; c += 64) {
                    umma::tmem_have32(v0);
                    if (c + 32 < COLS) umma::tmem_ask32(base + c + 32, v1); else release(buf);
                    add_columns(acc + c / 2, v0, both);
                    if (c + 32 >= COLS) break;
                    umma::tmem_have32(v1);
                    if (c + 64 < COLS) umma::tmem_ask32(base + c + 64, v0); else release(buf);
                    add_columns(acc + c / 2 + 16, v1, both);
                }
                ++it;
            }
            }
            if (ok && row < p.M) {
#pragma unroll
                for (int c = 0; c < COLS; c += 32) {
                    if (n0 + c >= p.N) continue;
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        v[2 * j] = __uint_as_float((unsigned)acc[c / 2 + j]);
                        v[2 * j + 1] = __uint_as_float((unsigned)(acc[c / 2 + j] >> 32));
                    }
                    store_row<TO>(reinterpret_cast<TO*>(p.out) + (size_t)row * p.ldo + n0 + c, v, p.N - n0 - c);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(FEW_REGISTERS));
        auto there = [&](unsigned long long* bar, unsigned parity) {  // for the whole warp
            if (__all_sync(0xffffffffu, tma::mbar_wait(bar, parity))) return true;
            fail();
            return false;
        };
        if (warp == 0) {
            // ---- producer ----
            int it = 0, s = 0, turn = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int m0 = (tile % row_tiles) * BM, n0 = (tile / row_tiles) * BN;
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
                    if (it >= STAGES) ok = there(&empty[s], (turn - 1) & 1) && !failed();
                    if (!ok) break;
                    unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                    if (umma::elect_one()) {
                        tma::mbar_expect_tx(&full[s], SLOT_BYTES);
                        tma::load_2d(slot, &xmap, kb * BK, m0, &full[s]);
                        tma::load_2d(slot + A_BYTES, &wmap, kb * BK, n0, &full[s]);
                    }
                    __syncwarp();
                    if (++s == STAGES) s = 0, ++turn;
                }
            }
            if (!ok)  // nobody waits for the copies on their way any more
                for (int i = it < STAGES ? 0 : it - STAGES; i < it; ++i) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
        } else if (warp == 1) {
            // ---- tensor-core issuer ----
            int it = 0, s = 0, turn = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                for (int kb = 0; kb < kblocks; ++kb, ++it) {
                    const int buf = it % NBUF;
                    ok = there(&full[s], turn & 1) && (it < NBUF || there(&acc_empty[buf], ((it / NBUF) - 1) & 1));
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
                    if (++s == STAGES) s = 0, ++turn;
                }
            }
            if (!ok) {  // nor for the products
                if (umma::elect_one()) umma::commit(&drained);
                (void)tma::mbar_wait(&drained, 0);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "n"(TMEM_COLS) : "memory");
    }
}

template <int BN, int STAGES, typename TO>
int launch(const linear8::Operands& p, int* error_flag, cudaStream_t stream) {
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK + 1024;
    auto kernel = gemm8_tcgen05_kernel<BN, STAGES, TO>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap xmap, wmap;
    if (!tma::make_map_2d_u8(&xmap, p.x, p.M, p.K, p.K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tma::make_map_2d_u8(&wmap, p.w, p.N, p.K, p.K, BN, BK, CU_TENSOR_MAP_SWIZZLE_128B))
        return LLM_ERR_UNSUPPORTED;
    const long long tiles = (long long)((p.N + BN - 1) / BN) * ((p.M + BM - 1) / BM);
    if (tiles > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    const int sms = device_sms();
    return launch_pdl(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(THREADS), smem, stream, p, error_flag, xmap, wmap);
}

template <typename TO>
int by_shape(const linear8::Operands& p, int* error_flag, cudaStream_t stream) {
    const int sms = device_sms(), row_tiles = (p.M + BM - 1) / BM;
    int best = 64;
    double least = 1e30;
    for (int bn : {256, 128, 64}) {
        const long long tiles = (long long)((p.N + bn - 1) / bn) * row_tiles;
        const double cost = (double)((tiles + sms - 1) / sms) * (bn + 40);
        if (cost < least) least = cost, best = bn;
    }
    if (best == 256) return launch<256, 4, TO>(p, error_flag, stream);
    if (best == 128) return launch<128, 6, TO>(p, error_flag, stream);
    return launch<64, 8, TO>(p, error_flag, stream);
}

}  // namespace

int linear8::many(const Operands& p, int* error_flag, cudaStream_t stream) {
    return p.out_dtype == LLM_F32 ? by_shape<float>(p, error_flag, stream) : by_shape<__nv_bfloat16>(p, error_flag, stream);
}
