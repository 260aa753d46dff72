// y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} x[m, k] w[n, k] for many rows: x and w in e4m3, a scale for every 128 k,
// on tcgen05 (kind::f8f6f4) with TMA-fed tiles.
//
// A k-block is a block of the scales: 128 bytes of a row, which is also the swizzle's width, so a slot of the ring holds one
// k-block of both operands.  Its four products (K = 32 each) start from zero in tensor memory and leave it at once: the epilogue
// warps add them to 32-bit sums in registers, times sx of their row and sw of their columns.  Scales of any value are allowed
// that way, and no sum is longer than 128 terms before it is rounded to 32 bits.  Roles, by warp:
//   warp 0, one thread : TMA producer, a ring of STAGES slots;
//   warp 1, one thread : issues the products into one of NBUF accumulators of tensor memory, in turn;
//   warps 2-9          : the sums.  A warp owns its 32 rows (lanes) and half of the tile's columns.
// One CTA per SM walks 128 x BN tiles, column tiles outermost, so that CTAs that run at the same time share their weights.  What lies beyond
// the matrices arrives as zeros and is masked at the store.  Every wait is bounded; one that gives up sets *error_flag and the
// roles run to their ends.
#include "common.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace {

constexpr int BM = 128, BK = 128, UMMA_K = 32, EPI_WARPS = 8;
constexpr int THREADS = 64 + EPI_WARPS * 32;

struct Gemm8Params {
    const float* sx;  // [M, kblocks]
    const float* sw;  // [ceil(N / 128), kblocks]
    void* out;
    int M, N, kblocks, ldo;
    int* error_flag;
};

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
gemm8_tcgen05_kernel(const Gemm8Params p, const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap) {
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

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
        if (p.error_flag) atomicExch(p.error_flag, 1);
    };
    auto failed = [&]() { return *(volatile int*)&gave_up != 0; };

    if (warp == 0 && lane == 0) {
        // ---- producer ----
        int it = 0;
        for (int tile = blockIdx.x; tile < tiles && !failed(); tile += gridDim.x) {
            const int m0 = (tile % row_tiles) * BM, n0 = (tile / row_tiles) * BN;
            for (int kb = 0; kb < kblocks && !failed(); ++kb, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES && !tma::mbar_wait(&empty[s], ((it / STAGES) - 1) & 1)) {
                    fail();
                    break;
                }
                unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                tma::mbar_expect_tx(&full[s], SLOT_BYTES);
                tma::load_2d(slot, &xmap, kb * BK, m0, &full[s]);
                tma::load_2d(slot + A_BYTES, &wmap, kb * BK, n0, &full[s]);
            }
        }
        if (failed())  // nobody waits for the copies on their way any more
            for (int i = it < STAGES ? 0 : it - STAGES; i < it; ++i) (void)tma::mbar_wait(&full[i % STAGES], (i / STAGES) & 1);
    } else if (warp == 1 && lane == 0) {
        // ---- tensor-core issuer ----
        int it = 0;
        for (int tile = blockIdx.x; tile < tiles && !failed(); tile += gridDim.x) {
            for (int kb = 0; kb < kblocks && !failed(); ++kb, ++it) {
                const int s = it % STAGES, buf = it % NBUF;
                if (!tma::mbar_wait(&full[s], (it / STAGES) & 1) ||
                    (it >= NBUF && !tma::mbar_wait(&acc_empty[buf], ((it / NBUF) - 1) & 1))) {
                    fail();
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const unsigned char* slot = ring + (size_t)s * SLOT_BYTES;
                const unsigned long long a = umma::desc_sw128(slot), b = umma::desc_sw128(slot + A_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)  // 32 k = 32 bytes further along the rows: two 16-byte units
                    umma::mma_e4m3(tmem_base + buf * BN, a + 2 * k, b + 2 * k, IDESC, k != 0);
                umma::commit(&empty[s]);
                umma::commit(&acc_full[buf]);
            }
        }
        if (failed()) {  // nor for the products
            umma::commit(&drained);
            (void)tma::mbar_wait(&drained, 0);
        }
    } else if (warp >= 2) {
        // ---- sums: warp w may touch the 32 lanes (warp % 4) * 32 .. of tensor memory ----
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        int it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
            const int m0 = (tile % row_tiles) * BM, n0 = (tile / row_tiles) * BN + half * COLS;
            const int row = m0 + quarter * 32 + lane;
            const float* sx = p.sx + (size_t)min(row, p.M - 1) * kblocks;
            const float* sw = p.sw + (size_t)(min(n0, p.N - 1) >> 7) * kblocks;  // the warp's columns lie in one block of 128
            float acc[COLS];
#pragma unroll
            for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
            float scale = sx[0] * sw[0];
            for (int kb = 0; kb < kblocks; ++kb, ++it) {
                const int buf = it % NBUF;
                const float next = kb + 1 < kblocks ? sx[kb + 1] * sw[kb + 1] : 0.f;
                ok = __all_sync(0xffffffffu, !failed() && tma::mbar_wait(&acc_full[buf], (it / NBUF) & 1));
                if (!ok) {
                    if (lane == 0) fail();
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const unsigned base = tmem_base + buf * BN + half * COLS + ((unsigned)(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < COLS; c += 32) {
                    float v[32];
                    umma::tmem_ld32(base + c, v);
                    if (c + 32 == COLS) {  // this warp has read its part: the accumulator may be filled again
                        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                        __syncwarp();
                        if (lane == 0) tma::mbar_arrive(&acc_empty[buf]);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c + j] = fmaf(v[j], scale, acc[c + j]);
                }
                scale = next;
            }
            if (ok && row < p.M) {
#pragma unroll
                for (int c = 0; c < COLS; c += 32)
                    if (n0 + c < p.N) store_row<TO>(reinterpret_cast<TO*>(p.out) + (size_t)row * p.ldo + n0 + c, acc + c, p.N - n0 - c);
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
int launch(const void* x, const void* w, int K, const Gemm8Params& p, cudaStream_t stream) {
    constexpr size_t smem = (size_t)STAGES * (BM + BN) * BK + 1024;
    auto kernel = gemm8_tcgen05_kernel<BN, STAGES, TO>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap xmap, wmap;
    if (!tma::make_map_2d_u8(&xmap, x, p.M, K, K, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !tma::make_map_2d_u8(&wmap, w, p.N, K, K, BN, BK, CU_TENSOR_MAP_SWIZZLE_128B))
        return LLM_ERR_UNSUPPORTED;
    const long long tiles = (long long)((p.N + BN - 1) / BN) * ((p.M + BM - 1) / BM);
    if (tiles > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    const int sms = device_sms();
    return launch_pdl(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(THREADS), smem, stream, p, xmap, wmap);
}

template <typename TO>
int by_shape(const void* x, const void* w, int K, const Gemm8Params& p, cudaStream_t stream) {
    const int sms = device_sms(), row_tiles = (p.M + BM - 1) / BM;
    int best = 64;
    double least = 1e30;
    for (int bn : {256, 128, 64}) {
        const long long tiles = (long long)((p.N + bn - 1) / bn) * row_tiles;
        const double cost = (double)((tiles + sms - 1) / sms) * (bn + 40);
        if (cost < least) least = cost, best = bn;
    }
    if (best == 256) return launch<256, 4, TO>(x, w, K, p, stream);
    if (best == 128) return launch<128, 6, TO>(x, w, K, p, stream);
    return launch<64, 8, TO>(x, w, K, p, stream);
}

}  // namespace

// x [M, K] and w [N, K] e4m3, contiguous, on 16 bytes, K a multiple of 16; sx [M, ceil(K / 128)], sw [ceil(N / 128), ceil(K / 128)] float32;
// out [M, N] (row stride ldo), float32 or bfloat16.
LLM_EXPORT int llm_gemm8_tcgen05(const void* x, const float* sx, const void* w, const float* sw, void* out, int out_dtype, int M, int N, int K,
                                 int ldo, int* error_flag, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K < 16 || (K & 15) || ((uintptr_t)x & 15) || ((uintptr_t)w & 15)) return LLM_ERR_BAD_ARGUMENT;
    Gemm8Params p = {sx, sw, out, M, N, (K + BK - 1) / BK, ldo, error_flag};
    if (out_dtype == LLM_F32) return by_shape<float>(x, w, K, p, stream);
    if (out_dtype == LLM_BF16) return by_shape<__nv_bfloat16>(x, w, K, p, stream);
    return LLM_ERR_BAD_ARGUMENT;
}
