// A step's query heads rotated in place, its key heads rotated and its value heads as they are written into 8-bit pages: e4m3
// values and, for every head's vector, a power of two (fp8.cuh) as its biased exponent in a byte.
//
//   pool      [pages, 2, KV, page_size, D] e4m3     (keys, values)
//   exponents [pages, 2, KV, page_size]    uint8    value = e4m3 * 2^(exponent - 127)
//
// Lanes j and j + D/2 of a head form a pair; D/16 neighbouring threads share a vector, eight pairs a thread, so that a vector is read
// with 16-byte loads and its largest value found without shared memory.  The rotation is rounded as it is written (two products, a
// sum), so that an element does not depend on what the compiler contracts.
//
// The bytes bound it, behind a chain of loads (position, the table's row): 3,600 tokens of 32 query and 8 key heads of 128 lanes take 20 us, 4.2
// TB/s of rows and pages; two or four vectors a thread, or registers for more blocks an SM, did not change that.  A step of 8 tokens takes 3.9
// us, a launch and the chain.
#include "fp8.cuh"

namespace {

using fp8::load8;
using fp8::store8;

constexpr int THREADS = 256;

template <int D>
__global__ void __launch_bounds__(THREADS)
rope_kv_write8_kernel(__nv_bfloat16* __restrict__ qkv, long long row_stride, const int* __restrict__ positions, const float* __restrict__ table,
                      int table_rows, const int* __restrict__ slot_map, unsigned char* __restrict__ pool, unsigned char* __restrict__ exponents,
                      int n, int H, int KV, int page_size, int pages) {
    constexpr int LANES = D / 16, HALF = D / 2;  // threads of a vector
    pdl_wait();
    pdl_trigger();
    const unsigned vectors = H + 2 * KV, unit = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;  // (2^32 vectors fill more than the memory)
    if (unit >= n * vectors) return;
    const int sub = threadIdx.x % LANES;
    const int t = unit / vectors, v = unit - t * vectors;
    __nv_bfloat16* x = qkv + t * row_stride + (long long)v * D + sub * 8;
    float lo[8], hi[8];
    load8(x, lo);
    load8(x + HALF, hi);
    if (v < H + KV && table) {
        const int pos = min(max(positions[t], 0), table_rows - 1);
        float c[8], s[8];
        load8(table + (size_t)pos * D + sub * 8, c);
        load8(table + (size_t)pos * D + HALF + sub * 8, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = lo[e], b = hi[e];
            lo[e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
            hi[e] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
        }
    }
    if (v < H) {
        if (table) {
            store8(x, lo);
            store8(x + HALF, hi);
        }
        return;
    }
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, max(fp8::finite_bits(lo[e]), fp8::finite_bits(hi[e])));
    // the vector's threads alone: a neighbour may hold a query's, which has left
    const unsigned mask = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u)) << ((threadIdx.x & 31) / LANES * LANES);
    const unsigned e = fp8::scale_exponent(__reduce_max_sync(mask, top));
    const int slot = slot_map[t], page = slot / page_size;
    if (slot < 0 || page >= pages) return;
    const int which = v >= H + KV, head = v - H - which * KV;
    const long long at = (((long long)page * 2 + which) * KV + head) * page_size + (slot - page * page_size);
    const float inv = fp8::inverse(e);
    unsigned char* dst = pool + at * D + sub * 8;
    *reinterpret_cast<uint2*>(dst) = make_uint2(fp8::pack4(lo[0], lo[1], lo[2], lo[3], inv), fp8::pack4(lo[4], lo[5], lo[6], lo[7], inv));
    *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(fp8::pack4(hi[0], hi[1], hi[2], hi[3], inv), fp8::pack4(hi[4], hi[5], hi[6], hi[7], inv));
    if (sub == 0) exponents[at] = (unsigned char)e;
}

template <int D>
int launch(void* qkv, long long row_stride, const int* positions, const float* table, int table_rows, const int* slot_map, void* pool,
           unsigned char* exponents, int n, int H, int KV, int page_size, int pages, cudaStream_t stream) {
    const long long units = (long long)n * (H + 2 * KV), per = THREADS / (D / 16), blocks = (units + per - 1) / per;
    if (units > 0xffffffffLL || blocks > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    return launch_pdl(rope_kv_write8_kernel<D>, dim3((unsigned)blocks), dim3(THREADS), 0, stream, (__nv_bfloat16*)qkv, row_stride, positions,
                      table, table_rows, slot_map, (unsigned char*)pool, exponents, n, H, KV, page_size, pages);
}

}  // namespace

// qkv [n, >= (H + 2 KV) D] bfloat16 (row stride a multiple of 8, 16-byte aligned, as the table is); table [table_rows, D] float32 (cos | sin) or null: no
// rotation; D 64 or 128.  A token whose slot lies outside the pool is not written.
LLM_EXPORT int llm_rope_kv_write8(void* qkv, long long row_stride, const int* positions, const float* table, int table_rows, const int* slot_map,
                                  void* pool, unsigned char* exponents, int n, int H, int KV, int D, int page_size, int pages, cudaStream_t stream) {
    if (n <= 0) return 0;
    if (H < 0 || KV <= 0 || page_size <= 0 || pages <= 0 || (table && table_rows <= 0) || (row_stride & 7) || ((uintptr_t)qkv & 15) ||
        ((uintptr_t)table & 15) || ((uintptr_t)pool & 7))
        return LLM_ERR_BAD_ARGUMENT;
    if (D == 64) return launch<64>(qkv, row_stride, positions, table, table_rows, slot_map, pool, exponents, n, H, KV, page_size, pages, stream);
    if (D == 128) return launch<128>(qkv, row_stride, positions, table, table_rows, slot_map, pool, exponents, n, H, KV, page_size, pages, stream);
    return LLM_ERR_UNSUPPORTED;
}
