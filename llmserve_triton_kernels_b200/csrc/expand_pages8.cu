// Pages in 8 bits as bfloat16 pages, for requests that bring so many tokens that the products bound their attention: there the tcgen05
// kernel over bfloat16 pages does it, and what every tile of rows would unpack anew is unpacked once.  A number e4m3 * 2^e is a bfloat16
// number, so nothing is rounded, but for the smallest of all and for 2^128, to which bfloat16's largest numbers are rounded in 8 bits: it becomes
// the largest of bfloat16 again, 2^-8 less, because an infinity would make NaN of the rows that do not see it.
//
// Request r's pages lie one after another from page rank(r) * width on, rank counting the requests that bring at least `least` tokens.
// Three portions of up to 301 tokens in contexts of up to 1,501 (32 query and 4 key heads of 64 lanes) take 43 us this way, and 128 by the
// tiles of attention8.cu, which unpack a page for every 16 rows.
// Places behind a request's end become zeros.  One CTA a page: 16 values a thread at a time, a 16-byte read and two 16-byte writes.
//
// That kernel gives a key that a row does not see a weight of zero, and zero times NaN is NaN.  So NaN among the values becomes zero here, the page is
// marked, and a second kernel behind the attention writes NaN where a row sees one: the lane's last NaN at or before the row's position lies in its
// window.  One CTA for a request's key head walks the keys of marked pages, a lane a thread; where no page is marked it ends at once (four portions
// of up to 128 tokens behind 1,000 keys, 32 query and 4 key heads of 64 lanes, 24.1 us with it and 23.0 without).
#include "fp8.cuh"

namespace {

constexpr int THREADS = 256;

// Within bfloat16's numbers; a key's NaN stays one.
__device__ __forceinline__ float held(float v) {
    const float most = __uint_as_float(0x7f7f0000u);
    return v > most ? most : v < -most ? -most : v;
}

template <int D>
__global__ void __launch_bounds__(THREADS)
expand_pages8_kernel(const unsigned char* __restrict__ pool, const unsigned char* __restrict__ exponents, const int* __restrict__ page_table, int width,
                     const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, int KV, int page_size, int pages, int window, int least,
                     __nv_bfloat16* __restrict__ out, int* __restrict__ out_table, int* __restrict__ marks) {
    const int r = blockIdx.y, at = blockIdx.x;
    pdl_wait();
    pdl_trigger();
    const int n = cu_tokens[r + 1] - cu_tokens[r];
    int before = 0;
    for (int r0 = 0; r0 < r; r0 += THREADS) {
        const int i = r0 + threadIdx.x;
        before += __syncthreads_count(i < r && cu_tokens[min(i, r) + 1] - cu_tokens[min(i, r)] >= least);
    }
    const int ctx = context_lens[r], first = window > 0 ? max(0, ctx - n - window + 1) : 0;
    const bool needed = n >= least && at * page_size < ctx && (at + 1) * page_size > first;
    const int to = before * width + at;
    if (threadIdx.x == 0) {
        out_table[(long long)r * width + at] = needed ? to : 0;
        if (!needed) marks[(long long)r * width + at] = 0;
    }
    if (!needed) return;
    bool spoilt = false;
    const long long from = min(max(page_table[(long long)r * width + at], 0), pages - 1);
    const long long keys = 2LL * KV * page_size;
    constexpr int PIECES = D / 16;
    for (int i = threadIdx.x; i < keys * PIECES; i += THREADS) {
        const int key = i / PIECES, c = (i - key * PIECES) * 16;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        float scale = 0.f;
        if (at * page_size + key % page_size < ctx) {
            w = *reinterpret_cast<const uint4*>(pool + (from * keys + key) * D + c);
            scale = fp8::power(exponents[from * keys + key]);
        }
        unsigned words[4] = {w.x, w.y, w.z, w.w};
        if (key >= KV * page_size) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned bad = __vcmpeq4(words[k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                spoilt |= bad != 0u;
                words[k] &= ~bad;
            }
        }
        float v[2][8];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 f = fp8::unpack2((unsigned short)(words[k] >> (16 * e)));
                v[k >> 1][(k & 1) * 4 + 2 * e] = held(f.x * scale);
                v[k >> 1][(k & 1) * 4 + 2 * e + 1] = held(f.y * scale);
            }
        __nv_bfloat16* dst = out + (to * keys + key) * D + c;
        fp8::store8(dst, v[0]);
        fp8::store8(dst + 8, v[1]);
    }
    spoilt = __syncthreads_or(spoilt);
    if (threadIdx.x == 0) marks[(long long)r * width + at] = spoilt;
}

template <int D>
__global__ void __launch_bounds__(D)
spread_nan8_kernel(const unsigned char* __restrict__ pool, const int* __restrict__ page_table, const int* __restrict__ marks, int width,
                   const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, int KV, int G, int page_size, int pages, int window,
                   __nv_bfloat16* __restrict__ out, long long out_stride) {
    const int h = blockIdx.x, r = blockIdx.y, lane = threadIdx.x;
    marks += (long long)r * width;
    page_table += (long long)r * width;
    pdl_trigger();
    pdl_wait();
    bool any = false;
    for (int at = lane; at < width; at += D) any |= marks[at] != 0;
    if (!__syncthreads_or(any)) return;
    const int first = cu_tokens[r], n = cu_tokens[r + 1] - first, ctx = context_lens[r], start = ctx - n;
    const int lo = window > 0 ? max(0, start - window + 1) / page_size : 0, hi = (int)(((long long)ctx + page_size - 1) / page_size);
    int latest = -1;  // the lane's last NaN so far
    for (int at = lo; at < hi; ++at) {
        const bool marked = at < width && marks[at] != 0;
        const long long page = marked ? min(max(page_table[at], 0), pages - 1) : 0;
        const unsigned char* values = pool + (((page * 2 + 1) * KV + h) * page_size) * D + lane;
        const int j0 = at * page_size, here = min(page_size, ctx - j0);
#pragma unroll 4
        for (int i = 0; i < here; ++i) {
            const int j = j0 + i;
            if (marked && (values[(long long)i * D] & 0x7fu) == 0x7fu) latest = j;
            if (j < start || latest < 0 || (window > 0 && j - latest >= window)) continue;
            __nv_bfloat16* row = out + (first + j - start) * out_stride + (long long)h * G * D + lane;
            for (int m = 0; m < G; ++m) row[m * D] = __ushort_as_bfloat16((unsigned short)0x7fffu);
        }
    }
}

}  // namespace

// pool and exponents as rope_kv_write8.cu leaves them (the pool on 16 bytes).  out: bfloat16 [requests with at least `least` tokens x width pages, 2, KV,
// page_size, D]; out_table and marks [requests, width].  window 0: none; else pages that no token's window reaches are left as they are.  D 64 or 128.
LLM_EXPORT int llm_expand_pages8(const void* pool, const void* exponents, const int* page_table, int width, const int* cu_tokens,
                                 const int* context_lens, int requests, int KV, int D, int page_size, int pages, int window, int least, void* out,
                                 int* out_table, int* marks, cudaStream_t stream) {
    if (requests <= 0 || width <= 0) return 0;
    if (KV <= 0 || page_size <= 0 || pages <= 0 || least <= 0 || window < 0 || ((uintptr_t)pool & 15) || ((uintptr_t)out & 15) ||
        2LL * KV * page_size * (D / 16) > 0x7fffffffLL)
        return LLM_ERR_BAD_ARGUMENT;
    if (requests > 65535 || (D != 64 && D != 128)) return LLM_ERR_UNSUPPORTED;
    return launch_pdl(D == 64 ? expand_pages8_kernel<64> : expand_pages8_kernel<128>, dim3(width, requests), dim3(THREADS), 0, stream,
                      (const unsigned char*)pool, (const unsigned char*)exponents, page_table, width, cu_tokens, context_lens, KV, page_size, pages,
                      window, least, (__nv_bfloat16*)out, out_table, marks);
}

// ... behind the attention over what llm_expand_pages8 unpacked, from the same arguments and its marks: NaN for the rows and lanes of out [n, H D]
// (row stride out_stride, H = KV G) that see a NaN among the pages' values.
LLM_EXPORT int llm_spread_nan8(const void* pool, const int* page_table, const int* marks, int width, const int* cu_tokens, const int* context_lens,
                               int requests, int KV, int G, int D, int page_size, int pages, int window, void* out, long long out_stride,
                               cudaStream_t stream) {
    if (requests <= 0 || width <= 0) return 0;
    if (KV <= 0 || G <= 0 || page_size <= 0 || pages <= 0 || window < 0 || (long long)width * page_size > 0x7fff0000) return LLM_ERR_BAD_ARGUMENT;
    if (requests > 65535 || (D != 64 && D != 128)) return LLM_ERR_UNSUPPORTED;
    return launch_pdl(D == 64 ? spread_nan8_kernel<64> : spread_nan8_kernel<128>, dim3(KV, requests), dim3(D), 0, stream, (const unsigned char*)pool,
                      page_table, marks, width, cu_tokens, context_lens, KV, G, page_size, pages, window, (__nv_bfloat16*)out, out_stride);
}
