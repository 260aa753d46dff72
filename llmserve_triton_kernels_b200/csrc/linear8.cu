// A product with 8-bit weights as one call: the rows of x are quantised (unless they come so), then go to the kernel for so
// many of them.
#include "linear8.h"

#include "common.cuh"

// x [M, K]: float32 or bfloat16 (x_dtype; row stride ldx, unit inner stride), quantised into `scratch` (16-byte aligned, M K + 4 M ceil(K / 128)
// bytes); or, with sx [M, ceil(K / 128)] float32 (not null), e4m3, contiguous, on 16 bytes.  w [N, K] e4m3, contiguous, on 16 bytes; sw
// [ceil(N / 128), ceil(K / 128)] float32; `powers`: these scales, and those of an x that comes quantised, are powers of two.  K a
// multiple of 16.  out [M, N] (row stride ldo), float32 or bfloat16.
LLM_EXPORT int llm_linear8(const void* x, int x_dtype, long long ldx, const float* sx, void* scratch, const void* w, const float* sw, int powers, void* out,
                           int out_dtype, int M, int N, int K, int ldo, int* error_flag, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K < 16 || (K & 15) || ((uintptr_t)w & 15) || (out_dtype != LLM_F32 && out_dtype != LLM_BF16)) return LLM_ERR_BAD_ARGUMENT;
    const bool given = sx != nullptr;
    if (given ? ((uintptr_t)x & 15) != 0 : !scratch || ((uintptr_t)scratch & 15)) return LLM_ERR_BAD_ARGUMENT;
    linear8::Operands p = {(const unsigned char*)x, sx, given ? (K + 127) / 128 : 1, given ? 1 : M, (const unsigned char*)w, sw, out, M, N, K,
                           (K + 127) / 128, ldo, out_dtype};
    if (!given) {
        unsigned char* values = (unsigned char*)scratch;
        float* scales = reinterpret_cast<float*>(values + (size_t)M * K);  // K is a multiple of 16
        const int code = linear8::quantize_rows(x, x_dtype, ldx, values, scales, M, K, stream);
        if (code) return code;
        p.x = values;
        p.sx = scales;
    }
    // The weights may be asked for early only if the kernel in front is the one that quantised x here: it began when all before it
    // had ended, whoever wrote the weights among them.
    if (M <= linear8::FEW_ROWS || (M <= 2 * linear8::FEW_ROWS && (long long)N * K <= linear8::FEW_BYTES)) return linear8::few(p, !given, stream);
    // The weights as the tall operand where x fills no tile of 128 rows by half, and where there are so few tiles that several CTAs may
    // share one's k-blocks (which those kernels do).
    const long long tiles = (long long)((M + 127) / 128) * ((N + 127) / 128), pair_tiles = (long long)((M + 255) / 256) * ((N + 255) / 256), sms = device_sms();
    if (M <= 64 || tiles * 2 <= sms) return powers ? linear8::some_scaled(p, !given, error_flag, stream) : linear8::some(p, !given, error_flag, stream);
    // Powers of two go to the pairs of CTAs that leave them to the tensor cores where tiles of 128 x 128 go round more than once (measured with
    // x quantised in front: 4,096 rows by 28,672 features of 4,096 357 us against 459; 512 by 4,096, once round, 20.3 against 18.5), two pairs to
    // a tile where clusters of four find room for all tiles (some SMs are left over) and have k-blocks to share (512 by 4,096 of
    // 14,336 36.5 us against 51.9, 1,024 by 2,048 of 5,632 22.5 against 24.8; 512 by 2,560 of 2,048 13.6 against 12.0).
    if (powers && pair_tiles * 4 <= sms * 7 / 8 && p.kblocks >= 32) return linear8::many_scaled(p, 2, !given, error_flag, stream);
    return powers && tiles > sms ? linear8::many_scaled(p, 1, !given, error_flag, stream) : linear8::many(p, !given, error_flag, stream);
}
