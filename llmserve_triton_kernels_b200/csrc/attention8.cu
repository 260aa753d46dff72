// Attention over 8-bit pages (rope_kv_write8.cu), split over the cache's length and joined.
//
//   s_j = scale * 2^(ek_j) * q . k_j        out = sum_j 2^(s_j) 2^(ev_j) v_j / sum_j 2^(s_j)     (scale holds log2 e)
//
// Rows are (token, query head of the key head's group): 16 a CTA, the height of an mma.sync tile, so that one new token of a
// request whose group has up to 16 heads is one tile.  What bounds it is the pages' bytes; everything between them and the
// products is registers: with the lanes of a head permuted alike in q and k (a dot product does not notice) a thread's 16-byte
// load of a key holds the B elements of four products, and since the output's columns may come in any order, a thread's 16
// bytes of four values are the B elements of sixteen.  e4m3 becomes half precision (one instruction for two values, exact) on the
// way; q becomes half precision too, its row divided by a power of two so that it neither overflows nor loses bits.
//
// A value's weight 2^(s_j + ev_j) has a running maximum of its own, apart from that of 2^(s_j): whatever the values' scales, the
// weights that enter the half-precision product are at most one and the largest is one.
//
// The keys of a row tile are shared out over `splits` CTAs and their warps, 16 keys at a time; the warps meet in shared memory, the
// CTAs in a second kernel, through scratch memory of the call's own: nothing is kept from call to call.
//
// Masks: a key that no row of the tile may see, or that lies behind the request's end, is never multiplied (its 8 bits may be NaN).
// Where rows differ in what they see, NaN among the values is counted apart, so that it reaches the rows that see it alone.
#include "common.cuh"

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32, TILE = 16;

struct Attn8Params {
    const __nv_bfloat16* q;
    long long q_stride;
    __nv_bfloat16* out;
    long long out_stride;
    const unsigned char* pool;
    const unsigned char* exponents;
    const int* page_table;
    int table_width;
    const int* cu_tokens;
    const int* context_lens;
    int H, KV, G, page_size, pages, window, splits;
    float scale;      // times log2 e
    float* part_o;    // [rows of the step, splits, D]
    float* part_stat; // [rows of the step, splits, 3]: largest score, largest score with the value's scale, sum
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned half2_of(unsigned short v) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// What a thread holds of 16 keys: 16-byte pieces of keys g and g + 8, and of the values 2 t, 2 t + 1, 2 t + 8, 2 t + 9.
template <int D>
struct Keys {
    static constexpr int KW = D / 16;  // words of a key a thread: D / 4 bytes
    static constexpr int VW = D / 32;  // words of a value: D / 8 bytes
    unsigned k[2][KW], v[4][VW];
    unsigned ek[2], ev[2];  // exponents of keys / values (2 t | 2 t + 1), (2 t + 8 | 2 t + 9), a byte each
};

template <int WORDS>
__device__ __forceinline__ void load_words(unsigned (&w)[WORDS], const unsigned char* p) {
    if constexpr (WORDS >= 4) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        if constexpr (WORDS == 8) {
            const uint4 b = __ldg(reinterpret_cast<const uint4*>(p + 64));
            w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        }
    } else {
        const uint2 a = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = a.x; w[1] = a.y;
    }
}

// ALIGNED: a page holds whole tiles of 16 keys.
template <int D, bool ALIGNED>
__global__ void __launch_bounds__(THREADS)
attention8_kernel(const Attn8Params p) {
    constexpr int KSTEPS = D / 16, NTILES = D / 8;
    extern __shared__ __align__(16) float merge[];  // [WARPS][16][D + 4], then [WARPS][16][3]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int r = blockIdx.x / p.KV, h = blockIdx.x - r * p.KV, split = blockIdx.z;
    pdl_wait();
    pdl_trigger();
    const int first = p.cu_tokens[r], n = p.cu_tokens[r + 1] - first, ctx = p.context_lens[r];
    const int row0 = blockIdx.y * 16, rows = n * p.G;
    if (row0 >= rows) return;
    const int start = ctx - n;  // position of the request's first new token
    const int pos_min = start + row0 / p.G, pos_max = start + min(row0 + 15, rows - 1) / p.G;
    const int key_end = min(pos_max + 1, p.table_width * p.page_size);
    const int key_begin = p.window > 0 ? max(0, pos_min - p.window + 1) : 0;
    const int tile_begin = key_begin / TILE, tile_count = max(0, (key_end + TILE - 1) / TILE - tile_begin);
    const int per = (tile_count + p.splits - 1) / p.splits;
    const int tile_lo = tile_begin + split * per, tile_hi = tile_begin + min(tile_count, (split + 1) * per);

    // this thread's two rows
    int pos[2], token[2], head[2];
    bool live[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rho = row0 + g + 8 * i;
        live[i] = rho < rows;
        token[i] = live[i] ? rho / p.G : 0;
        head[i] = h * p.G + (live[i] ? rho - token[i] * p.G : 0);
        pos[i] = live[i] ? start + token[i] : -1;
        token[i] += first;
    }
    // q in half precision: product j of a key takes lanes (64 (j / 4) + 16 t + 4 (j % 4)) + 0 .. 3, or for D = 64 16 t + 4 j + 0 .. 3
    unsigned qa[KSTEPS][4];
    float factor[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        unsigned raw[KSTEPS][2];
        unsigned top = 0;
        const __nv_bfloat16* src = p.q + token[i] * p.q_stride + (long long)head[i] * D + 16 * t;
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j) {
            const uint2 w = live[i] ? *reinterpret_cast<const uint2*>(src + 64 * (j / 4) + 4 * (j % 4)) : make_uint2(0u, 0u);
            raw[j][0] = w.x;
            raw[j][1] = w.y;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const unsigned a = raw[j][e] & 0x7fffu, b = (raw[j][e] >> 16) & 0x7fffu;
                top = max(top, max(a < 0x7f80u ? a : 0u, b < 0x7f80u ? b : 0u));
            }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row's largest value to [2^14, 2^15): 2^shift, in two factors because either end may leave 32 bits' exponents
        const int shift = top ? 141 - max((int)(top >> 7), 1) : 0;
        const float f0 = __uint_as_float((unsigned)(127 + shift / 2) << 23), f1 = __uint_as_float((unsigned)(127 + shift - shift / 2) << 23);
        factor[i] = p.scale / f0 / f1;
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float a = __uint_as_float(raw[j][e] << 16) * f0 * f1, b = __uint_as_float(raw[j][e] & 0xffff0000u) * f0 * f1;
                qa[j][i + 2 * e] = pack_half(a, b);
            }
    }

    const int* table = p.page_table + (long long)r * p.table_width;
    const long long head_keys = (long long)p.page_size;  // keys of one head in a page
    // key `j` of the request as an index over [pages, 2, KV, page_size]
    auto place = [&](int j) -> long long {
        j = min(j, key_end - 1);  // behind the end: some key that is there, masked later
        const int at = j / p.page_size;
        const int page = min(max(table[at], 0), p.pages - 1);
        return ((long long)page * 2 * p.KV + h) * head_keys + (j - at * p.page_size);
    };
    const long long to_values = (long long)p.KV * head_keys;
    auto fetch = [&](Keys<D>& x, int tile) {
        const int j0 = tile * TILE;
        if constexpr (ALIGNED) {
            const long long base = place(j0);
            const unsigned char* kp = p.pool + base * D;
            const unsigned char* vp = kp + to_values * D;
#pragma unroll
            for (int i = 0; i < 2; ++i) load_words(x.k[i], kp + (g + 8 * i) * D + 16 * t);
#pragma unroll
            for (int i = 0; i < 4; ++i) load_words(x.v[i], vp + (2 * t + (i & 1) + 8 * (i >> 1)) * D + (D / 8) * g);
            const unsigned char* ep = p.exponents + base + 2 * t;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x.ek[i] = __ldg(reinterpret_cast<const unsigned short*>(ep + 8 * i));
                x.ev[i] = __ldg(reinterpret_cast<const unsigned short*>(ep + to_values + 8 * i));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) load_words(x.k[i], p.pool + place(j0 + g + 8 * i) * D + 16 * t);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                unsigned ek = 0, ev = 0;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const long long at = place(j0 + 2 * t + 8 * i + e);
                    load_words(x.v[2 * i + e], p.pool + (at + to_values) * D + (D / 8) * g);
                    ek |= (unsigned)__ldg(p.exponents + at) << (8 * e);
                    ev |= (unsigned)__ldg(p.exponents + at + to_values) << (8 * e);
                }
                x.ek[i] = ek;
                x.ev[i] = ev;
            }
        }
    };

    float o[NTILES][4];
#pragma unroll
    for (int i = 0; i < NTILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m1[2] = {-INFINITY, -INFINITY}, m2[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};  // sum: this thread's keys alone

    Keys<D> now, next;
    int tile = tile_lo + warp;
    if (tile < tile_hi) fetch(now, tile);
    for (; tile < tile_hi; tile += WARPS) {
        if (tile + WARPS < tile_hi) fetch(next, tile + WARPS);
        const int j0 = tile * TILE;
        // ---- scores: [row g | g + 8][key 2 t, 2 t + 1, 2 t + 8, 2 t + 9] ----
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
                mma_f16(c, qa[j], half2_of((unsigned short)now.k[i][j]), half2_of((unsigned short)(now.k[i][j] >> 16)));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float ks = __uint_as_float(((now.ek[i] >> (8 * e)) & 255u) << 23);
                s[0][2 * i + e] = c[e] * (ks * factor[0]);
                s[1][2 * i + e] = c[2 + e] * (ks * factor[1]);
            }
        }
        const bool whole = j0 + TILE - 1 <= pos_min && j0 + TILE <= key_end && (p.window <= 0 || j0 > pos_max - p.window);
        bool split_rows = false;  // some row sees a key of this tile that another does not
        if (!whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = j0 + 2 * t + (e & 1) + 8 * (e >> 1);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (j > pos[i] || j >= key_end || (p.window > 0 && j <= pos[i] - p.window)) s[i][e] = -INFINITY;
                // a value that no row of the tile sees is nobody's
                if (j > pos_max || j >= key_end || (p.window > 0 && j <= pos_min - p.window)) {
#pragma unroll
                    for (int w = 0; w < Keys<D>::VW; ++w) now.v[e][w] = 0u;
                }
            }
            split_rows = pos_min != pos_max;
        }
        // ---- running maxima and weights ----
        unsigned pa[4];
        float u[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float a = -INFINITY, b = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float ev = (float)((now.ev[e >> 1] >> (8 * (e & 1))) & 255u) - 127.f;
                u[i][e] = s[i][e] + ev;
                a = fmaxf(a, s[i][e]);
                b = fmaxf(b, u[i][e]);
            }
            a = fmaxf(m1[i], quad_max(a));
            b = fmaxf(m2[i], quad_max(b));
            const float a0 = a == -INFINITY ? 0.f : a, b0 = b == -INFINITY ? 0.f : b;
            const float keep = exp2_fast(m2[i] - b0);
            sum[i] *= exp2_fast(m1[i] - a0);
            m1[i] = a;
            m2[i] = b;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[i] += exp2_fast(s[i][e] - a0);
                u[i][e] = exp2_fast(u[i][e] - b0);
            }
#pragma unroll
            for (int x = 0; x < NTILES; ++x) {
                o[x][2 * i] *= keep;
                o[x][2 * i + 1] *= keep;
            }
        }
        pa[0] = pack_half(u[0][0], u[0][1]);
        pa[1] = pack_half(u[1][0], u[1][1]);
        pa[2] = pack_half(u[0][2], u[0][3]);
        pa[3] = pack_half(u[1][2], u[1][3]);
        // ---- values: column tile x takes lane (D / 8) g + x of every key ----
        bool nan_here = false;
        if (split_rows) {
            unsigned any = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < Keys<D>::VW; ++w) any |= __vcmpeq4(now.v[e][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
            nan_here = __any_sync(0xffffffffu, any != 0);
        }
        if (nan_here) {
            // NaN times a weight of zero is NaN: its places are taken out and counted by a product of their own, of ones where a
            // row sees a key and where a value is NaN
            unsigned seen[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = q & 1, e = 2 * (q >> 1);
                seen[q] = (s[i][e] == -INFINITY ? 0u : 0x3c00u) | (s[i][e + 1] == -INFINITY ? 0u : 0x3c000000u);
            }
#pragma unroll
            for (int x = 0; x < NTILES; ++x) {
                unsigned bad[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const unsigned lo = (now.v[2 * q][x / 4] >> (8 * (x & 3))) & 0x7fu, hi = (now.v[2 * q + 1][x / 4] >> (8 * (x & 3))) & 0x7fu;
                    bad[q] = (lo == 0x7fu ? 0x3c00u : 0u) | (hi == 0x7fu ? 0x3c000000u : 0u);
                }
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(c, seen, bad[0], bad[1]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c[e] > 0.f) o[x][e] = NAN;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < Keys<D>::VW; ++w) now.v[e][w] &= ~__vcmpeq4(now.v[e][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
        }
#pragma unroll
        for (int x = 0; x < NTILES; ++x) {
            const unsigned pick = 0x0040u + 0x0011u * (x & 3);  // byte x of the first word, byte x of the second
            const unsigned b0 = __byte_perm(now.v[0][x / 4], now.v[1][x / 4], pick), b1 = __byte_perm(now.v[2][x / 4], now.v[3][x / 4], pick);
            mma_f16(o[x], pa, half2_of((unsigned short)b0), half2_of((unsigned short)b1));
        }
        now = next;
    }

    // ---- the warps meet ----
    float* mine = merge + (size_t)warp * 16 * (D + 4);
    float* stats = merge + (size_t)WARPS * 16 * (D + 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        if (t == 0) {
            float* at = stats + (warp * 16 + g + 8 * i) * 3;
            at[0] = m1[i];
            at[1] = m2[i];
            at[2] = sum[i];
        }
    }
#pragma unroll
    for (int x = 0; x < NTILES; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e)  // column 2 t + (e & 1) of tile x is lane (D / 8) (2 t + (e & 1)) + x of the head
            mine[(g + 8 * (e >> 1)) * (D + 4) + (D / 8) * (2 * t + (e & 1)) + x] = o[x][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += THREADS) {
        const int row = i / (D / 4), c = (i - row * (D / 4)) * 4;
        const int rho = row0 + row;
        if (rho >= rows) continue;
        float a = -INFINITY, b = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            a = fmaxf(a, stats[(w * 16 + row) * 3]);
            b = fmaxf(b, stats[(w * 16 + row) * 3 + 1]);
        }
        const float a0 = a == -INFINITY ? 0.f : a, b0 = b == -INFINITY ? 0.f : b;
        float total = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* st = stats + (w * 16 + row) * 3;
            const float f = exp2_fast(st[1] - b0);
            total += st[2] * exp2_fast(st[0] - a0);
            const float4 x = *reinterpret_cast<const float4*>(merge + ((size_t)w * 16 + row) * (D + 4) + c);
            v[0] = fmaf(x.x, f, v[0]);
            v[1] = fmaf(x.y, f, v[1]);
            v[2] = fmaf(x.z, f, v[2]);
            v[3] = fmaf(x.w, f, v[3]);
        }
        const int tok = first + rho / p.G, hd = h * p.G + rho % p.G;
        if (p.splits == 1) {
            // a row that sees no key: zeros
            const float f = a == -INFINITY && total == 0.f ? 0.f : exp2f(b0 - a0) / total;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= f;
            store4(p.out + tok * p.out_stride + (long long)hd * D + c, v);
        } else {
            const long long at = ((long long)tok * p.H + hd) * p.splits + split;
            store4(p.part_o + at * D + c, v);
            if (c == 0) {
                p.part_stat[at * 3] = a;
                p.part_stat[at * 3 + 1] = b;
                p.part_stat[at * 3 + 2] = total;
            }
        }
    }
}

// Joins the splits of every row: D / 4 threads a row.
template <int D>
__global__ void __launch_bounds__(128)
attention8_join_kernel(const Attn8Params p, long long rows) {
    constexpr int LANES = D / 4;
    pdl_wait();
    pdl_trigger();
    const long long row = (long long)blockIdx.x * (128 / LANES) + threadIdx.x / LANES;
    if (row >= rows) return;
    const int c = (threadIdx.x % LANES) * 4;
    const float* stat = p.part_stat + row * p.splits * 3;
    float a = -INFINITY, b = -INFINITY;
    for (int s = 0; s < p.splits; ++s) {
        a = fmaxf(a, stat[s * 3]);
        b = fmaxf(b, stat[s * 3 + 1]);
    }
    const float a0 = a == -INFINITY ? 0.f : a, b0 = b == -INFINITY ? 0.f : b;
    float total = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        const float f = exp2_fast(stat[s * 3 + 1] - b0);
        total += stat[s * 3 + 2] * exp2_fast(stat[s * 3] - a0);
        float x[4];
        load4(p.part_o + (row * p.splits + s) * D + c, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
    }
    const float f = a == -INFINITY && total == 0.f ? 0.f : exp2f(b0 - a0) / total;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= f;
    const long long tok = row / p.H;
    store4(p.out + tok * p.out_stride + (row - tok * p.H) * D + c, v);
}

template <int D, bool ALIGNED>
int launch(const Attn8Params& p, int requests, int n, int longest, cudaStream_t stream) {
    constexpr size_t smem = (size_t)WARPS * 16 * (D + 4 + 3) * sizeof(float);
    const long long row_tiles = ((long long)longest * p.G + 15) / 16;
    if (row_tiles > 65535 || p.splits > 65535 || (long long)requests * p.KV > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    auto kernel = attention8_kernel<D, ALIGNED>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    const int code = launch_pdl(kernel, dim3(requests * p.KV, (unsigned)row_tiles, p.splits), dim3(THREADS), smem, stream, p);
    if (code || p.splits == 1) return code;
    const long long rows = (long long)n * p.H, per = 128 / (D / 4), blocks = (rows + per - 1) / per;
    if (blocks > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    return launch_pdl(attention8_join_kernel<D>, dim3((unsigned)blocks), dim3(128), 0, stream, p, rows);
}

}  // namespace

// q rows [n, >= H D] bfloat16 (row stride a multiple of 4, 8-byte aligned); pool and exponents as rope_kv_write8.cu leaves them; request r's
// new tokens are rows cu_tokens[r] .. cu_tokens[r + 1] - 1, the last one at position context_lens[r] - 1; `longest`: the most tokens a request
// brings.  out [n, H D].  splits > 1: part_o [n H splits D] and part_stat [n H splits 3] float32.  window 0: none.  D 64 or 128.
LLM_EXPORT int llm_attention8(const void* q, long long q_stride, void* out, long long out_stride, const void* pool, const void* exponents,
                              const int* page_table, int table_width, const int* cu_tokens, const int* context_lens, int requests, int n,
                              int longest, int H, int KV, int D, int page_size, int pages, int window, float scale, int splits, float* part_o,
                              float* part_stat, cudaStream_t stream) {
    if (n <= 0 || requests <= 0) return 0;
    if (H <= 0 || KV <= 0 || H % KV || page_size <= 0 || pages <= 0 || table_width <= 0 || longest <= 0 || splits <= 0 || window < 0 ||
        (splits > 1 && (!part_o || !part_stat)) || (q_stride & 3) || ((uintptr_t)q & 7) || (out_stride & 3) || ((uintptr_t)out & 7) ||
        ((uintptr_t)pool & 15) || ((uintptr_t)exponents & 15))
        return LLM_ERR_BAD_ARGUMENT;
    Attn8Params p = {(const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, (const unsigned char*)pool, (const unsigned char*)exponents,
                     page_table, table_width, cu_tokens, context_lens, H, KV, H / KV, page_size, pages, window, splits,
                     scale * 1.4426950408889634f, part_o, part_stat};
    const bool aligned = page_size % TILE == 0;
    if (D == 64) return aligned ? launch<64, true>(p, requests, n, longest, stream) : launch<64, false>(p, requests, n, longest, stream);
    if (D == 128) return aligned ? launch<128, true>(p, requests, n, longest, stream) : launch<128, false>(p, requests, n, longest, stream);
    return LLM_ERR_UNSUPPORTED;
}
