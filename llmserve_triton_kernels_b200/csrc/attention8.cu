// Attention over 8-bit pages (rope_kv_write8.cu), split over the cache's length and joined.
//
//   s_j = scale * 2^(ek_j) * q . k_j        out = sum_j 2^(s_j) 2^(ev_j) v_j / sum_j 2^(s_j)     (scale holds log2 e)
//
// Rows are (token, query head of the key head's group).  They ride along as the narrow side of both products: a tile of mma.sync is 16
// keys (then: 16 lanes of the output) high and 8 rows wide, so that a group of up to 8 heads wastes nothing; a CTA takes one or two
// such tiles of rows.  What bounds it is the pages' bytes, and behind them the instructions that unpack them.  Both products are in
// half precision, which holds every e4m3 number: with the lanes of a head permuted alike in q and k (a dot product does not
// notice) a thread's 16 bytes of a key are the A elements of four products once they are converted, one instruction for two; and
// since the output's lanes may come in any order, so are its bytes of four values, two by two interleaved, for the second product.
// q, its row scaled to [128, 256), loses nothing but what lies 2^-22 and more below the row's largest value.  (Products of e4m3 would
// save the conversion but for mma.sync, which converts by itself: q as two e4m3 numbers took 125 of 497 instructions a tile, q in half
// precision takes 40 fewer.)  The weights stay in half precision too: e4m3's 18 powers of two would drop the many small weights of
// a long context.  They turn from the first product's result into the second's operand by a transposition of 8 x 8 (movmatrix).
//
// A value's weight 2^(s_j + ev_j) has a running reference of its own, apart from that of 2^(s_j): what enters the half-precision product
// is the weight over that reference, which is kept 2^ABOVE below the largest of some time ago, so that the largest lies in [2^11, 2^15]
// once references have settled and every weight down to 2^-25 of the largest has all 11 bits of half precision.  A weight below that loses at
// most 2^-36 of the largest, times its value: it shows only in lanes where the largest's own value is next to nothing.  Vectors of zeros,
// which are written with a scale of one, have no part in the reference, however large their weights: they enter the weights' sum alone.
//
// Work is counted in tiles of 16 keys for one tile of rows: a step's tiles, request after request, form one list, and every CTA takes an
// equal stretch of it, wherever requests begin and end (their lengths are the device's business: a captured step is replayed at any
// lengths).  A CTA's stretch is cut into segments, one for each tile of rows that it touches; a segment that holds all keys of its
// rows writes their outputs, one that holds some leaves its sums in the call's scratch memory, and a second kernel joins those.
// Within a segment the tiles go round the CTA's warps; a warp's tiles come through a ring of its own in shared memory, and the warps meet
// once, in shared memory.  The ring is filled by TMA, swizzled so that neither keys nor values meet in a bank.  A page holds a head's keys
// side by side, and their values a fixed distance behind, so one box is a tile's keys and values (where pages hold tiles whole; two
// boxes of eight keys where they hold eights): four boxes, or copies by the threads, cost a warp some 600 cycles a tile to ask for.
//
// Cutting and joining cost 8 us and more, so short or many units of work go without: a CTA takes a tile of rows with all its keys, of two
// warps instead of eight where there are many units of few keys, whose time is a CTA's 4 us of loads that wait for one another (q and
// the page table, the pages, the warps' meeting) and not the bytes.  The host picks, from the longest context it is told.
// Heads of 128 lanes, requests of random lengths, 32 heads over 8: 32 of up to 8,191 keys 68 us, 5.2 TB/s of pages; 64 of up to 4,000 77 us,
// 4.5 TB/s; 8 of up to 4,000 19 us, of which 8 are laying out, cutting and joining.  32 heads of their own: 64 of up to 4,000 227 us, 6.0 TB/s.
// It is not the memory that bounds the first but the warps' own chains: some 390 instructions a tile of 16 keys with the 4 warps that an SM's
// quarter has registers for (500 instructions a tile took 73 us, the same pages all in the L2 5 % less).
//
// Masks: a key that no row of the tile may see, or that lies behind the request's end, is never multiplied (its 8 bits may be NaN).
// Where rows differ in what they see, NaN among the values is counted apart, so that it reaches the rows that see it alone.
#include "fp8.cuh"
#include "tma.cuh"

#include <type_traits>

namespace {

constexpr int TILE = 16, STAGES = 3;
// What it costs a CTA to begin and end a segment, in tiles (q, the first copies, the warps' meeting: some 5,000 cycles): a unit counts for so
// many tiles more than it has.  32 requests of up to 8,191 keys: 83 us with 0, 81 with 6, 79 with 12, 77 with 20, less with 28 than with 40.
constexpr int UNIT_COST = 28;
// Tiles of keys up to which a CTA takes a unit whole (8 requests of 500 keys, 8 key heads: 10.7 us instead of 12.3; of 100: 7.7 instead of 10).
constexpr int WHOLE = 32;
constexpr int JOIN_THREADS = 512;
constexpr int MAX_REQUESTS = 1024;  // of a step whose work is counted tile by tile

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
    int requests, H, KV, G, page_size, pages, window;
    int below;          // requests that bring so many tokens or more are left out (0: none)
    int* error_flag;
    int warps;          // of a CTA that takes a tile of rows with all its keys
    int ranges;         // stretches of the step's list of tiles at most; 0: a CTA takes a tile of rows with all its keys
    float scale;        // times log2 e
    float* part_sums;   // [ranges][2][ROWS][D + 4]: what a stretch holds of the rows at its beginning and at its end,
    float* part_stats;  // [ranges][2][ROWS][3]      as warps leave it to one another
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
// Over the eight lanes that hold the same row.
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// An 8 x 8 matrix of half-precision numbers, row g's elements 2 t and 2 t + 1 in lane (g, t), turned round.
__device__ __forceinline__ unsigned transpose(unsigned v) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}

// A stage of a warp's ring: a tile's keys and values in runs of RUN keys (8 or 16): [run][keys, values][RUN][D bytes], the 16-byte chunks
// of a row swizzled as TMA does it.
template <int D, int RUN>
struct Stage {
    static constexpr int BYTES = 2 * TILE * D, VALUES = RUN * D, SECOND = RUN == 8 ? 16 * D : 8 * D;  // to the values; to keys 8 .. 15
    static constexpr CUtensorMapSwizzle SWIZZLE = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    static __device__ __forceinline__ int chunk(int row, int c) { return (D == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) * 16; }
    static __device__ __forceinline__ int key(int row, int c) { return (row >> 3) * SECOND + (row & 7) * D + chunk(row, c); }
};

template <int BYTES>
__device__ __forceinline__ void copy_async(unsigned dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(dst), "l"(src) : "memory");
}

// References start below every score; a row whose weights' sum is zero has seen nothing.
constexpr float NOTHING = -3.4028234e38f;
// In powers of two: how far the values' reference is put below the largest weight, and how far a weight may then lie above that largest before
// the reference moves.  Together 15, half precision's range above one: each more of the first is a power of two more for small weights, each more of
// the second fewer meetings of the lanes.
constexpr float ABOVE = 11.f, LAG = 4.f;

// Two lanes of a row's output, columns c and c + 1 of the sums: its sum over the weights' sum; zeros for a row that saw no key.
template <int D>
__device__ __forceinline__ void finish(const Attn8Params& p, int first, int h, int rho, int c, float a, float b, float total, float y0, float y1) {
    // 2^(b - a) in two factors: beside the smallest and the largest scales of values it may leave 32 bits' exponents where the output does not
    const float f = exp2f(0.5f * (b - a)), each = total == 0.f ? 0.f : f / total;
    const int token = rho / p.G, lane = (D / 8) * ((c & 15) >> 1) + 2 * (c >> 4);
    __nv_bfloat16* at = p.out + (first + token) * p.out_stride + (long long)(h * p.G + rho - token * p.G) * D + lane;
    *reinterpret_cast<__nv_bfloat162*>(at) = __floats2bfloat162_rn(y0 * f * each, y1 * f * each);
}

// A request's share of the list: tiles of rows for every key head, and the tiles of keys that any of its rows sees.
struct Share {
    int row_tiles, first_tile, tiles;
};
template <int ROWS>
__device__ __forceinline__ Share share_of(const Attn8Params& p, int r) {
    int n = p.cu_tokens[r + 1] - p.cu_tokens[r];
    if (p.below && n >= p.below) n = 0;
    const int ctx = p.context_lens[r];
    const int end = min(ctx, p.table_width * p.page_size), begin = p.window > 0 ? max(0, ctx - n - p.window + 1) : 0;
    Share s;
    s.row_tiles = (n * p.G + ROWS - 1) / ROWS;
    s.first_tile = begin / TILE;
    s.tiles = n > 0 ? max(0, (end + TILE - 1) / TILE - s.first_tile) : 0;
    return s;
}

// Where the requests' shares begin in the list, [requests + 1], by the whole block.  Returns whether units are cut: a captured step is laid
// out for the longest context there may be, and where no request holds more than WHOLE tiles of keys by now, a unit counts as one place,
// which some CTA takes with all its keys.
template <int ROWS>
__device__ __forceinline__ bool lay_out(const Attn8Params& p, long long* begins) {
    int most = 0;
    for (int r = threadIdx.x; r < p.requests; r += blockDim.x) most = max(most, share_of<ROWS>(p, r).tiles);
    const bool cut = __syncthreads_or(most > WHOLE);
    for (int r = threadIdx.x; r < p.requests; r += blockDim.x) {
        const Share s = share_of<ROWS>(p, r);
        begins[r + 1] = s.tiles ? (long long)p.KV * s.row_tiles * (cut ? UNIT_COST + s.tiles : 1) : 0;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        long long run = 0;
        for (int r0 = 0; r0 < p.requests; r0 += 32) {
            const int r = r0 + threadIdx.x;
            long long v = r < p.requests ? begins[r + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, v, o);
                if ((int)threadIdx.x >= o) v += u;
            }
            if (r < p.requests) begins[r + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
        if (threadIdx.x == 0) begins[0] = 0;
    }
    __syncthreads();
    return cut;
}

// Stretches of a list of `total` places: no more than there are CTAs, none (but the last) shorter than a tile a warp, or than a unit.
__device__ __forceinline__ int stretches(const Attn8Params& p, long long total, bool cut) {
    return (int)max(1LL, min((long long)p.ranges, cut ? total / 8 : total));
}

// RUN: pages hold whole runs of 8 or 16 keys; 0: they do not, and the threads copy every key from its own place.
template <int D, int NT, int RUN, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (NT == 1 ? 16 : 8) / WARPS)
attention8_kernel(const Attn8Params p, const __grid_constant__ CUtensorMap map) {
    constexpr int THREADS = WARPS * 32;
    constexpr int KSTEPS = D / 32, MTILES = D / 16, ROWS = 8 * NT, PITCH = D + 4;
    using S = Stage<D, RUN ? RUN : TILE>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // the warps' rings; at a segment's end [WARPS][ROWS][PITCH] sums
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ float stats[WARPS][ROWS][3];  // largest score, largest score with the value's scale, sum of weights
    __shared__ long long begins[WARPS == 8 ? MAX_REQUESTS + 1 : 1];
    __shared__ __align__(16) unsigned char scales[WARPS][STAGES][2 * TILE];  // exponents of a stage's keys and values
    __shared__ __align__(8) unsigned long long full[WARPS][STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * STAGES * S::BYTES;
    if (RUN && lane == 0) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) tma::mbar_init(&full[warp][i], 1);
        tma::mbar_fence_init();
    }
    __syncwarp();
    int filled = 0;  // stages this warp has asked for: the barriers' phases go on from segment to segment
    pdl_wait();
    pdl_trigger();
    long long at = 0, end = 1;
    bool cut = false;
    const bool shared_out = WARPS == 8 && p.ranges;  // (stretches are CTAs of eight warps)
    if (shared_out) {
        cut = lay_out<ROWS>(p, begins);
        const long long total = begins[p.requests];
        const int count = stretches(p, total, cut);
        if ((int)blockIdx.x >= count) return;
        at = total * blockIdx.x / count;
        end = total * (blockIdx.x + 1) / count;
    }
    while (at < end) {
        // ---- the segment: request r, key head h, rows from row0 on, tiles tile_lo .. tile_hi - 1 ----
        int r, h, row0, tile_lo, tile_hi, part = -1;  // part: the place in scratch memory of a segment without all keys
        if (shared_out) {
            int lo = 0, hi = p.requests;  // the last request whose share begins at or before `at`
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (begins[mid] <= at) lo = mid; else hi = mid;
            }
            r = lo;
            const Share s = share_of<ROWS>(p, r);
            const long long within = at - begins[r];
            // a unit is UNIT_COST places without tiles, then its tiles; or one place
            const int before = cut ? UNIT_COST : 1 - s.tiles, places = before + s.tiles, unit = (int)(within / places), off = (int)(within - (long long)unit * places);
            const int to = (int)min((long long)places, off + end - at), skip = max(0, off - (cut ? UNIT_COST : 0)), take = to - before - skip;
            at += to - off;
            if (take <= 0) continue;
            h = unit / s.row_tiles;
            row0 = (unit - h * s.row_tiles) * ROWS;
            tile_lo = s.first_tile + skip;
            tile_hi = tile_lo + take;
            if (take < s.tiles) part = blockIdx.x * 2 + (skip == 0);
        } else {
            r = blockIdx.x / p.KV;
            h = blockIdx.x - r * p.KV;
            row0 = blockIdx.y * ROWS;
            const Share s = share_of<ROWS>(p, r);
            tile_lo = s.first_tile;
            tile_hi = tile_lo + s.tiles;
            at = end;
        }
        const int first = p.cu_tokens[r], n = p.cu_tokens[r + 1] - first, rows = n * p.G;
        if (row0 >= rows || (p.below && n >= p.below)) return;
        const int start = p.context_lens[r] - n;  // position of the request's first new token
        const int pos_min = start + row0 / p.G, pos_max = start + min(row0 + ROWS - 1, rows - 1) / p.G;
        // the request's tiles may reach further back or on than these rows see
        const int key_end = min(pos_max + 1, p.table_width * p.page_size);
        if (p.window > 0) tile_lo = max(tile_lo, max(0, pos_min - p.window + 1) / TILE);
        tile_hi = min(tile_hi, (key_end + TILE - 1) / TILE);
        const int mine = max(0, (tile_hi - tile_lo - warp + WARPS - 1) / WARPS);  // this warp's tiles: tile_lo + warp + i WARPS

        // q's loads go out before the ring's, whose places take a trip to the page table first
        unsigned raw[NT][KSTEPS][4];
        int own_pos[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int rho = row0 + 8 * nt + g;
            const bool live = rho < rows;
            const int token = live ? rho / p.G : 0, head = h * p.G + (live ? rho - token * p.G : 0);
            const __nv_bfloat16* src = p.q + (first + token) * p.q_stride + (long long)head * D + (D / 4) * t;
            own_pos[nt] = live ? start + token : -1;
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint2 w = live ? *reinterpret_cast<const uint2*>(src + 8 * j + 4 * e) : make_uint2(0u, 0u);
                    raw[nt][j][2 * e] = w.x;
                    raw[nt][j][2 * e + 1] = w.y;
                }
        }

        // ---- the ring ----
        const int* table = p.page_table + (long long)r * p.table_width;
        // key `j` of the request as an index over [pages, 2, KV, page_size]
        auto place = [&](int j) -> long long {
            const int at = j / p.page_size;
            const int page = min(max(table[at], 0), p.pages - 1);
            return ((long long)page * 2 * p.KV + h) * p.page_size + (j - at * p.page_size);
        };
        const long long to_values = (long long)p.KV * p.page_size;
        int run[2] = {0, 0};  // this lane's tile of the next 32: the places of its runs
        // a place behind the request's end is some place of the pool: what lies there is masked
        auto issue = [&](int i, int slot) {
            const int j0 = (tile_lo + warp + i * WARPS) * TILE;
            unsigned char* dst = ring + slot * S::BYTES;
            const unsigned scale_dst = tma::smem_addr(scales[warp][slot]);
            if constexpr (RUN != 0) {
                if ((i & 31) == 0) {
                    const int j = j0 + lane * (WARPS * TILE);
#pragma unroll
                    for (int x = 0; x < TILE / RUN; ++x) run[x] = j + 8 * x < key_end ? (int)place(j + 8 * x) : 0;
                }
                // lanes 0 to 3 ask for the exponents of the keys' and the values' eights, lane 0 for the boxes
                const int at0 = __shfl_sync(0xffffffffu, run[0], i & 31), at1 = RUN == 8 ? __shfl_sync(0xffffffffu, run[1], i & 31) : at0 + 8;
                if (lane < 4) copy_async<8>(scale_dst + 8 * lane, p.exponents + ((lane & 1) ? at1 : at0) + (lane >> 1) * to_values);
                if (lane == 0) {
                    tma::mbar_expect_tx(&full[warp][slot], S::BYTES);
                    tma::load_3d(dst, &map, 0, at0, 0, &full[warp][slot]);
                    if (RUN == 8) tma::load_3d(dst + S::SECOND, &map, 0, at1, 0, &full[warp][slot]);
                }
            } else {
                // lane l finds key l's place
                const bool is_there = j0 + (lane & 15) < key_end;
                const long long own = is_there ? place(j0 + (lane & 15)) : 0;
                const unsigned char exponent = is_there ? __ldg(p.exponents + own + (lane >> 4) * to_values) : 127;
                asm volatile("st.shared.u8 [%0], %1;\n" ::"r"(scale_dst + lane), "r"((unsigned)exponent) : "memory");
                constexpr int CHUNKS = D / 16, AT_ONCE = 32 / CHUNKS;  // of a row; rows a copy
#pragma unroll
                for (int k = 0; k < TILE / AT_ONCE; ++k) {
                    const int row = k * AT_ONCE + lane / CHUNKS, c = lane % CHUNKS;
                    const long long key = (long long)__shfl_sync(0xffffffffu, (unsigned long long)own, row);
                    const unsigned to = tma::smem_addr(dst) + S::key(row, c);
                    copy_async<16>(to, p.pool + key * D + 16 * c);
                    copy_async<16>(to + S::VALUES, p.pool + (key + to_values) * D + 16 * c);
                }
            }
        };
        for (int i = 0; i < STAGES - 1; ++i) {
            if (i < mine) issue(i, (filled + i) % STAGES);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }

        // ---- q in half precision: product i of a key takes lanes (D / 4) t + 4 i + 0 .. 3 of a row, as the keys' bytes lie ----
        unsigned qh[NT][D / 16][2];
        float factor[NT][2];  // of this thread's rows, which are 2 t and 2 t + 1 of every tile in the products' results
        int pos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned a = raw[nt][j][e] & 0x7fffu, b = (raw[nt][j][e] >> 16) & 0x7fffu;
                    top = max(top, max(a < 0x7f80u ? a : 0u, b < 0x7f80u ? b : 0u));
                }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the row's largest value to [2^7, 2^8): 2^shift, in two factors because either end may leave 32 bits' exponents
            const int shift = top ? 134 - max((int)(top >> 7), 1) : 0;
            const float f0 = __uint_as_float((unsigned)(127 + shift / 2) << 23), f1 = __uint_as_float((unsigned)(127 + shift - shift / 2) << 23);
            const float own = p.scale / f0 / f1;
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = __uint_as_float(raw[nt][j][e] << 16) * f0 * f1, b = __uint_as_float(raw[nt][j][e] & 0xffff0000u) * f0 * f1;
                    qh[nt][2 * j + (e >> 1)][e & 1] = pack_half(fmaf(a, 0.f, a), fmaf(b, 0.f, b));  // infinities become NaN
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                factor[nt][e] = __shfl_sync(0xffffffffu, own, (2 * t + e) * 4);
                pos[nt][e] = __shfl_sync(0xffffffffu, own_pos[nt], (2 * t + e) * 4);
            }
        }

        // o[nt][x]: lanes (D / 8) g + 2 x (+ 1) of the head, rows 2 t, 2 t + 1 of tile nt: [lane][row]
        float o[NT][MTILES][4], m1[NT][2], m2[NT][2], sum[NT][2];  // sum: this thread's keys alone
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int x = 0; x < MTILES; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][x][e] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) m1[nt][e] = m2[nt][e] = NOTHING, sum[nt][e] = 0.f;
        }

        // tiles that begin in here are seen whole by every row
        const int whole_from = p.window > 0 ? pos_max - p.window + 1 : 0, whole_to = min(pos_min + 1, key_end) - TILE;
        bool broken = false;
        int i0 = 0;
        for (; i0 < mine; ++i0, ++filled) {
            const int slot = filled % STAGES;
            asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory");
            if (RUN) {
                // one answer for all lanes: those that gave up would part from the others in the products.  (The vote costs 0.2 us of 68; as part of the
                // tile's other vote, below, 2.)
                broken = !__all_sync(0xffffffffu, tma::mbar_wait(&full[warp][slot], (filled / STAGES) & 1));
                if (broken) break;  // nothing more is asked for
            }
            __syncwarp();  // copies by other lanes have arrived; and everyone has read the stage that is filled next
            if (i0 + STAGES - 1 < mine) issue(i0 + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            const int j0 = (tile_lo + warp + i0 * WARPS) * TILE;
            const unsigned char* stage = ring + slot * S::BYTES;

            const auto work = [&](auto masked) {
                // ---- scores: [key g | g + 8][row 2 t | 2 t + 1] of every tile of rows ----
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
                for (int x = 0; x < D / 64; ++x) {
                    const unsigned char* at = stage + S::key(g, (D / 64) * t + x);
                    const uint4 k0 = *reinterpret_cast<const uint4*>(at), k1 = *reinterpret_cast<const uint4*>(at + S::SECOND);
                    const unsigned w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned a[4] = {half2_of((unsigned short)w0[i]), half2_of((unsigned short)w1[i]), half2_of((unsigned short)(w0[i] >> 16)),
                                               half2_of((unsigned short)(w1[i] >> 16))};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a, qh[nt][4 * x + i][0], qh[nt][4 * x + i][1]);
                    }
                }
                unsigned v[4][D / 32];  // D / 8 bytes of the values 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 2 * t + (e & 1) + 8 * (e >> 1);
                    if constexpr (D == 128) {
                        const uint4 w = *reinterpret_cast<const uint4*>(stage + S::VALUES + S::key(row, g));
                        v[e][0] = w.x, v[e][1] = w.y, v[e][2] = w.z, v[e][3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(stage + S::VALUES + S::key(row, g >> 1) + (g & 1) * 8);
                        v[e][0] = w.x, v[e][1] = w.y;
                    }
                }
                float ev[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const unsigned char* at = scales[warp][slot] + g + 8 * x;
                    const float ks = __uint_as_float((unsigned)at[0] << 23);
                    ev[x] = __uint_as_float(0x4b000000u | at[TILE]) - (8388608.f + 127.f);  // 2^23 + b has b as its lowest bits
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) s[nt][2 * x + e] *= ks * factor[nt][e];
                }
                if constexpr (decltype(masked)::value) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int j = j0 + g + 8 * x;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (j > pos[nt][e] || j >= key_end || (p.window > 0 && j <= pos[nt][e] - p.window)) s[nt][2 * x + e] = -INFINITY;
                    }
                    // a value that no row of the tile sees is nobody's
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + 2 * t + (e & 1) + 8 * (e >> 1);
                        if (j > pos_max || j >= key_end || (p.window > 0 && j <= pos_min - p.window)) {
#pragma unroll
                            for (int w = 0; w < D / 32; ++w) v[e][w] = 0u;
                        }
                    }
                    if (pos_min != pos_max) {
                        // Some row may see a key that another does not, and NaN times a weight of zero is NaN: NaN among the values is taken out and
                        // counted by a product of its own, of ones where a value is NaN and where a row sees a key.
                        unsigned any = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int w = 0; w < D / 32; ++w) any |= __vcmpeq4(v[e][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                unsigned seen[2];
#pragma unroll
                                for (int x = 0; x < 2; ++x)
                                    seen[x] = transpose((s[nt][2 * x] == -INFINITY ? 0u : 0x3c00u) | (s[nt][2 * x + 1] == -INFINITY ? 0u : 0x3c000000u));
#pragma unroll
                                for (int x = 0; x < MTILES; ++x) {
                                    unsigned bad[4];
#pragma unroll
                                    for (int q = 0; q < 4; ++q) {  // lane byte 2 x + (q & 1), keys 2 t + 8 (q >> 1) and the next
                                        const int b = 2 * x + (q & 1), e = 2 * (q >> 1);
                                        bad[q] = (((v[e][b / 4] >> (8 * (b & 3))) & 0x7fu) == 0x7fu ? 0x3c00u : 0u) |
                                                 (((v[e + 1][b / 4] >> (8 * (b & 3))) & 0x7fu) == 0x7fu ? 0x3c000000u : 0u);
                                    }
                                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_f16(c, bad, seen[0], seen[1]);
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        if (c[e] > 0.f) o[nt][x][e] = NAN;
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e)
#pragma unroll
                                for (int w = 0; w < D / 32; ++w) v[e][w] &= ~__vcmpeq4(v[e][w] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        }
                    }
                }
                // ---- weights.  The references m1 and m2 belong to maxima of some time ago: they move only when a score has left these 2^16 or 2^LAG
                // behind, which the 32-bit sums and half precision bear, so that most tiles need no meeting of the lanes ----
                unsigned pb[NT][2];
                float u[NT][4];
                bool behind = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        u[nt][e] = s[nt][e] + ev[e >> 1];
                        behind |= s[nt][e] > m1[nt][e & 1] + 16.f || u[nt][e] > m2[nt][e & 1] + (ABOVE + LAG);
                    }
                if (__any_sync(0xffffffffu, behind)) {
                    // A vector of zeros is written with a scale of one.  (To look at the values of every tile that comes here took 8 requests of up to 1,000 keys
                    // with 4 key heads of 64 lanes 8.8 us, to look where a scale is one 8.5, as without.)
                    if (__any_sync(0xffffffffu, ev[0] == 0.f || ev[1] == 0.f)) {
                        unsigned bits = 0;  // half of value lane & 15, read anew: what is seldom done holds no registers
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            const uint4 w = *reinterpret_cast<const uint4*>(stage + S::VALUES + S::key(lane & 15, (lane >> 4) * (D / 32) + c));
                            bits |= w.x | w.y | w.z | w.w;
                        }
                        unsigned some = __ballot_sync(0xffffffffu, (bits & 0x7f7f7f7fu) != 0u);
                        some |= some >> 16;  // bit j: value j is no vector of zeros
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            if (!(some >> (g + 8 * x) & 1u)) {  // (its weight might not be a number of half precision)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) u[nt][2 * x] = u[nt][2 * x + 1] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float a = fmaxf(m1[nt][e], row_max(fmaxf(s[nt][e], s[nt][2 + e])));
                            const float b = fmaxf(m2[nt][e], row_max(fmaxf(u[nt][e], u[nt][2 + e])) - ABOVE);
                            const float keep = exp2_fast(m2[nt][e] - b);
                            sum[nt][e] *= exp2_fast(m1[nt][e] - a);
                            m1[nt][e] = a;
                            m2[nt][e] = b;
#pragma unroll
                            for (int x = 0; x < MTILES; ++x) {
                                o[nt][x][e] *= keep;
                                o[nt][x][2 + e] *= keep;
                            }
                        }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sum[nt][e] += exp2_fast(s[nt][e] - m1[nt][e]) + exp2_fast(s[nt][2 + e] - m1[nt][e]);
                        u[nt][e] = exp2_fast(u[nt][e] - m2[nt][e]);
                        u[nt][2 + e] = exp2_fast(u[nt][2 + e] - m2[nt][e]);
                    }
                    pb[nt][0] = transpose(pack_half(u[nt][0], u[nt][1]));
                    pb[nt][1] = transpose(pack_half(u[nt][2], u[nt][3]));
                }
                // ---- values: tile x takes bytes 2 x and 2 x + 1 of the thread's of every key ----
#pragma unroll
                for (int x = 0; x < MTILES; ++x) {
                    unsigned a[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {  // lane bytes 2 x and 2 x + 1 of keys 2 t + 4 e and the next
                        const unsigned w = __byte_perm(v[e][x / 2], v[e + 1][x / 2], x & 1 ? 0x7362u : 0x5140u);
                        a[e] = half2_of((unsigned short)w);
                        a[e + 1] = half2_of((unsigned short)(w >> 16));
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][x], a, pb[nt][0], pb[nt][1]);
                }
            };
            // (written out twice: with the masks in the same code a tile took 57 instructions more)
            if (j0 < whole_from || j0 > whole_to)
                work(std::true_type{});
            else
                work(std::false_type{});
        }

        // ---- the warps meet, where the rings were ----
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        if (RUN && broken) {  // what is on its way (the tile that was waited for and those behind it) must land before the CTA ends
            if (lane == 0 && p.error_flag) atomicExch(p.error_flag, 1);
            for (int i = 0; i < min(STAGES - 1, mine - i0); ++i) (void)tma::mbar_wait(&full[warp][(filled + i) % STAGES], ((filled + i) / STAGES) & 1);
        }
        // the rings were written by the other proxy too, and will be: order what threads do to the same places
        if (RUN) asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        if (RUN == 0)
            __syncthreads();
        else if (__syncthreads_or(broken))
            return;  // a wait gave up: the result is void
        float* merge = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum[nt][e] += __shfl_xor_sync(0xffffffffu, sum[nt][e], x);
                const int row = 8 * nt + 2 * t + e;
                if (row0 + row >= rows) continue;
                if (g == 0) {
                    stats[warp][row][0] = m1[nt][e];
                    stats[warp][row][1] = m2[nt][e];
                    stats[warp][row][2] = sum[nt][e];
                }
                // lanes (D / 8) g + 2 x, + 1 at columns 16 x + 2 g, + 1: the warp's stores meet in no bank
                float* at = merge + ((size_t)warp * ROWS + row) * PITCH + 2 * g;
#pragma unroll
                for (int x = 0; x < MTILES; ++x) *reinterpret_cast<float2*>(at + 16 * x) = make_float2(o[nt][x][e], o[nt][x][2 + e]);
            }
        __syncthreads();
        const int live_rows = min(ROWS, rows - row0);
        for (int i = threadIdx.x; i < live_rows * (D / 2); i += THREADS) {
            const int row = i / (D / 2), c = (i - row * (D / 2)) * 2;
            float a = NOTHING, b = NOTHING;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                a = fmaxf(a, stats[w][row][0]);
                b = fmaxf(b, stats[w][row][1]);
            }
            float total = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                total += stats[w][row][2] * exp2_fast(stats[w][row][0] - a);
                const float f = exp2_fast(stats[w][row][1] - b);
                const float2 x = *reinterpret_cast<const float2*>(merge + ((size_t)w * ROWS + row) * PITCH + c);
                y0 = fmaf(x.x, f, y0);
                y1 = fmaf(x.y, f, y1);
            }
            if (part < 0) {
                finish<D>(p, first, h, row0 + row, c, a, b, total, y0, y1);
            } else {
                *reinterpret_cast<float2*>(p.part_sums + ((size_t)part * ROWS + row) * PITCH + c) = make_float2(y0, y1);
                if (c == 0) {
                    float* st = p.part_stats + ((size_t)part * ROWS + row) * 3;
                    st[0] = a;
                    st[1] = b;
                    st[2] = total;
                }
            }
        }
        if (RUN) asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncthreads();  // the rings are filled again
    }
}

// Joins what stretches left of a tile of rows that no stretch held alone: GROUPS groups of threads take every GROUPS-th stretch each.
template <int D, int NT>
__global__ void __launch_bounds__(JOIN_THREADS)
attention8_join_kernel(const Attn8Params p) {
    constexpr int ROWS = 8 * NT, PITCH = D + 4, COLS = ROWS * (D / 4), GROUPS = JOIN_THREADS / (8 * (D / 4));
    __shared__ long long begins[MAX_REQUESTS + 1];
    __shared__ float references[ROWS][2];
    __shared__ float4 sums[GROUPS][8 * (D / 4)];
    __shared__ float totals[GROUPS][ROWS];
    const int r = blockIdx.x / p.KV, h = blockIdx.x - r * p.KV, row0 = blockIdx.y * ROWS;
    // The step's arrays are older than the kernel in front, which began behind everything before it: where the parts are is worked
    // out while that one runs.
    const int first = p.cu_tokens[r], n = p.cu_tokens[r + 1] - first, rows = p.below && n >= p.below ? 0 : n * p.G, live_rows = min(ROWS, rows - row0);
    const Share share = share_of<ROWS>(p, r);
    const bool cut = lay_out<ROWS>(p, begins);
    const long long total = begins[p.requests], from = begins[r] + (long long)(h * share.row_tiles + blockIdx.y) * (UNIT_COST + share.tiles) + UNIT_COST;
    int c0 = 0, c1 = -1;  // the stretches that hold a tile of these rows
    if (live_rows > 0 && share.tiles && cut) {
        const int count = stretches(p, total, cut);
        c0 = (int)(from * count / total);
        while (total * (c0 + 1) / count <= from) ++c0;
        c1 = c0;
        while (total * (c1 + 1) / count < from + share.tiles) ++c1;
    }
    pdl_wait();
    pdl_trigger();
    if (live_rows <= 0 || (share.tiles && (!cut || c0 == c1))) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto place = [&](int k, int row) { return (size_t)(2 * k + (k == c0)) * ROWS + row; };
    for (int row = warp; row < live_rows; row += JOIN_THREADS / 32) {
        float a = NOTHING, b = NOTHING;
        for (int k = c0 + lane; k <= c1; k += 32) {
            a = fmaxf(a, p.part_stats[place(k, row) * 3]);
            b = fmaxf(b, p.part_stats[place(k, row) * 3 + 1]);
        }
        a = warp_max(a);
        b = warp_max(b);
        if (lane == 0) {
            references[row][0] = a;
            references[row][1] = b;
        }
    }
    __syncthreads();
    const int group = threadIdx.x / (8 * (D / 4)), col = threadIdx.x - group * (8 * (D / 4));
    for (int i0 = 0; i0 < COLS; i0 += 8 * (D / 4)) {
        const int row = (i0 + col) / (D / 4), c = (i0 + col - row * (D / 4)) * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        float weights = 0.f;
        if (row < live_rows) {
            const float a = references[row][0], b = references[row][1];
#pragma unroll 4
            for (int k = c0 + group; k <= c1; k += GROUPS) {
                const size_t at = place(k, row);
                const float s0 = p.part_stats[at * 3], s1 = p.part_stats[at * 3 + 1], s2 = p.part_stats[at * 3 + 2];
                const float4 x = *reinterpret_cast<const float4*>(p.part_sums + at * PITCH + c);
                const float f = exp2_fast(s1 - b);
                weights += s2 * exp2_fast(s0 - a);
                y.x = fmaf(x.x, f, y.x);
                y.y = fmaf(x.y, f, y.y);
                y.z = fmaf(x.z, f, y.z);
                y.w = fmaf(x.w, f, y.w);
            }
            sums[group][col] = y;
            if (c == 0) totals[group][row] = weights;
        }
        __syncthreads();
        if (group == 0 && row < live_rows) {
            weights = totals[0][row];
#pragma unroll
            for (int k = 1; k < GROUPS; ++k) {
                const float4 x = sums[k][col];
                y.x += x.x;
                y.y += x.y;
                y.z += x.z;
                y.w += x.w;
                weights += totals[k][row];
            }
            finish<D>(p, first, h, row0 + row, c, references[row][0], references[row][1], weights, y.x, y.y);
            finish<D>(p, first, h, row0 + row, c + 2, references[row][0], references[row][1], weights, y.z, y.w);
        }
        __syncthreads();
    }
}

template <int D, int NT, int RUN, int WARPS>
int launch_warps(const Attn8Params& p, int longest, cudaStream_t stream) {
    constexpr size_t ring = (size_t)WARPS * STAGES * 2 * TILE * D, merge = (size_t)WARPS * 8 * NT * (D + 4) * sizeof(float);
    constexpr size_t smem = (ring > merge ? ring : merge) + 1024;
    const long long row_tiles = ((long long)longest * p.G + 8 * NT - 1) / (8 * NT), pairs = (long long)p.requests * p.KV;
    if (row_tiles > 65535 || pairs > 0x7fffffffLL) return LLM_ERR_UNSUPPORTED;
    auto kernel = attention8_kernel<D, NT, RUN, WARPS>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // of the current device
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map = {};
    const uint64_t values = (uint64_t)p.KV * p.page_size, keys = p.pages * 2 * values;  // a key's value lies so many places behind it
    if (RUN && !tma::make_map_2d_u8_twice(&map, p.pool, keys - values, D, D, values * D, RUN, D, Stage<D, RUN ? RUN : TILE>::SWIZZLE))
        return LLM_ERR_UNSUPPORTED;
    const dim3 units((unsigned)pairs, (unsigned)row_tiles);
    const int code = launch_pdl(kernel, p.ranges ? dim3(p.ranges) : units, dim3(WARPS * 32), smem, stream, p, map);
    if (code || !p.ranges) return code;
    return launch_pdl(attention8_join_kernel<D, NT>, units, dim3(JOIN_THREADS), 0, stream, p);
}

template <int D, int NT, int RUN>
int launch(const Attn8Params& p, int longest, cudaStream_t stream) {
    return p.warps == 2 && !p.ranges ? launch_warps<D, NT, RUN, 2>(p, longest, stream) : launch_warps<D, NT, RUN, 8>(p, longest, stream);
}

}  // namespace

// q rows [n, >= H D] bfloat16 (row stride a multiple of 4, 8-byte aligned); pool and exponents as rope_kv_write8.cu leaves them, the pool on 16
// bytes, the exponents anywhere; request r's new tokens are rows cu_tokens[r] .. cu_tokens[r + 1] - 1, the last one at position context_lens[r] - 1; `longest`: the
// most tokens a request brings; with `below` requests that bring so many or more are left out, and their
// rows of out as they are.  out [n, H D].  window 0: none.  ranges: CTAs of eight warps that share the step's keys evenly, with scratch
// memory of ranges * 2 * R * (D + 7) floats on 16 bytes, R the rows of a tile (8 where the longest request has no more, else 16), at most 1,024
// requests; 0: a CTA of `warps` (2 or 8) for each key head and tile of rows.  D 64 or 128.
LLM_EXPORT int llm_attention8(const void* q, long long q_stride, void* out, long long out_stride, const void* pool, const void* exponents,
                              const int* page_table, int table_width, const int* cu_tokens, const int* context_lens, int requests, int n,
                              int longest, int below, int H, int KV, int D, int page_size, int pages, int window, float scale, int warps, int ranges,
                              float* scratch, int* error_flag, cudaStream_t stream) {
    if (n <= 0 || requests <= 0) return 0;
    if (H <= 0 || KV <= 0 || H % KV || page_size <= 0 || pages <= 0 || table_width <= 0 || longest <= 0 || (warps != 2 && warps != 8) || ranges < 0 || window < 0 ||
        (ranges && (!scratch || requests > MAX_REQUESTS || ((uintptr_t)scratch & 15))) || (q_stride & 3) || ((uintptr_t)q & 7) ||
        (out_stride & 3) || ((uintptr_t)out & 7) || ((uintptr_t)pool & 15) ||
        (long long)table_width * page_size > 0x7fff0000)
        return LLM_ERR_BAD_ARGUMENT;
    const int rows = (long long)longest * (H / KV) <= 8 ? 8 : 16;
    Attn8Params p = {(const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride, (const unsigned char*)pool, (const unsigned char*)exponents,
                     page_table, table_width, cu_tokens, context_lens, requests, H, KV, H / KV, page_size, pages, window, below, error_flag, warps, ranges,
                     scale * 1.4426950408889634f, scratch, ranges ? scratch + (size_t)ranges * 2 * rows * (D + 4) : nullptr};
    // a tensor map's rows are counted in 32 bits, and runs' exponents are copied eight at a time (a cache's planes start on 16 bytes where pages
    // hold runs, anywhere where they do not)
    const int run = (long long)pages * 2 * KV * page_size > 0x7fffffffLL || ((uintptr_t)exponents & 7) ? 0 : page_size % 16 == 0 ? 16 : page_size % 8 == 0 ? 8 : 0;
#define ATTENTION8(D_, NT_) \
    (run == 16 ? launch<D_, NT_, 16>(p, longest, stream) : run == 8 ? launch<D_, NT_, 8>(p, longest, stream) : launch<D_, NT_, 0>(p, longest, stream))
    if (D == 64) return rows == 8 ? ATTENTION8(64, 1) : ATTENTION8(64, 2);
    if (D == 128) return rows == 8 ? ATTENTION8(128, 1) : ATTENTION8(128, 2);
#undef ATTENTION8
    return LLM_ERR_UNSUPPORTED;
}
