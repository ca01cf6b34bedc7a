// block_product.hip -- the product of two matrices in 8 bits with a scale for each block of 128 (blocks.hip), fused with
// add_difference into a base key.
#include <type_traits>
#include "blocks.h"

namespace {

// out[m][n] = base[m][n] + alpha * sum over the blocks kb of sa[m][kb] sb[n][kb] * (sum over the block's k of a[m][k] b[n][k]),
// on v_mfma_scale_f32_16x16x128_f8f6f4: one instruction takes a whole block of 128 of 16 rows of each side and, with
// power-of-two scales, the two scales of every row as well, so they cost nothing.  With float32 scales the block's sum comes out of the
// matrix unit by itself, is multiplied by b's scale and added with one fma by a's: one after the other, because sa * sb can leave
// float32's range where what it multiplies is 0 or brings it back.  Sums are float32.
//
// What the 8-bit matrix instructions lose (all of them; measured with single products): the products of 8 neighbouring k are aligned to
// the largest, and what lies under 2^-13 of it is cut off; the groups are then added in float32.  That is 1.5e-5 of a result (2-norm, normal
// codes), 1/14 of what rounding to float16 loses and 1/110 of bfloat16's, so results of 16 bits are made this way: about 1 % of bfloat16
// results are the neighbour of the nearest number, and the error after the rounding is the rounding's (1.658e-3 at 8192 x 10240 x 1280, either
// way).  A float32 result would show it: there the codes are turned into bfloat16, which holds each exactly, and multiplied on
// v_mfma_f32_16x16x32_bf16, which adds in float32 (7e-8 to 1.2e-7 measured) at half the rate.
//
// b's rows are the instruction's A operand (accumulator rows) and a's rows its B operand (accumulator columns): lane l holds 4
// accumulators of output row m = l % 16.  b's rows are dealt to the fragments so that a lane's accumulators of 2 fragments are 8
// CONTIGUOUS columns and the 4 lanes of an output row write 64 bytes (16-bit results) side by side: row r of fragment f is column
// 32 (f / 2) + 8 (r / 4) + 4 (f % 2) + r % 4 of the wave's 64.
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char lds_byte;

struct ProductParams {
    const uint8_t *a; int64_t a_pitch; const void *sa; int64_t sa_pitch; int a_tile;
    const uint8_t *b; int64_t b_pitch; const void *sb; int64_t sb_pitch; int b_tile;
    const void *base; void *out;
    int64_t m, n, k;
    int base_dt, out_dt;
    float alpha;
    uint32_t *flags;
    int tiles_m, tiles_n;
    int64_t ld;                        // the large kernel: elements from one row of out and base to the next
    int splits;                        // and parts of k, each with a result of its own, m * ld float32 behind the one before
    int aligned;                       // and whether rows are whole 16 bytes that start at such (WHOLE)
};

// global -> LDS: lane l's 16 bytes at base + off go to dst + 16 l (dst wave-uniform).  Inline assembly because the compiler cannot tell
// which LDS bytes the builtin form writes and would wait for all of them in front of every LDS read; the kernels wait with counted
// s_waitcnt vmcnt themselves.  M0 is the compiler's and is put back.
__device__ __forceinline__ void dma4(const uint8_t *base, uint32_t o0, uint32_t o1, uint32_t o2, uint32_t o3, uint32_t dst) {
    unsigned keep;
    const uint32_t d1 = dst + 1024u, d2 = dst + 2048u, d3 = dst + 3072u;
    asm volatile("s_mov_b32 %0, m0\n\t"
                 "s_mov_b32 m0, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\t"
                 "s_mov_b32 m0, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %5\n\t"
                 "s_mov_b32 m0, %8\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5\n\t"
                 "s_mov_b32 m0, %9\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %5\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(base), "s"(dst), "s"(d1), "s"(d2), "s"(d3) : "memory");
}
__device__ __forceinline__ void wait_vm0() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// 16-byte slot of a row's 128 bytes in LDS.  A fragment's lane (g, r) = (l / 16, l % 16) reads parts g and g + 4 of row r -- any dealing of k
// to the lanes does, if both sides have the same.  Row r's part c lies in slot c ^ (r / 2): measured, the four parts g side by side and 8
// different slots for the rows of one parity make a 1-KiB read take 4 cycles; parts 2 g and 2 g + 1 instead, 8.
// a's fragments are 16 consecutive rows; b's are rows 8 (r / 4) + r % 4 (+ 4, + 32) and get the same slots for the same r.
__device__ __forceinline__ int swz_a(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int swz_b(int row) { return ((row >> 1) & 1) | ((row >> 2) & 6); }
// first row of b's fragment f, and of lane r's 8 columns, in a wave's 64
__device__ __forceinline__ constexpr int b_row(int f) { return 32 * (f >> 1) + 4 * (f & 1); }

__device__ __forceinline__ i32x8 join(u32x4 lo, u32x4 hi) {
    return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}
// the first n of 16 bytes
__device__ __forceinline__ u32x4 first_bytes(u32x4 w, int n) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int left = n - 4 * j;
        w[j] = left >= 4 ? w[j] : left <= 0 ? 0u : (w[j] & ((1u << (8 * left)) - 1u));
    }
    return w;
}

// a block's sums from codes as bfloat16: a quarter of the lane's 32 codes an instruction
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 codes_to_bf16(int lo, int hi, float scale = 1.0f) {       // scale: a power of two
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// (power-of-two scales go into the conversion: code * 2^e is a bfloat16)
__device__ __forceinline__ f32x4v exact_block(i32x8 a, i32x8 b, f32x4v c, float a_scale = 1.0f, float b_scale = 1.0f) {
#pragma unroll
    for (int q = 0; q < 4; q++)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_to_bf16(a[2 * q], a[2 * q + 1], a_scale), codes_to_bf16(b[2 * q], b[2 * q + 1], b_scale), c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// the larger magnitude, NaN if one is (gfx950's v_maximum3_f32), and the flags of results of which `top` is the largest
__device__ __forceinline__ float larger(float top, float x) { return __builtin_elementwise_maximum(top, fabsf(x)); }
__device__ __forceinline__ void report(uint32_t *flags, float poison_in, float top, int out_dt) {
    const bool over = !(top < stored_as_inf(out_dt)), in = top != top || poison_in != 0.0f;
    if (flags && (in || over)) atomicOr(flags, (in ? MECHA_FLAG_INPUT_NONFINITE : 0u) | (over ? MECHA_FLAG_OUTPUT_NONFINITE : 0u));
}

// 8 contiguous columns of one output row, of any base and alignment: base + alpha * acc.  Finite checks: fma(x, 0, poison) stays 0
// while every x is finite; results by their largest magnitude or NaN.
template <int OUT_DT, bool VEC>
__device__ __forceinline__ void store_any8(const ProductParams &p, int64_t m, int64_t n, const float (&acc)[8]) {
    if (m >= p.m || n >= p.n) return;
    const int64_t i = m * p.n + n;
    float r[8], b[8], poison_in = 0.0f, top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = 0.0f;
    const int left = p.n - n < 8 ? (int)(p.n - n) : 8;
    if (p.base) {
        const int dt = p.base_dt;
        if constexpr (VEC) {
            if (dt == MECHA_F32) load8<MECHA_F32>(p.base, i, b);
            else if (dt == MECHA_F16) load8<MECHA_F16>(p.base, i, b);
            else load8<MECHA_BF16>(p.base, i, b);
        } else if (dt == MECHA_F32) {
            const float *at = static_cast<const float *>(p.base) + i;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int l = left - 4 * h;
                const u32x4 w = l >= 4 ? *reinterpret_cast<const u32x4_any *>(at + 4 * h) : l > 0 ? load_part(at + 4 * h, 4 * l) : u32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; j++) b[4 * h + j] = __uint_as_float(w[j]);
            }
        } else {
            const uint16_t *at = static_cast<const uint16_t *>(p.base) + i;
            const u32x4 w = left == 8 ? *reinterpret_cast<const u32x4_any *>(at) : load_part(at, 2 * left);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t half = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
                b[j] = dt == MECHA_BF16 ? bf16_bits_to_f32(half) : f16_bits_to_f32(half);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        r[j] = p.base ? __builtin_fmaf(acc[j], p.alpha, b[j]) : acc[j] * p.alpha;
        if (n + j < p.n) {
            poison_in = __builtin_fmaf(b[j], 0.0f, poison_in);
            top = larger(top, r[j]);
        }
    }
    if constexpr (VEC) store8<OUT_DT>(p.out, i, r);
    else if constexpr (OUT_DT == MECHA_F32) {
        float *const at = static_cast<float *>(p.out) + i;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const u32x4 w = {__float_as_uint(r[4 * h]), __float_as_uint(r[4 * h + 1]), __float_as_uint(r[4 * h + 2]), __float_as_uint(r[4 * h + 3])};
            const int l = left - 4 * h;
            if (l >= 4) *reinterpret_cast<u32x4_any *>(at + 4 * h) = w;
            else if (l > 0) store_part(at + 4 * h, w, 4 * l);
        }
    } else {
        uint16_t *const at = static_cast<uint16_t *>(p.out) + i;
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = OUT_DT == MECHA_BF16 ? pack_bf16(r[2 * j], r[2 * j + 1]) : pack_f16(r[2 * j], r[2 * j + 1]);
        if (left == 8) *reinterpret_cast<u32x4_any *>(at) = w;
        else store_part(at, w, 2 * left);
    }
    report(p.flags, poison_in, top, OUT_DT);
}

// Scales of a tile's 128 rows, CH words each: four blocks a word for the matrix unit, else a block's float, or its exponent where a float has it.
constexpr int CH = 16;
enum : int { HW_SCALES = 0, F32_SCALES = 1, EXACT_F32 = 2, EXACT_E8M0 = 3 };   // how a kernel multiplies and what its scales are
template <int MODE>
__device__ __forceinline__ void fill_scales(uint32_t (*to)[128], const void *s, int64_t pitch, int tile, int64_t row0, int64_t rows, int64_t kb0, int64_t n_kb) {
    for (int i = threadIdx.x; i < CH * 128; i += MECHA_BLOCK) {
        const int r = i & 127, w = i >> 7;
        int64_t row = row0 + r;
        if (row >= rows) row = rows - 1;
        if (tile) row /= SCALE_BLOCK;
        uint32_t v = 0;
        if constexpr (MODE == HW_SCALES) {
            const uint8_t *at = static_cast<const uint8_t *>(s) + row * pitch;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t kb = kb0 + 4 * w + j;
                if (kb < n_kb) v |= (uint32_t)at[kb] << (8 * j);
            }
        } else {
            const int64_t kb = kb0 + w;
            if (kb < n_kb) {
                if constexpr (MODE == EXACT_E8M0) v = (uint32_t)static_cast<const uint8_t *>(s)[row * pitch + kb] << 23;
                else v = __float_as_uint(static_cast<const float *>(s)[row * pitch + kb]);
            }
        }
        to[w][r] = v;
    }
}

// 128 x 128 outputs, 4 waves of 64 x 64; a K step is one block of 128, two stages of 32 KiB in LDS, the next one in flight while
// this one is multiplied; two workgroups a CU.  For a base of another type than the result's, for 3 blocks of k
// at most, and where its smaller tiles fill the chip better.  Bound by the wait for each step's 32 KiB, 0.9 us a step (1.6 for float32 results).
template <int MODE, int OUT_DT, bool VEC>
__global__ __launch_bounds__(MECHA_BLOCK) void product_kernel(ProductParams p) {
    __shared__ __attribute__((aligned(1024))) uint8_t stage[2][2][128 * 128];     // [stage][a, b][row][128]
    __shared__ __attribute__((aligned(16))) uint32_t s_a[CH][128], s_b[CH][128];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int tile_m = blockIdx.x % p.tiles_m, tile_n = blockIdx.x / p.tiles_m;
    const int64_t m0 = (int64_t)tile_m * 128, n0 = (int64_t)tile_n * 128;
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int64_t n_kb = (p.k + SCALE_BLOCK - 1) / SCALE_BLOCK;
    const int tail = (int)(p.k - (n_kb - 1) * SCALE_BLOCK);                       // k's in the last block

    // DMA: piece 4 wave + i of each side = 8 rows; rows behind the last one read the last one
    uint32_t oa[4], ob[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = 8 * (4 * wave + i) + (lane >> 3), slot = lane & 7;
        int64_t ra = p.m - 1 - m0, rb = p.n - 1 - n0;
        ra = row < ra ? row : ra;
        rb = row < rb ? row : rb;
        oa[i] = (uint32_t)(ra * p.a_pitch) + 16u * (uint32_t)(slot ^ swz_a(row));
        ob[i] = (uint32_t)(rb * p.b_pitch) + 16u * (uint32_t)(slot ^ swz_b(row));
    }
    const uint8_t *ga = p.a + m0 * p.a_pitch, *gb = p.b + n0 * p.b_pitch;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_byte *)&stage[0][0][0]) + (uint32_t)wave * 4096u;
    auto issue = [&](int64_t kb) {
        const uint32_t dst = lds0 + (uint32_t)(kb & 1) * 32768u;
        dma4(ga + kb * SCALE_BLOCK, oa[0], oa[1], oa[2], oa[3], dst);
        dma4(gb + kb * SCALE_BLOCK, ob[0], ob[1], ob[2], ob[3], dst + 16384u);
    };
    f32x4v acc[4][4];                                                             // [a fragment][b fragment]
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < 4; f++) acc[i][f] = f32x4v{0, 0, 0, 0};

    auto step = [&](int64_t kb, bool last) {
        const uint8_t *la = &stage[kb & 1][0][0], *lb = &stage[kb & 1][1][0];
        i32x8 fa[4], fb[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int ra = wm + 16 * i + r, rb = wn + b_row(i) + 8 * (r >> 2) + (r & 3);
            u32x4 a0 = *reinterpret_cast<const u32x4 *>(la + ra * 128 + 16 * (g ^ swz_a(ra)));
            u32x4 a1 = *reinterpret_cast<const u32x4 *>(la + ra * 128 + 16 * ((g + 4) ^ swz_a(ra)));
            u32x4 b0 = *reinterpret_cast<const u32x4 *>(lb + rb * 128 + 16 * (g ^ swz_b(rb)));
            u32x4 b1 = *reinterpret_cast<const u32x4 *>(lb + rb * 128 + 16 * ((g + 4) ^ swz_b(rb)));
            if (last) {                                                           // bytes behind column k are not the matrix's
                a0 = first_bytes(a0, tail - 16 * g); a1 = first_bytes(a1, tail - 64 - 16 * g);
                b0 = first_bytes(b0, tail - 16 * g); b1 = first_bytes(b1, tail - 64 - 16 * g);
            }
            fa[i] = join(a0, a1);
            fb[i] = join(b0, b1);
        }
        if constexpr (MODE == HW_SCALES) {
            const int w = (int)(kb >> 2) & (CH - 1), sh = 8 * (int)(kb & 3);
            uint32_t ka[4], kbs[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ka[i] = s_a[w][wm + 16 * i + r] >> sh;
                kbs[i] = s_b[w][wn + b_row(i) + 8 * (r >> 2) + (r & 3)] >> sh;
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int f = 0; f < 4; f++)
                    acc[i][f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa[i], acc[i][f], 0, 0, 0, (int)kbs[f], 0, (int)ka[i]);
        } else if constexpr (MODE == EXACT_E8M0) {
            const int w = (int)kb & (CH - 1);
            float ka[4], kbs[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ka[i] = __uint_as_float(s_a[w][wm + 16 * i + r]);
                kbs[i] = __uint_as_float(s_b[w][wn + b_row(i) + 8 * (r >> 2) + (r & 3)]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int f = 0; f < 4; f++) acc[i][f] = exact_block(fb[f], fa[i], acc[i][f], kbs[f], ka[i]);
        } else {
            const int w = (int)kb & (CH - 1);
            float sa[4];
            f32x4v sb[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sa[i] = __uint_as_float(s_a[w][wm + 16 * i + r]);
                sb[i] = *reinterpret_cast<const f32x4v *>(&s_b[w][wn + b_row(i) + 8 * g]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    f32x4v d = {0, 0, 0, 0};
                    if constexpr (MODE == F32_SCALES) d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa[i], d, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
                    else d = exact_block(fb[f], fa[i], d);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][f][e] = __builtin_fmaf(d[e] * sb[f][e], sa[i], acc[i][f][e]);
                }
        }
    };

    constexpr int PER = MODE == HW_SCALES ? 4 * CH : CH;                                       // blocks whose scales are in LDS
    if (n_kb > 0) issue(0);
    for (int64_t kb = 0; kb < n_kb; kb++) {
        if (kb % PER == 0) {
            __syncthreads();                                                      // the last chunk's scales have been read
            fill_scales<MODE>(s_a, p.sa, p.sa_pitch, p.a_tile, m0, p.m, kb, n_kb);
            fill_scales<MODE>(s_b, p.sb, p.sb_pitch, p.b_tile, n0, p.n, kb, n_kb);
        }
        wait_vm0();                                                               // this wave's part of stage kb has landed
        __syncthreads();                                                          // everyone's has, and stage kb - 1 has been read
        if (kb + 1 < n_kb) issue(kb + 1);
        step(kb, kb + 1 == n_kb && tail < SCALE_BLOCK);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float row[8];
#pragma unroll
            for (int f = 0; f < 2; f++)
#pragma unroll
                for (int e = 0; e < 4; e++) row[4 * f + e] = acc[i][2 * h + f][e];
            store_any8<OUT_DT, VEC>(p, m0 + wm + 16 * i + r, n0 + wn + 32 * h + 8 * g, row);
        }
}

// ---------------------------------------------------------------------------------------------------- small products
// 16 AI x 16 BI outputs by 8 waves that share out the blocks of k: a wave's codes go from memory straight into its registers, all of
// them in flight at once, and the 8 partial sums meet in LDS, added in the order of the waves.  For results of few tiles, down to one
// row: what counts there is one trip to memory, and that every CU has a piece of b.  2 x 1280 x 2816 4.8 us, of which a launch and two dependent
// trips to memory are about 4 (through LDS in 128 x 128 tiles 21), 154 x 640 x 2048 with float32 scales 7.2.
constexpr int DIRECT_WAVES = 8, DIRECT_THREADS = 64 * DIRECT_WAVES;

template <int MODE, int AI, int BI>
__global__ __launch_bounds__(DIRECT_THREADS, 2) void product_direct_kernel(ProductParams p) {
    constexpr int TM = 16 * AI, TN = 16 * BI, LINE = TN + 4;                      // floats of a line in LDS
    constexpr bool EXACT = MODE == EXACT_F32 || MODE == EXACT_E8M0;
    extern __shared__ __attribute__((aligned(16))) float sums[];                  // [wave][row][LINE]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int64_t m0 = (int64_t)(blockIdx.x % (uint32_t)p.tiles_m) * TM, n0 = (int64_t)(blockIdx.x / (uint32_t)p.tiles_m) * TN;
    const int n_kb = (int)((p.k + SCALE_BLOCK - 1) / SCALE_BLOCK);
    const int tail = (int)(p.k - (int64_t)(n_kb - 1) * SCALE_BLOCK);

    // rows behind the last one read the last one
    const uint8_t *a[AI], *b[BI];
    int64_t as[AI], bs[BI];                                                       // first scale of this lane's row
#pragma unroll
    for (int i = 0; i < AI; i++) {
        int64_t row = m0 + 16 * i + r;
        row = row < p.m ? row : p.m - 1;
        a[i] = p.a + row * p.a_pitch + 16 * g;
        as[i] = (p.a_tile ? row / SCALE_BLOCK : row) * p.sa_pitch;
    }
#pragma unroll
    for (int f = 0; f < BI; f++) {
        int64_t row = n0 + 16 * f + r;
        row = row < p.n ? row : p.n - 1;
        b[f] = p.b + row * p.b_pitch + 16 * g;
        bs[f] = (p.b_tile ? row / SCALE_BLOCK : row) * p.sb_pitch;
    }
    // float32 scales of b belong to the accumulators' rows, 4 g + e of a fragment
    int64_t bse[BI][4];
    if constexpr (MODE == F32_SCALES || MODE == EXACT_F32) {
#pragma unroll
        for (int f = 0; f < BI; f++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                int64_t row = n0 + 16 * f + 4 * g + e;
                row = row < p.n ? row : p.n - 1;
                bse[f][e] = (p.b_tile ? row / SCALE_BLOCK : row) * p.sb_pitch;
            }
    }
    f32x4v acc[AI][BI];
#pragma unroll
    for (int i = 0; i < AI; i++)
#pragma unroll
        for (int f = 0; f < BI; f++) acc[i][f] = f32x4v{0, 0, 0, 0};

    struct Step { i32x8 a[AI], b[BI]; uint32_t sa[AI], sb[BI]; f32x4v sbe[BI]; };
    auto load = [&](int kb, Step &s) {
        const int64_t at = (int64_t)kb * SCALE_BLOCK;
#pragma unroll
        for (int f = 0; f < BI; f++) s.b[f] = join(*reinterpret_cast<const u32x4 *>(b[f] + at), *reinterpret_cast<const u32x4 *>(b[f] + at + 64));
#pragma unroll
        for (int i = 0; i < AI; i++) s.a[i] = join(*reinterpret_cast<const u32x4 *>(a[i] + at), *reinterpret_cast<const u32x4 *>(a[i] + at + 64));
        if constexpr (MODE == HW_SCALES || MODE == EXACT_E8M0) {
#pragma unroll
            for (int i = 0; i < AI; i++) s.sa[i] = static_cast<const uint8_t *>(p.sa)[as[i] + kb];
#pragma unroll
            for (int f = 0; f < BI; f++) s.sb[f] = static_cast<const uint8_t *>(p.sb)[bs[f] + kb];
        } else {
#pragma unroll
            for (int i = 0; i < AI; i++) s.sa[i] = static_cast<const uint32_t *>(p.sa)[as[i] + kb];
#pragma unroll
            for (int f = 0; f < BI; f++)
#pragma unroll
                for (int e = 0; e < 4; e++) s.sbe[f][e] = static_cast<const float *>(p.sb)[bse[f][e] + kb];
        }
    };
    auto cut = [&](i32x8 &v) {                                                    // bytes behind column k are not the matrix's
        const u32x4 lo = first_bytes(u32x4{(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]}, tail - 16 * g);
        const u32x4 hi = first_bytes(u32x4{(uint32_t)v[4], (uint32_t)v[5], (uint32_t)v[6], (uint32_t)v[7]}, tail - 64 - 16 * g);
        v = join(lo, hi);
    };
    auto multiply = [&](int kb, Step &s) {
        if (kb + 1 == n_kb && tail < SCALE_BLOCK) {
#pragma unroll
            for (int i = 0; i < AI; i++) cut(s.a[i]);
#pragma unroll
            for (int f = 0; f < BI; f++) cut(s.b[f]);
        }
        if constexpr (MODE == HW_SCALES) {
#pragma unroll
            for (int i = 0; i < AI; i++)
#pragma unroll
                for (int f = 0; f < BI; f++) acc[i][f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(s.b[f], s.a[i], acc[i][f], 0, 0, 0, (int)s.sb[f], 0, (int)s.sa[i]);
        } else if constexpr (MODE == EXACT_E8M0) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                bf16x8 bq[BI];
#pragma unroll
                for (int f = 0; f < BI; f++) bq[f] = codes_to_bf16(s.b[f][2 * q], s.b[f][2 * q + 1], __uint_as_float(s.sb[f] << 23));
#pragma unroll
                for (int i = 0; i < AI; i++) {
                    const bf16x8 aq = codes_to_bf16(s.a[i][2 * q], s.a[i][2 * q + 1], __uint_as_float(s.sa[i] << 23));
#pragma unroll
                    for (int f = 0; f < BI; f++) acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bq[f], aq, acc[i][f], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < AI; i++)
#pragma unroll
                for (int f = 0; f < BI; f++) {
                    f32x4v d = {0, 0, 0, 0};
                    if constexpr (EXACT) d = exact_block(s.b[f], s.a[i], d);
                    else d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(s.b[f], s.a[i], d, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][f][e] = __builtin_fmaf(d[e] * s.sbe[f][e], __uint_as_float(s.sa[i]), acc[i][f][e]);
                }
        }
    };
    // two steps in flight
    Step s0, s1;
    int kb = wave;
    if (kb < n_kb) load(kb, s0);
    while (kb < n_kb) {
        if (kb + DIRECT_WAVES < n_kb) load(kb + DIRECT_WAVES, s1);
        multiply(kb, s0);
        kb += DIRECT_WAVES;
        if (kb >= n_kb) break;
        if (kb + DIRECT_WAVES < n_kb) load(kb + DIRECT_WAVES, s0);
        multiply(kb, s1);
        kb += DIRECT_WAVES;
    }
#pragma unroll
    for (int i = 0; i < AI; i++)
#pragma unroll
        for (int f = 0; f < BI; f++) *reinterpret_cast<f32x4v *>(&sums[(wave * TM + 16 * i + r) * LINE + 16 * f + 4 * g]) = acc[i][f];
    __syncthreads();
    // 4 columns a thread
    const int used = n_kb < DIRECT_WAVES ? n_kb : DIRECT_WAVES;
    for (int x = t; x < TM * BI * 4; x += DIRECT_THREADS) {
        const int row = x / (BI * 4), col = 4 * (x - row * (BI * 4));
        const int64_t m = m0 + row, n = n0 + col, at = m * p.n + n;
        if (m >= p.m || n >= p.n) continue;
        const bool vec = n + 4 <= p.n;
        f32x4v sum = *reinterpret_cast<const f32x4v *>(&sums[row * LINE + col]);
        for (int w = 1; w < used; w++) {
            const f32x4v v = *reinterpret_cast<const f32x4v *>(&sums[(w * TM + row) * LINE + col]);
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += v[e];
        }
        float base[4] = {0, 0, 0, 0}, out[4];
        if (p.base) {
            if (vec && p.base_dt == MECHA_F32) {
                const u32x4 v = *reinterpret_cast<const u32x4_any *>(static_cast<const float *>(p.base) + at);
#pragma unroll
                for (int e = 0; e < 4; e++) base[e] = __uint_as_float(v[e]);
            } else if (vec) {
                const u32x2 v = *reinterpret_cast<const u32x2_any *>(static_cast<const uint16_t *>(p.base) + at);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t half = e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu;
                    base[e] = p.base_dt == MECHA_BF16 ? bf16_bits_to_f32(half) : f16_bits_to_f32(half);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (n + e < p.n) base[e] = p.base_dt == MECHA_F32 ? load1<MECHA_F32>(p.base, at + e) : p.base_dt == MECHA_F16 ? load1<MECHA_F16>(p.base, at + e) : load1<MECHA_BF16>(p.base, at + e);
            }
        }
        float top = 0.0f, poison_in = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            out[e] = p.base ? __builtin_fmaf(sum[e], p.alpha, base[e]) : sum[e] * p.alpha;
            if (n + e < p.n) {
                top = larger(top, out[e]);
                poison_in = __builtin_fmaf(base[e], 0.0f, poison_in);
            }
        }
        if (vec && p.out_dt == MECHA_F32)
            *reinterpret_cast<u32x4_any *>(static_cast<float *>(p.out) + at) = u32x4{__float_as_uint(out[0]), __float_as_uint(out[1]), __float_as_uint(out[2]), __float_as_uint(out[3])};
        else if (vec)
            *reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(p.out) + at) =
                p.out_dt == MECHA_BF16 ? u32x2{pack_bf16(out[0], out[1]), pack_bf16(out[2], out[3])} : u32x2{pack_f16(out[0], out[1]), pack_f16(out[2], out[3])};
        else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < p.n) {
                    if (p.out_dt == MECHA_F32) store1<MECHA_F32>(p.out, at + e, out[e]);
                    else if (p.out_dt == MECHA_F16) store1<MECHA_F16>(p.out, at + e, out[e]);
                    else store1<MECHA_BF16>(p.out, at + e, out[e]);
                }
        }
        report(p.flags, poison_in, top, p.out_dt);
    }
}

template <int MODE, int AI, int BI>
int launch_direct(ProductParams p, hipStream_t s) {
    auto *const kernel = &product_direct_kernel<MODE, AI, BI>;
    constexpr int bytes = DIRECT_WAVES * 16 * AI * (16 * BI + 4) * (int)sizeof(float);
    if (bytes > 64 * 1024) MECHA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    p.tiles_m = (int)((p.m + 16 * AI - 1) / (16 * AI));
    p.tiles_n = (int)((p.n + 16 * BI - 1) / (16 * BI));
    MECHA_LAUNCH(MK_BLOCKS_PRODUCT, kernel, dim3((unsigned)p.tiles_m * (unsigned)p.tiles_n), dim3(DIRECT_THREADS), bytes, s, p);
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}
template <int MODE>
int launch_direct(int shape, const ProductParams &p, hipStream_t s) {
    if (shape == 0) return launch_direct<MODE, 1, 1>(p, s);
    if (shape == 1) return launch_direct<MODE, 1, 2>(p, s);
    if constexpr (MODE != EXACT_F32) {
        if (shape == 3) return launch_direct<MODE, 2, 4>(p, s);
    }
    return launch_direct<MODE, 2, 2>(p, s);
}

// ---------------------------------------------------------------------------------------------------- large products
// 32 MI x 256 outputs by 8 waves of 16 MI x 64, one workgroup a CU that goes on from tile to tile.  A K step is one block of 128: up to
// 64 KiB of codes in one of two LDS stages, 4 MI matrix instructions a wave (16 MI for float32 results).  The next step's codes -- the next
// tile's at a tile's end -- are on their way while this one is multiplied, also over the epilogue; so are the scales of the next BIG_CH
// words of blocks.  One barrier a step: behind it every wave's part of the next stage has landed and the other stage has been read.
// Workgroups go round the 8 XCDs, each with its own L2: an XCD gets a run of tiles, ordered so that the 32 at work at a time are 8 x 4
// tiles (2 MiB of a and 1 MiB of b at k = 1024, MI = 8).
//
// Measured (no base): 8192 x 8192 x 8192 426 to 454 us (2.4 to 2.6 PFLOP/s; the matrix unit's own rate is 4.3, and a plain per-tensor library product
// takes 428); 8192 x 10240 x 1280 100 to 112 us (2.0 PFLOP/s with 168 MB of results; the library 108); 8269 x 1280 x 5120 58 us (float32 scales: 64).  A
// 256 x 256 step takes 3900 cycles: 2048 of products at the unit's rate, and 1600 in which its 64 KiB come from L2 to LDS, which overlap
// only in part: fewer or more of them asked for at a step's start, by four waves or by eight, made no difference.  Float32 results
// multiply at bfloat16's rate (2.1 PFLOP/s): 1280 x 5120 x 8269 109 us (0.99 PFLOP/s on 200 of the 256 CUs).
constexpr int BIG_N = 256, BIG_M = 256, BIG_THREADS = 512, BIG_CH = 4, BIG_CUS = 256, BIG_BAND = 8;
struct BigLds {
    uint8_t stage[2][2][BIG_M * 128];             // [stage][a, b][row][128]
    uint32_t scale[2][2][BIG_CH][BIG_M];          // [parity of the chunk][a, b][word][row]
};

// 1 KiB, as dma4
__device__ __forceinline__ void dma1(const uint8_t *base, uint32_t off, uint32_t dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(base), "s"(dst) : "memory");
}
__device__ __forceinline__ uint32_t from_pair(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true); }   // lane ^ 1's
// Lanes 2 q and 2 q + 1 hold two 16-byte pieces of rows 2 q and 2 q + 1 each; afterwards lane 2 q holds the first pieces of both
// rows and lane 2 q + 1 the second ones (and back again: the exchange is its own inverse).
__device__ __forceinline__ void exchange(u32x4 &c0, u32x4 &c1, bool odd) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t got = from_pair(odd ? c0[j] : c1[j]);
        c0[j] = odd ? got : c0[j];
        c1[j] = odd ? c1[j] : got;
    }
}
template <int MODE, bool B_UNIFORM, int MI, int OUT, bool BASE, bool WHOLE>
__global__ __launch_bounds__(BIG_THREADS, 2) void product_big_kernel(ProductParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds_raw[];
    BigLds &lds = *reinterpret_cast<BigLds *>(lds_raw);
    constexpr bool EXACT = MODE == EXACT_F32 || MODE == EXACT_E8M0;              // float32 results; else float32 (OUT) are the sums of a part of k
    constexpr bool BF16 = OUT == MECHA_BF16;
    const uint32_t splits = MI == 4 && OUT == MECHA_F32 && !BASE ? (uint32_t)p.splits : 1u;
    constexpr int ROWS = 32 * MI, PER = MODE == HW_SCALES ? 4 * BIG_CH : BIG_CH; // rows of a tile; blocks a chunk of scales
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int wm = (wave & 1) * (16 * MI), wn = (wave >> 1) * 64;
    const int n_kb = (int)((p.k + SCALE_BLOCK - 1) / SCALE_BLOCK);
    const int tail = (int)(p.k - (int64_t)(n_kb - 1) * SCALE_BLOCK);

    // this workgroup's tiles: every (gridDim / 8)-th of its XCD's run (of the tiles of the first part of k, then the second, ...)
    const uint32_t tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n, all_tiles = tiles * splits;                   // < 2^24
    const uint32_t xcd = blockIdx.x & 7, per_xcd = gridDim.x >> 3;
    const uint32_t run0 = all_tiles * xcd / 8, run1 = all_tiles * (xcd + 1) / 8;
    uint32_t tile = run0 + (blockIdx.x >> 3);
    if (tile >= run1) return;
    // Tiles of one size end at one time, and all CUs' results together are bound by memory (5.4 us a round of 256 x 256 16-bit ones) while the matrix
    // units wait.  Where workgroups have several tiles, half of an XCD's -- those that have the fewer, if any do -- begin about half a round's stores
    // later (64 cycles a unit), and one half stores while the other multiplies: 8192 x 10240 x 1280 112 us, 116 without, 16384 x 5120 x 640 64 and 67,
    // 4096 x 8192 x 512 28 and 33.  More groups (4, 8, 32) gain less.
    if (run1 - run0 > per_xcd && (blockIdx.x >> 3) >= per_xcd / 2) {
        constexpr int UNITS = ROWS * (OUT == MECHA_F32 ? 4 : 2) / 4;
        for (int i = 0; i < UNITS; i += 16) __builtin_amdgcn_s_sleep(16);
    }
    // bands of BIG_BAND rows of tiles, down the band first; blocks k0 .. k0 + count - 1 of k
    struct Place { uint32_t m0, n0, part; int k0, count; };
    auto one = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };      // the same in every lane
    auto place = [&](uint32_t i) {
        Place at;
        at.part = splits > 1 ? one(i / tiles) : 0u;
        i -= at.part * tiles;
        const uint32_t band_tiles = BIG_BAND * (uint32_t)p.tiles_n, band = i / band_tiles, in = i - band * band_tiles;
        const uint32_t left = (uint32_t)p.tiles_m - band * BIG_BAND, high = left < BIG_BAND ? left : BIG_BAND;
        at.n0 = one(in / high * BIG_N);
        at.m0 = one((band * BIG_BAND + in % high) * ROWS);
        at.k0 = 0; at.count = n_kb;
        if (splits > 1) {
            at.k0 = (int)one((uint32_t)n_kb * at.part / splits);
            at.count = (int)one((uint32_t)n_kb * (at.part + 1) / splits) - at.k0;
        }
        return at;
    };

    // b's rows of fragment f: 16-bit results: 8 contiguous columns a lane and pair of fragments; float32: 4 a fragment
    auto b_at = [](int f, int rr) { return EXACT ? 16 * f + rr : b_row(f) + 8 * (rr >> 2) + (rr & 3); };
    auto swz_n = [](int row) { return EXACT ? swz_a(row) : swz_b(row); };

    // DMA: wave w brings rows 8 w .. + 7 of every 64 of each side, 1 KiB a piece; rows behind the last one read the last one
    constexpr int PIECES = 4 + (ROWS + 63) / 64;                                  // 6, 7 or 8
    const int bring_row = 8 * wave + (lane >> 3);
    const uint32_t part_a = 16u * (uint32_t)((lane & 7) ^ swz_a(bring_row)), part_b = 16u * (uint32_t)((lane & 7) ^ swz_n(bring_row));
    int last_a, last_b;
    const uint8_t *ga, *gb;
    auto aim = [&](const Place &at) {
        last_a = p.m - 1 - at.m0 < BIG_M ? (int)(p.m - 1 - at.m0) : BIG_M;
        last_b = p.n - 1 - at.n0 < BIG_N ? (int)(p.n - 1 - at.n0) : BIG_N;
        ga = p.a + (int64_t)at.m0 * p.a_pitch + (int64_t)at.k0 * SCALE_BLOCK;
        gb = p.b + (int64_t)at.n0 * p.b_pitch + (int64_t)at.k0 * SCALE_BLOCK;
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_byte *)lds_raw) + (uint32_t)wave * 1024u;
    auto issue = [&](int kb, int to, int x) {                                     // piece x: b's four, then a's
        if (x >= PIECES) return;
        const bool of_b = x < 4;
        const int y = of_b ? x : x - 4, row = 64 * y + bring_row, end = of_b ? last_b : last_a;
        dma1((of_b ? gb : ga) + (int64_t)kb * SCALE_BLOCK, (uint32_t)(row < end ? row : end) * (uint32_t)(of_b ? p.b_pitch : p.a_pitch) + (of_b ? part_b : part_a),
             lds0 + (uint32_t)to * (2 * BIG_M * 128) + (of_b ? BIG_M * 128 : 0) + 8192u * y);
    };
    // scales: thread (side, row) holds the words of a chunk between load and store
    uint32_t held[BIG_CH];
    const int side = __builtin_amdgcn_readfirstlane(t >> 8), srow = t & 255;
    auto load_scales = [&](uint32_t m0, uint32_t n0, int kb0) {
        const void *s = side ? p.sb : p.sa;
        const int64_t rows = side ? p.n : p.m, pitch = side ? p.sb_pitch : p.sa_pitch;
        int64_t row = (int64_t)(side ? n0 : m0) + srow;
        if (row >= rows) row = rows - 1;
        if (side ? p.b_tile : p.a_tile) row /= SCALE_BLOCK;
        if constexpr (MODE == HW_SCALES) {                                        // four bytes at a time, at the end the row's last four
            const uint8_t *at = static_cast<const uint8_t *>(s) + row * pitch;
#pragma unroll
            for (int w = 0; w < BIG_CH; w++) {
                const int kb = kb0 + 4 * w, from = kb < n_kb - 4 ? kb : n_kb - 4;
                uint32_t v;
                __builtin_memcpy(&v, at + from, 4);
                held[w] = v >> (8 * ((kb - from) & 3));
            }
        } else {
#pragma unroll
            for (int w = 0; w < BIG_CH; w++) {
                const int64_t at = row * pitch + (kb0 + w < n_kb ? kb0 + w : n_kb - 1);
                if constexpr (MODE == EXACT_E8M0) held[w] = static_cast<const uint8_t *>(s)[at];
                else held[w] = __float_as_uint(static_cast<const float *>(s)[at]);
            }
        }
    };
    auto put_scales = [&](int to) {
#pragma unroll
        for (int w = 0; w < BIG_CH; w++) lds.scale[to][side][w][srow] = MODE == EXACT_E8M0 ? held[w] << 23 : held[w];
    };

    // fragment addresses inside a stage and a row of scales
    uint32_t fa_at[2], fb_at[2];                                                  // of fragment 0; the others lie whole rows on, in the same slots
    const int ra0 = wm + r, rb0 = wn + b_at(0, r);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        fa_at[h] = (uint32_t)(ra0 * 128 + 16 * ((g + 4 * h) ^ swz_a(ra0)));
        fb_at[h] = (uint32_t)(rb0 * 128 + 16 * ((g + 4 * h) ^ swz_n(rb0)));
    }

    f32x4v acc[MI][4];                                                            // [a fragment][b fragment]
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int f = 0; f < 4; f++) acc[i][f] = f32x4v{0, 0, 0, 0};
    };
    Place here = place(tile), next = here;
    aim(here);
    load_scales(here.m0, here.n0, here.k0);
#pragma unroll
    for (int x = 0; x < PIECES; x++) issue(0, 0, x);
    put_scales(0);
    clear();
    wait_vm0();
    int stage = 0, chunk = 0, kb = 0;
    auto cut_tail = [&]() {                                                       // bytes behind column k are not the matrix's
        const int row = t >> 1;                                                   // thread: half of a row of each side
#pragma clang loop unroll(disable)
        for (int c = 0; c < 8; c++) {
            const int sd = c >> 2, piece = 4 * (t & 1) + (c & 3), left = tail - 16 * piece;
            if (left < 16) {
                u32x4 *at = reinterpret_cast<u32x4 *>(&lds.stage[stage][sd][row * 128 + 16 * (piece ^ (sd ? swz_n(row) : swz_a(row)))]);
                *at = first_bytes(*at, left);
            }
        }
        lds_barrier();
    };
    auto finish = [&]() {
        if constexpr (!EXACT && OUT == MECHA_F32) {                                // a part's sums; what joins the parts reads them from the caches
            float *const out = static_cast<float *>(p.out) + (int64_t)here.part * p.m * p.ld;
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    const int64_t m = (int64_t)here.m0 + wm + 16 * i + r, n = (int64_t)here.n0 + wn + b_row(f) + 8 * g;
                    if (m < p.m && n < p.ld) *reinterpret_cast<f32x4v *>(out + m * p.ld + n) = acc[i][f];
                }
            return;
        }
        // 16-byte pieces of two rows change places between two lanes, so that 8 lanes store a row's 128 bytes with one instruction;
        // base comes in the same way.  Non-temporal: whole lines, touched once (8192 x 10240 x 1280 112 us, 130 through the caches).
        constexpr int EACH = EXACT ? 4 : 8, ESIZE = EXACT ? 4 : 2;        // elements of a piece, bytes of one
        const bool odd = lane & 1;
        const int64_t row0 = (int64_t)here.m0 + wm + (r & ~1), line = p.ld * ESIZE;
        const int rows = p.m - row0 < BIG_M ? (int)(p.m - row0) : BIG_M;
        int64_t at0 = (((int64_t)here.part * p.m + row0) * p.ld + here.n0 + wn + (EXACT ? 16 * odd + 4 * g : 32 * odd + 8 * g)) * ESIZE;
        const int64_t behind = p.ld - ((int64_t)here.n0 + wn + (EXACT ? 16 * odd + 4 * g : 32 * odd + 8 * g));
        const int cols = behind < 64 ? (int)behind : 64;                          // from this lane's first piece to the row's end
        // rows that are whole 16 bytes: past the caches; else the pieces of a line meet there, and the row's last one is smaller
        auto get = [&](int64_t at, int left) -> u32x4 {
            const char *from = static_cast<const char *>(p.base) + at;
            if constexpr (WHOLE) return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from));
            else return left >= EACH ? *reinterpret_cast<const u32x4_any *>(from) : load_part(from, ESIZE * left);
        };
        auto put = [&](int64_t at, int left, u32x4 v) {
            char *to = static_cast<char *>(p.out) + at;
            if constexpr (WHOLE) __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(to));
            else if (left >= EACH) *reinterpret_cast<u32x4_any *>(to) = v;
            else store_part(to, v, ESIZE * left);
        };
        float poison_in = 0.0f, top = 0.0f;
        // base comes AHEAD fragments before it is added (8192 x 10240 x 1280 with a base 146 us, 153 with one; float32 results have no registers for it)
        constexpr int PAIRS = EXACT ? 2 : 1, AHEAD = EXACT ? 1 : 2;
        u32x4 pre[AHEAD][PAIRS][2];
        auto ask = [&](int i, int64_t from) {
            if constexpr (BASE) {
#pragma unroll
                for (int pair = 0; pair < PAIRS; pair++) {
                    const int64_t at = from + (EXACT ? 32 * ESIZE * pair : 0);
                    const int left = cols - (EXACT ? 32 * pair : 0);
                    u32x4 *c = pre[i % AHEAD][pair];
                    c[0] = c[1] = u32x4{0, 0, 0, 0};
                    if (left > 0 && 16 * i < rows) c[0] = get(at, left);
                    if (left > 0 && 16 * i + 1 < rows) c[1] = get(at + line, left);
                }
            }
        };
        int64_t ask_at = at0;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) { ask(i, ask_at); ask_at += 16 * line; asm volatile("" : "+v"(ask_at)); }
        if constexpr (BASE) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < MI; i++) {
#pragma unroll
            for (int pair = 0; pair < (EXACT ? 2 : 1); pair++) {
                // this lane's pieces in memory: number 0 (even lane) or 1 (odd) of the pair
                const int64_t at = at0 + (EXACT ? 32 * ESIZE * pair : 0);
                const int left = cols - (EXACT ? 32 * pair : 0);
                const bool in = left > 0, above = in && 16 * i < rows, below = in && 16 * i + 1 < rows;
                u32x4 c[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                if constexpr (BASE) {
                    c[0] = pre[i % AHEAD][pair][0]; c[1] = pre[i % AHEAD][pair][1];
                    exchange(c[0], c[1], odd);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float v[EACH];
#pragma unroll
                    for (int j = 0; j < EACH; j++) {
                        const float sum = EXACT ? acc[i][2 * pair + h][j & 3] : acc[i][2 * h + (j >> 2)][j & 3];
                        if constexpr (BASE) {
                            const uint32_t word = EXACT ? c[h][j & 3] : c[h][j >> 1];
                            const uint32_t half = j & 1 ? word >> 16 : word & 0xffffu;
                            const float bb = EXACT ? __uint_as_float(word) : BF16 ? bf16_bits_to_f32(half) : f16_bits_to_f32(half);
                            v[j] = __builtin_fmaf(sum, p.alpha, bb);
                            poison_in = __builtin_fmaf(bb, 0.0f, poison_in);
                        } else v[j] = sum * p.alpha;
                    }
                    // (rows and columns behind the last ones are made from the last ones, but without their base)
                    if (p.flags && row0 + 16 * i + odd < p.m) {
                        const int64_t in_row = p.n - ((int64_t)here.n0 + wn + (EXACT ? 32 * pair + 16 * h + 4 * g : 32 * h + 8 * g));
#pragma unroll
                        for (int j = 0; j < EACH; j++)
                            if (j < in_row) top = larger(top, v[j]);
                    }
                    if constexpr (EXACT) c[h] = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
                    else {
#pragma unroll
                        for (int j = 0; j < 4; j++) c[h][j] = BF16 ? pack_bf16(v[2 * j], v[2 * j + 1]) : pack_f16(v[2 * j], v[2 * j + 1]);
                    }
                }
                exchange(c[0], c[1], odd);
                if (above) put(at, left, c[0]);
                if (below) put(at + line, left, c[1]);
            }
            if (BASE && i + AHEAD < MI) { ask(i + AHEAD, ask_at); ask_at += 16 * line; }
            at0 += 16 * line;
            asm volatile("" : "+v"(at0));                                 // (addresses one after the other, not all at once)
            if (i % 2) __builtin_amdgcn_sched_barrier(0);
        }
        report(p.flags, poison_in, top, OUT);
    };
    if constexpr (EXACT) {
        // Float32 results.  A step is four fragments of a, each multiplied a quarter of its k at a time: 4 instructions of 16 cycles.  The matrix unit
        // leaves room for two other instructions beside each of its own, so the conversions to bfloat16 stand between them, one by one: the next
        // fragment's of a, and, while the last one is multiplied, the next step's of b, each in the place of the quarter that was used last (the last
        // quarter's in the next step).  Behind the second fragment all that is left of this stage is in registers: there the waves meet, the step
        // after the next is asked for into this one's place, and the next step's codes are read.  A wave that is in its last fragment goes first, which
        // keeps the two waves of a SIMD apart: 1280 x 5120 x 8269 110 us, 116 without.
        static_assert(MI == 4, "fragments");
        i32x8 fa[2], raw[4];
        uint32_t sa[2], rawscale[4];
        f32x4v sbf[4];
        i32x4 aq[2][4], bq[4][4];                                                // [fragment][quarter] of a and b
        int dkb = 0, dcount = here.count;                                         // the step that was asked for last
        uint32_t dtile = tile;
        auto advance = [&]() {                                                    // (behind the last tile it stays, and fetches what nobody reads)
            if (++dkb < dcount) return;
            dkb = 0;
            if (dtile + per_xcd >= run1) return;
            dtile += per_xcd;
            const Place to = place(dtile);
            dcount = to.count;
            aim(to);
        };
        const uint8_t *la = nullptr, *lb = nullptr;
        const uint32_t *sa_row = nullptr, *sb_row = nullptr;
        auto look = [&](int at_kb) {                                              // at the codes and scales of a step
            la = &lds.stage[stage][0][0]; lb = &lds.stage[stage][1][0];
            sa_row = &lds.scale[chunk][0][at_kb & (BIG_CH - 1)][ra0]; sb_row = &lds.scale[chunk][1][at_kb & (BIG_CH - 1)][0];
        };
        auto fetch_a = [&](int i) {
            fa[i & 1] = join(*reinterpret_cast<const u32x4 *>(la + fa_at[0] + 2048 * i), *reinterpret_cast<const u32x4 *>(la + fa_at[1] + 2048 * i));
            sa[i & 1] = sa_row[16 * i];
        };
        auto fetch_b = [&]() {
#pragma unroll
            for (int f = 0; f < 4; f++) {
                raw[f] = join(*reinterpret_cast<const u32x4 *>(lb + fb_at[0] + 2048 * f), *reinterpret_cast<const u32x4 *>(lb + fb_at[1] + 2048 * f));
                if constexpr (MODE == EXACT_E8M0) rawscale[f] = sb_row[rb0 + 16 * f];
            }
        };
        auto fetch_sb = [&]() {
            if constexpr (MODE == EXACT_F32) {
#pragma unroll
                for (int f = 0; f < 4; f++) sbf[f] = *reinterpret_cast<const f32x4v *>(&sb_row[wn + 16 * f + 4 * g]);
            }
        };
        // Power-of-two scales go into the conversion: code * 2^e is a bfloat16.
        auto code2 = [](const i32x8 &v, int q, int w, uint32_t scale) {           // codes 2 w, 2 w + 1 of quarter q
            const float by = MODE == EXACT_E8M0 ? __uint_as_float(scale) : 1.0f;
            const int from = v[2 * q + w / 2];
            return __builtin_bit_cast(int, w & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(from, by, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(from, by, false));
        };
        // (the empty statements keep a conversion where it stands)
        auto make_a = [&](int i, int q, int w) {
            int v = code2(fa[i & 1], q, w, sa[i & 1]);
            asm volatile("" : "+v"(v));
            aq[i & 1][q][w] = v;
        };
        auto make_b = [&](int f, int q) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                int v = code2(raw[f], q, w, rawscale[f]);
                asm volatile("" : "+v"(v));
                bq[f][q][w] = v;
            }
        };
        auto multiply = [&](int i, float scale, auto between) {
            f32x4v d[4];
#pragma unroll
            for (int f = 0; f < 4; f++) d[f] = f32x4v{0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    const bf16x8 x = __builtin_bit_cast(bf16x8, bq[f][q]), y = __builtin_bit_cast(bf16x8, aq[i & 1][q]);
                    if constexpr (MODE == EXACT_E8M0) acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc[i][f], 0, 0, 0);
                    else d[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, d[f], 0, 0, 0);
                    between(q, f);
                    __builtin_amdgcn_sched_barrier(0);
                }
            if constexpr (MODE == EXACT_F32) {
#pragma unroll
                for (int f = 0; f < 4; f++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][f][e] = __builtin_fmaf(d[f][e] * sbf[f][e], scale, acc[i][f][e]);
            }
            // (nothing is executed here: the sums are made at this point, not sunk to the stores)
            asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]));
            __builtin_amdgcn_sched_barrier(0);
        };
        lds_barrier();
        advance();
#pragma unroll
        for (int x = 0; x < PIECES; x++) issue(dkb, 1, x);
        look(0);
        fetch_b();
        fetch_sb();
        fetch_a(0);
#pragma unroll
        for (int q = 0; q < 4; q++) {
#pragma unroll
            for (int f = 0; f < 4; f++) {
                if (q < 3) make_b(f, q);
                make_a(0, q, f);
            }
        }
        float si = __uint_as_float(sa[0]);
        fetch_a(1);
#pragma clang loop unroll(disable)
        while (true) {
            const bool last = kb + 1 == here.count, more = tile + per_xcd < run1;
            if (last && more) next = place(tile + per_xcd);
            const int next_kb = last ? 0 : kb + 1;
            const bool refill = last ? more : next_kb % PER == 0;
            if (refill) load_scales(last ? next.m0 : here.m0, last ? next.n0 : here.n0, last ? next.k0 : here.k0 + next_kb);
            float next_si = __uint_as_float(sa[1]);
            fetch_a(2);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            multiply(0, si, [&](int q, int f) {
                if (q == 0) make_b(f, 3);
                make_a(1, q, f);
            });
            si = next_si;
            fetch_a(3);
            __builtin_amdgcn_sched_barrier(0);
            next_si = __uint_as_float(sa[0]);
            multiply(1, si, [&](int q, int f) { make_a(2, q, f); });
            si = next_si;
            wait_vm0();                                                           // the next stage
            if (refill) { put_scales(chunk ^ 1); chunk ^= 1; }
            stage ^= 1;
            lds_barrier();                                                        // everyone's part of it, and this one has been read
            if (next_kb + 1 == here.count && here.k0 + here.count == n_kb && tail < SCALE_BLOCK) cut_tail();
            look(next_kb);
            fetch_b();
            fetch_a(0);
            advance();
            __builtin_amdgcn_sched_barrier(0);
            next_si = __uint_as_float(sa[1]);
            multiply(2, si, [&](int q, int f) {
                make_a(3, q, f);
                if (f == 3 && q < 3) issue(dkb, stage ^ 1, q);
            });
            si = next_si;
            fetch_a(1);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            multiply(3, si, [&](int q, int f) {
                if (q > 0) make_b(f, q - 1);
                make_a(0, q, f);
                if (f == 3 && q < 3) issue(dkb, stage ^ 1, 3 + q);
            });
            si = __uint_as_float(sa[0]);
            fetch_sb();
            if (last) {
                finish();
                if (!more) break;
                tile += per_xcd; here = next;
                clear();
            }
            kb = next_kb;
        }
        wait_vm0();                                                               // what nobody reads has landed, too
    } else {
        // Fragment i + 2 of a is read while fragment i is multiplied, and a step's last fragment is multiplied behind the next barrier, while
        // the next step's first ones come from LDS.
        constexpr int SLOTS = MI == 4 ? 4 : 3;                                        // the carried fragment keeps its slot while fragment 0 is read
        static_assert((MI - 1) % SLOTS != 0, "slots");
        i32x8 fa[SLOTS], fb[4];
        uint32_t sa[SLOTS], sb[4];                                                    // sb: the matrix unit's
        f32x4v sbf[4];
        float sb1 = 0.0f;                                                             // one scale of b for the wave's columns: a power of two for the
        int sb1_byte = 0;                                                             // matrix unit, and what is left of it, under 2
#pragma clang loop unroll(disable)
        while (true) {
            const bool last = kb + 1 == here.count, more = tile + per_xcd < run1;
            lds_barrier();
            if (last && here.k0 + here.count == n_kb && tail < SCALE_BLOCK) cut_tail();
            if (last && more) {
                next = place(tile + per_xcd);
                aim(next);
            }
            const int next_kb = last ? 0 : kb + 1;
            const bool refill = last ? more : next_kb % PER == 0;
            if (refill) load_scales(last ? next.m0 : here.m0, last ? next.n0 : here.n0, last ? next.k0 : here.k0 + next_kb);

            const uint8_t *la = &lds.stage[stage][0][0], *lb = &lds.stage[stage][1][0];
            const int w = MODE == HW_SCALES ? (kb / 4) & (BIG_CH - 1) : kb & (BIG_CH - 1), sh = 8 * (kb & 3);
            const uint32_t *sa_row = &lds.scale[chunk][0][w][ra0], *sb_row = &lds.scale[chunk][1][w][0];
            auto read_a = [&](int i) { return join(*reinterpret_cast<const u32x4 *>(la + fa_at[0] + 2048 * i), *reinterpret_cast<const u32x4 *>(la + fa_at[1] + 2048 * i)); };
            auto read_b = [&](int f) {
                const int on = 128 * (b_at(f, 0) - b_at(0, 0));
                return join(*reinterpret_cast<const u32x4 *>(lb + fb_at[0] + on), *reinterpret_cast<const u32x4 *>(lb + fb_at[1] + on));
            };
            auto bring = [&](int x) { issue(next_kb, stage ^ 1, x); };
            // One 16 x 16 x 128 product; shift: the byte of the scales' words that belongs to the step (HW_SCALES).
            auto multiply = [&](int i, int f, int shift) {
                if constexpr (MODE == HW_SCALES) {
                    acc[i][f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa[i % SLOTS], acc[i][f], 0, 0, 0, (int)sb[f], 0, (int)(sa[i % SLOTS] >> shift));
                } else {
                    const f32x4v d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa[i % SLOTS], f32x4v{0, 0, 0, 0}, 0, 0, 0, B_UNIFORM ? sb1_byte : 0x7f7f7f7f, 0, 0x7f7f7f7f);
                    const float sf = __uint_as_float(sa[i % SLOTS]) * (B_UNIFORM ? sb1 : 1.0f);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][f][e] = __builtin_fmaf(B_UNIFORM ? d[e] : d[e] * sbf[f][e], sf, acc[i][f][e]);
                }
            };
            auto pin = [&](int i) {                                               // (nothing is executed here: the sums are made at this point, not sunk to the stores)
                asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]));
                __builtin_amdgcn_sched_barrier(0);
            };
            auto fetch_a = [&](int i) { fa[i % SLOTS] = read_a(i); sa[i % SLOTS] = sa_row[16 * i]; };
            auto fetch_b = [&](int f) {
                if constexpr (MODE == HW_SCALES) sb[f] = sb_row[rb0 + b_row(f)] >> sh;
                if constexpr (MODE == F32_SCALES && !B_UNIFORM) sbf[f] = *reinterpret_cast<const f32x4v *>(&sb_row[wn + b_row(f) + 8 * g]);
                fb[f] = read_b(f);
            };
            constexpr int Z = MI - 1;                                             // the fragment carried over
            // The next stage is asked for in pieces between the products: the memory pipeline takes 1600 cycles for 64 KiB, and a wave that asks
            // for more than it takes stands still.  Short steps need all the time there is for it.
            constexpr int EARLY = MI == 4 ? PIECES : 2;
            fetch_a(0);
            __builtin_amdgcn_sched_barrier(0);
            if (kb > 0) {
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    multiply(Z, f, (sh - 8) & 31);
                    asm volatile("" : "+v"(acc[Z][f]));
                    __builtin_amdgcn_sched_barrier(0);
                    fetch_b(f);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int f = 0; f < 4; f++) fetch_b(f);
            }
            if constexpr (B_UNIFORM) {                                            // (0, inf and NaN: 2^0 and themselves; a subnormal one: 2^-127 and under 1)
                const float whole = __uint_as_float(sb_row[wn]);
                const int e = 127 + __builtin_amdgcn_frexp_expf(whole);
                sb1_byte = e < 0 ? 0 : e > 254 ? 254 : e;
                sb1 = ldexpf(whole, 127 - sb1_byte);
            }
            fetch_a(1);
#pragma unroll
            for (int x = 0; x < EARLY; x++) bring(x);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < Z; i++) {
                if (i + 2 < MI) fetch_a(i + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    multiply(i, f, sh);
                    if (f % 2) bring(EARLY + 2 * i + f / 2);
                }
                pin(i);
            }
            if (last) {
#pragma unroll
                for (int f = 0; f < 4; f++) multiply(Z, f, sh);
                pin(Z);
            }
            wait_vm0();                                                               // the next stage; before the stores, which the same counter counts
            if (refill) { put_scales(chunk ^ 1); chunk ^= 1; }
            stage ^= 1;
            kb = next_kb;
            if (last) {
                finish();
                if (!more) break;
                tile += per_xcd; here = next;
                clear();
            }
        }
    }
}

// The parts of k together: out = base + alpha * (part 0 + part 1 + ...), added in that order in float32.  4 columns a thread; the parts
// (rows of ld, a multiple of 8) come out of the caches: 1280 x 1280 of 5 parts 7.3 us, 1024 x 1280 to bfloat16 5.0.
template <int DT, bool BASE>
__global__ __launch_bounds__(MECHA_BLOCK) void join_kernel(const float *parts, int splits, int64_t m, int64_t n, int64_t ld, const void *base, void *out, float alpha, uint32_t *flags) {
    const int64_t i = ((int64_t)blockIdx.x * MECHA_BLOCK + threadIdx.x) * 4, count = m * ld;
    if (i >= count) return;
    const int64_t row = count < (1ll << 31) ? (int64_t)((uint32_t)i / (uint32_t)ld) : i / ld, col = i - row * ld;
    const int left = n - col < 4 ? (int)(n - col) : 4;
    if (left <= 0) return;
    f32x4v sum = *reinterpret_cast<const f32x4v *>(parts + i);
    const float *at = parts + i;
#pragma unroll 4
    for (int x = 1; x < splits; x++) {
        at += count;
        const f32x4v v = *reinterpret_cast<const f32x4v *>(at);
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] += v[e];
    }
    constexpr int ESIZE = DT == MECHA_F32 ? 4 : 2;
    const int64_t to = (row * n + col) * ESIZE;
    float v[4], b[4] = {0, 0, 0, 0}, poison_in = 0.0f, top = 0.0f;
    if constexpr (BASE) {
        const char *from = static_cast<const char *>(base) + to;
        if constexpr (DT == MECHA_F32) {
            const u32x4 w = left == 4 ? *reinterpret_cast<const u32x4_any *>(from) : load_part(from, 4 * left);
#pragma unroll
            for (int e = 0; e < 4; e++) b[e] = __uint_as_float(w[e]);
        } else {
            u32x2 w;
            if (left == 4) w = *reinterpret_cast<const u32x2_any *>(from);
            else { const u32x4 x = load_part(from, 2 * left); w = u32x2{x.x, x.y}; }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t half = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
                b[e] = DT == MECHA_BF16 ? bf16_bits_to_f32(half) : f16_bits_to_f32(half);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[e] = BASE ? __builtin_fmaf(sum[e], alpha, b[e]) : sum[e] * alpha;
        if (e < left) {
            poison_in = __builtin_fmaf(b[e], 0.0f, poison_in);
            top = larger(top, v[e]);
        }
    }
    char *const put = static_cast<char *>(out) + to;
    if constexpr (DT == MECHA_F32) {
        const u32x4 w = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        if (left == 4) *reinterpret_cast<u32x4_any *>(put) = w;
        else store_part(put, w, 4 * left);
    } else {
        const u32x2 w = DT == MECHA_BF16 ? u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])} : u32x2{pack_f16(v[0], v[1]), pack_f16(v[2], v[3])};
        if (left == 4) *reinterpret_cast<u32x2_any *>(put) = w;
        else store_part(put, u32x4{w.x, w.y, 0u, 0u}, 2 * left);
    }
    report(flags, poison_in, top, DT);
}
constexpr int64_t part_ld(int64_t n) { return (n + 7) / 8 * 8; }
int launch_join(const ProductParams &p, const void *parts, hipStream_t s) {
    const int64_t ld = part_ld(p.n), blocks = (p.m * ld / 4 + MECHA_BLOCK - 1) / MECHA_BLOCK;
    auto go = [&](auto dt, auto base) {
        MECHA_LAUNCH(MK_BLOCKS_PRODUCT, (join_kernel<decltype(dt)::value, decltype(base)::value>), dim3((unsigned)blocks), dim3(MECHA_BLOCK), 0, s, static_cast<const float *>(parts),
                     p.splits, p.m, p.n, ld, p.base, p.out, p.alpha, p.flags);
    };
    auto with_base = [&](auto dt) { if (p.base) go(dt, std::true_type{}); else go(dt, std::false_type{}); };
    switch (p.out_dt) {
        case MECHA_F32: with_base(std::integral_constant<int, MECHA_F32>{}); break;
        case MECHA_F16: with_base(std::integral_constant<int, MECHA_F16>{}); break;
        default: with_base(std::integral_constant<int, MECHA_BF16>{}); break;
    }
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

template <int MODE, bool B_UNIFORM, int MI, int OUT, bool BASE, bool PART = false>
int launch_tiles(ProductParams p, hipStream_t s) {
    p.tiles_m = (int)((p.m + 32 * MI - 1) / (32 * MI));
    p.tiles_n = (int)((p.n + BIG_N - 1) / BIG_N);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.splits, grid = tiles < BIG_CUS ? (tiles + 7) / 8 * 8 : BIG_CUS;
    auto *kernel = &product_big_kernel<MODE, B_UNIFORM, MI, OUT, BASE, true>;
    if constexpr (!PART) {
        if (!p.aligned) kernel = &product_big_kernel<MODE, B_UNIFORM, MI, OUT, BASE, false>;
    }
    MECHA_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(BigLds)));
    MECHA_LAUNCH(MK_BLOCKS_PRODUCT, kernel, dim3((unsigned)grid), dim3(BIG_THREADS), sizeof(BigLds), s, p);
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}
template <int MODE, bool B_UNIFORM, int MI>
int launch_big(const ProductParams &p, void *workspace, hipStream_t s) {
    constexpr bool EXACT = MODE == EXACT_F32 || MODE == EXACT_E8M0;
    if constexpr (MI == 4) {
        if (p.splits > 1) {
            ProductParams part = p;
            part.out = workspace; part.out_dt = MECHA_F32; part.base = nullptr; part.alpha = 1.0f; part.flags = nullptr;
            part.ld = part_ld(p.n); part.aligned = 1;
            const int st = launch_tiles<MODE, B_UNIFORM, MI, MECHA_F32, false, true>(part, s);
            return st ? st : launch_join(p, workspace, s);
        }
    }
    if constexpr (EXACT) return p.base ? launch_tiles<MODE, B_UNIFORM, MI, MECHA_F32, true>(p, s) : launch_tiles<MODE, B_UNIFORM, MI, MECHA_F32, false>(p, s);
    else if (p.out_dt == MECHA_F16) return p.base ? launch_tiles<MODE, B_UNIFORM, MI, MECHA_F16, true>(p, s) : launch_tiles<MODE, B_UNIFORM, MI, MECHA_F16, false>(p, s);
    else return p.base ? launch_tiles<MODE, B_UNIFORM, MI, MECHA_BF16, true>(p, s) : launch_tiles<MODE, B_UNIFORM, MI, MECHA_BF16, false>(p, s);
}
template <int MODE, bool B_UNIFORM>
int launch_big(int mi, const ProductParams &p, void *workspace, hipStream_t s) {
    if constexpr (MODE == HW_SCALES || MODE == F32_SCALES) {
        if constexpr (MODE == HW_SCALES || B_UNIFORM) {
            if (mi == 8) return launch_big<MODE, B_UNIFORM, 8>(p, workspace, s);
        }
        if (mi == 6) return launch_big<MODE, B_UNIFORM, 6>(p, workspace, s);
    }
    return launch_big<MODE, B_UNIFORM, 4>(p, workspace, s);
}

// ---------------------------------------------------------------------------------------------------- which kernel
// The time each would take, in microseconds, from what it measured on 256 CUs (138 random products up to 16384 x 10240 x 8192 of all four kinds, each
// with every kernel: the choice is 2 % over the best in the mean, 35 % at worst):
//   direct: a launch, the join of a workgroup's waves, and the slower of one workgroup's reads (33 KB a us) and all workgroups' (5 TB/s, 1 ns and their
//           joins): 600 x 1280 x 1280 (float32 scales and results) 17 us with 32 x 32 outputs a workgroup, 22 in 128 x 128 tiles;
//   tiled:  rounds of tiles over the CUs, each n_kb steps and an epilogue.  128 x 128 tiles (two workgroups a CU) fill a few CUs more evenly:
//           1024 x 1280 x 5120 38 us, 50 with 128 x 256 tiles; the larger ones share more: 8192 x 1280 x 5120 59 us (192 x 256), 84 with
//           128 x 128; 16384 x 5120 x 640 63 us (256 x 256), 79 (128 x 256).
//   in parts: results of fewer 128 x 256 tiles than CUs, k shared out among 2 to 32 workgroups a tile (4 blocks at least each): the parts are written
//           and read once as float32 and joined by a second launch: 1280 x 1280 x 8269 34 us in 5 parts (58 in 128 x 128 tiles; float32 results 41 and 80),
//           1024 x 1280 x 5120 27 (38), 300 x 2560 x 8192 26 (55).
constexpr int MAX_SPLITS = 32;
int mode_of(int scale_dtype, int out_dtype) {
    const bool e8m0 = scale_dtype == MECHA_SCALE_E8M0;
    return out_dtype == MECHA_F32 ? (e8m0 ? EXACT_E8M0 : EXACT_F32) : e8m0 ? HW_SCALES : F32_SCALES;
}
// The large kernel reads base as it stores the result, and scales four blocks at a time.
bool large_kernels(int64_t k, bool other_base) { return k > 3 * SCALE_BLOCK && !other_base; }
constexpr int DIRECT_ROWS[4] = {16, 16, 32, 32}, DIRECT_COLS[4] = {16, 32, 32, 64};
struct Choice { int direct = -1, mi = 0, splits = 1; };        // shape of the direct kernel; else MI of the large one; else the 128 x 128 one
Choice choose(int64_t m, int64_t n, int64_t k, int mode, int b_tile, bool large_ok, bool split_ok) {
    // a step of 128 x 128, MI = 4, 6, 8: power-of-two scales; float32 scales with one of b's in a square; with one in every row of b, where MI = 8
    // has no registers for them (8192 x 8192 x 2048: 264 us, 194 with MI = 6); float32 results
    static const double step[4][4] = {{0.75, 1.20, 1.36, 1.56}, {1.18, 1.34, 1.54, 1.81}, {1.18, 1.51, 1.78, 0.0}, {1.42, 1.60, 0.0, 0.0}};
    const double *us = step[mode == HW_SCALES ? 0 : mode != F32_SCALES ? 3 : b_tile ? 1 : 2];
    const double n_kb = (double)((k + SCALE_BLOCK - 1) / SCALE_BLOCK);
    auto up = [](int64_t a, int64_t b) { return (double)((a + b - 1) / b); };
    const double mid_tiles = up(m, 128) * up(n, 128) / BIG_CUS;
    double best = 6.0 + (mid_tiles > 1.0 ? mid_tiles : 1.0) * (n_kb * us[0] + 1.0);
    Choice c;
    if (large_ok) {
        for (int mi = 4; mi <= 8 && us[mi / 2 - 1] > 0.0; mi += 2) {
            const double rounds = up((int64_t)(up(m, 32 * mi) * up(n, BIG_N)), BIG_CUS), t = 3.5 + rounds * (n_kb * us[mi / 2 - 1] + 0.25 * mi);
            if (t < best) { best = t; c.mi = mi; }
        }
        const double tiles = up(m, 128) * up(n, BIG_N), part = (double)m * (double)n * 8.0 / 5e6;
        for (int x = 2; split_ok && x <= MAX_SPLITS && 4 * x <= n_kb && (x - 1) * tiles < BIG_CUS; x++) {
            const double rounds = up((int64_t)tiles * x, BIG_CUS), t = 8.5 + rounds * (up((int64_t)n_kb, x) * us[1] + 1.0) + x * part;
            if (t < best) { best = t; c.mi = 4; c.splits = x; }
        }
    }
    const int *const rows = DIRECT_ROWS, *const cols = DIRECT_COLS;
    for (int d = 0; d < (mode == EXACT_F32 ? 3 : 4); d++) {     // (float32 scales, float32 results: the last shape's registers spill, 600 x 1280 x 1280 34 us, 17 with 32 x 32)
        const double blocks = up(m, rows[d]) * up(n, cols[d]), bytes = (rows[d] + cols[d]) * n_kb * SCALE_BLOCK, one = bytes / 33e3, all = blocks * (bytes / 5e6 + 0.001 + 2e-6 * rows[d] * cols[d]);
        const double t = 2.5 + 0.001 * rows[d] * cols[d] + (one > all ? one : all);
        if (t < best && blocks * DIRECT_THREADS < 4294967296.0) { best = t; c.mi = 0; c.splits = 1; c.direct = d; }     // a launch's threads
    }
    return c;
}

}  // namespace

extern "C" {

size_t mecha_block_product_workspace_bytes(int64_t m, int64_t n, int64_t k, int scale_dtype, int b_tile, int out_dtype) {
    if (m < 1 || n < 1 || !large_kernels(k, false)) return 0;
    const Choice c = choose(m, n, k, mode_of(scale_dtype, out_dtype), b_tile, true, true);
    return c.splits > 1 ? (size_t)c.splits * (size_t)m * (size_t)part_ld(n) * sizeof(float) : 0;
}

int mecha_block_product_tile(int64_t m, int64_t n, int64_t k, int scale_dtype, int b_tile, int out_dtype, int other_base) {
    if (m < 1 || n < 1 || k < 1) return 0;
    const Choice c = choose(m, n, k, mode_of(scale_dtype, out_dtype), b_tile, large_kernels(k, other_base), !other_base);
    const int tm = c.direct >= 0 ? DIRECT_ROWS[c.direct] : c.mi ? 32 * c.mi : 128, tn = c.direct >= 0 ? DIRECT_COLS[c.direct] : c.mi ? BIG_N : 128;
    return tm << 20 | tn << 8 | c.splits;
}

int mecha_block_product(const mecha_block_matrix *a, const mecha_block_matrix *b, const void *base, int base_dtype, void *out, int out_dtype,
                        float alpha, uint32_t *flags, void *workspace, size_t workspace_bytes, void *stream) {
    MECHA_REQUIRE(a != nullptr && b != nullptr, "a matrix is NULL");
    MECHA_REQUIRE(mecha_valid_dtype(out_dtype) && (base == nullptr || mecha_valid_dtype(base_dtype)), "unknown dtype code (base %d, out %d)", base_dtype, out_dtype);
    int st = mecha_check_blocks("a", *a);
    if (st) return st;
    st = mecha_check_blocks("b", *b);
    if (st) return st;
    MECHA_REQUIRE(a->scale_dtype == b->scale_dtype, "scales of two types (%d, %d)", a->scale_dtype, b->scale_dtype);
    const int64_t m = a->rows, n = b->rows, k = a->cols;
    MECHA_REQUIRE(k >= 1 && b->cols == k, "a has %lld columns, b %lld: they must be the same, and some", (long long)k, (long long)b->cols);
    if (m == 0 || n == 0) return MECHA_OK;
    MECHA_REQUIRE(out != nullptr, "out is NULL");
    MECHA_REQUIRE(a->pitch <= (1 << 24) && b->pitch <= (1 << 24), "rows of more than 2^24 bytes (%lld, %lld)", (long long)a->pitch, (long long)b->pitch);
    const int64_t tm = (m + 127) / 128, tn = (n + 127) / 128;
    MECHA_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && tm * tn < (1ll << 24), "%lld x %lld outputs are beyond one launch", (long long)m, (long long)n);
    const size_t out_bytes = (size_t)m * n * mecha_dtype_size(out_dtype);
    for (const mecha_block_matrix *q : {a, b})
        MECHA_REQUIRE(!mecha_overlap(out, out_bytes, q->codes, mecha_codes_bytes(*q)) && !mecha_overlap(out, out_bytes, q->scales, mecha_scales_bytes(*q)),
                      "out shares memory with a or b");
    MECHA_REQUIRE(base == nullptr || (base == out && base_dtype == out_dtype) || !mecha_overlap(out, out_bytes, base, (size_t)m * n * mecha_dtype_size(base_dtype)),
                  "out may be base itself, of the same dtype, but not overlap it otherwise");
    ProductParams p{static_cast<const uint8_t *>(a->codes), a->pitch, a->scales, a->scale_pitch, a->tile, static_cast<const uint8_t *>(b->codes), b->pitch,
                    b->scales, b->scale_pitch, b->tile, base, out, m, n, k, base_dtype, out_dtype, alpha, flags, (int)tm, (int)tn, n, 1, 0};
    const int b_tile = b->tile, scale_dtype = a->scale_dtype;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool e8m0 = scale_dtype == MECHA_SCALE_E8M0;
    const bool wide = out_dtype == MECHA_F32;
    const bool large_ok = large_kernels(k, base != nullptr && base_dtype != out_dtype);
    p.aligned = n % (wide ? 4 : 8) == 0 && mecha_aligned16(out) && (base == nullptr || mecha_aligned16(base));
    const int mode = mode_of(scale_dtype, out_dtype);
    Choice c = choose(m, n, k, mode, b_tile, large_ok, workspace != nullptr);
    if (c.splits > 1 && ((size_t)c.splits * (size_t)m * (size_t)part_ld(n) * sizeof(float) > workspace_bytes || !mecha_aligned16(workspace))) c = choose(m, n, k, mode, b_tile, large_ok, false);
    p.splits = c.splits;
    if (c.splits > 1) {
        const size_t parts = (size_t)c.splits * (size_t)m * (size_t)part_ld(n) * sizeof(float);
        MECHA_REQUIRE(!mecha_overlap(workspace, parts, out, out_bytes) && !mecha_overlap(workspace, parts, base, (size_t)m * n * mecha_dtype_size(base_dtype)), "workspace shares memory with out or base");
        for (const mecha_block_matrix *q : {a, b})
            MECHA_REQUIRE(!mecha_overlap(workspace, parts, q->codes, mecha_codes_bytes(*q)) && !mecha_overlap(workspace, parts, q->scales, mecha_scales_bytes(*q)), "workspace shares memory with a or b");
    }
    if (c.direct >= 0) {
        if (wide) return e8m0 ? launch_direct<EXACT_E8M0>(c.direct, p, s) : launch_direct<EXACT_F32>(c.direct, p, s);
        return e8m0 ? launch_direct<HW_SCALES>(c.direct, p, s) : launch_direct<F32_SCALES>(c.direct, p, s);
    }
    if (c.mi) {
        if (wide) return e8m0 ? launch_big<EXACT_E8M0, false>(c.mi, p, workspace, s) : launch_big<EXACT_F32, false>(c.mi, p, workspace, s);
        if (e8m0) return launch_big<HW_SCALES, false>(c.mi, p, workspace, s);
        return b_tile ? launch_big<F32_SCALES, true>(c.mi, p, workspace, s) : launch_big<F32_SCALES, false>(c.mi, p, workspace, s);
    }
    auto go = [&](auto mode, auto dt) {
        constexpr int MODE = decltype(mode)::value, DT = decltype(dt)::value;
        const dim3 grid((unsigned)(tm * tn)), block(MECHA_BLOCK);
        if (n % 8 == 0 && mecha_aligned16(out) && (base == nullptr || mecha_aligned16(base))) MECHA_LAUNCH(MK_BLOCKS_PRODUCT, (product_kernel<MODE, DT, true>), grid, block, 0, s, p);
        else MECHA_LAUNCH(MK_BLOCKS_PRODUCT, (product_kernel<MODE, DT, false>), grid, block, 0, s, p);
    };
    auto with_mode = [&](auto power, auto real, auto dt) { if (e8m0) go(power, dt); else go(real, dt); };
    typedef std::integral_constant<int, HW_SCALES> Hw;
    typedef std::integral_constant<int, F32_SCALES> F32;
    switch (out_dtype) {
        case MECHA_F32: with_mode(std::integral_constant<int, EXACT_E8M0>{}, std::integral_constant<int, EXACT_F32>{}, std::integral_constant<int, MECHA_F32>{}); break;
        case MECHA_F16: with_mode(Hw{}, F32{}, std::integral_constant<int, MECHA_F16>{}); break;
        default: with_mode(Hw{}, F32{}, std::integral_constant<int, MECHA_BF16>{}); break;
    }
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

}  // extern "C"
