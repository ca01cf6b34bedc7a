// block_product.hip -- the product of two matrices in 8 bits with a scale for each block of 128 (blocks.hip), fused with
// add_difference into a base key.
#include <type_traits>
#include "blocks.h"

namespace {

// out[m][n] = base[m][n] + alpha * sum over the blocks kb of sa[m][kb] sb[n][kb] * (sum over the block's k of a[m][k] b[n][k]),
// on v_mfma_scale_f32_16x16x128_f8f6f4: one instruction takes a whole block of 128 of 16 rows of each side and, with
// power-of-two scales, the two scales of every row as well, so they cost nothing.  With float32 scales the block's sum comes out of the
// matrix unit by itself and is added with one fma an element.  Sums are float32.
//
// What the 8-bit matrix instructions lose (all of them; measured with single products): the products of 8 neighbouring k are aligned to
// the largest, and what lies under 2^-13 of it is cut off; the groups are then added in float32.  That is 1.5e-5 of a result (2-norm, normal
// codes), 1/14 of what rounding to float16 loses and 1/110 of bfloat16's, so results of 16 bits are made this way.  A float32 result
// would show it: there the codes are turned into bfloat16, which holds each exactly, and multiplied on v_mfma_f32_16x16x32_bf16, which
// adds in float32 (1e-8 to 5e-8 measured) at half the rate.
//
// b's rows are the instruction's A operand (accumulator rows) and a's rows its B operand (accumulator columns): lane l holds 4
// accumulators of output row m = l % 16.  b's rows are dealt to the fragments so that a lane's accumulators of 4 fragments are 16
// CONTIGUOUS columns: row r of fragment f is column 16 (r / 4) + 4 f + r % 4 of the wave's 64.
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

// 16-byte slot of a row's 128 bytes in LDS, so that the 16 rows of a fragment lie in 16 different (row parity, slot) places of
// the 256-byte bank row: a's fragments are 16 consecutive rows, b's are rows 16 (r / 4) + r % 4 (+ 4 f).
__device__ __forceinline__ int swz_a(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int swz_b(int row) { return ((row >> 1) & 1) | ((row >> 3) & 6); }

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
__device__ __forceinline__ bf16x8 codes_to_bf16(int lo, int hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
__device__ __forceinline__ f32x4v exact_block(i32x8 a, i32x8 b, f32x4v c) {
#pragma unroll
    for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_to_bf16(a[2 * q], a[2 * q + 1]), codes_to_bf16(b[2 * q], b[2 * q + 1]), c, 0, 0, 0);
    return c;
}

// 16 contiguous columns of one output row: base + alpha * acc.  Finite checks: fma(x, 0, poison) stays 0 while every x is finite.
template <int OUT_DT>
__device__ __forceinline__ void store_row16(const ProductParams &p, int64_t m, int64_t n, const float (&acc)[16], bool vec) {
    if (m >= p.m || n >= p.n) return;
    const int64_t i = m * p.n + n;
    const bool whole = vec && n + 16 <= p.n;
    float r[16], poison_in = 0.0f, poison_out = 0.0f;
    if (p.base) {
        const int dt = p.base_dt;
        float b[16];
        if (whole) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float t[8];
                if (dt == MECHA_F32) load8<MECHA_F32>(p.base, i + 8 * h, t);
                else if (dt == MECHA_F16) load8<MECHA_F16>(p.base, i + 8 * h, t);
                else load8<MECHA_BF16>(p.base, i + 8 * h, t);
#pragma unroll
                for (int j = 0; j < 8; j++) b[8 * h + j] = t[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++)
                b[j] = n + j < p.n ? (dt == MECHA_F32 ? load1<MECHA_F32>(p.base, i + j) : dt == MECHA_F16 ? load1<MECHA_F16>(p.base, i + j) : load1<MECHA_BF16>(p.base, i + j)) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) {
            if (p.flags) poison_in = __builtin_fmaf(b[j], 0.0f, poison_in);
            r[j] = __builtin_fmaf(acc[j], p.alpha, b[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) r[j] = acc[j] * p.alpha;
    }
    if (whole) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = r[8 * h + j];
            store8<OUT_DT>(p.out, i + 8 * h, t);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (n + j < p.n) store1<OUT_DT>(p.out, i + j, r[j]);
    }
    if (p.flags) {
        bool nan = poison_in != 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            if (n + j < p.n) {
                poison_out = __builtin_fmaf(r[j], 0.0f, poison_out);
                nan |= r[j] != r[j];
            }
        }
        if (nan || poison_out != 0.0f) atomicOr(p.flags, (nan ? MECHA_FLAG_INPUT_NONFINITE : 0u) | (poison_out != 0.0f ? MECHA_FLAG_OUTPUT_NONFINITE : 0u));
    }
}

// Scales of a tile's 128 rows, CH words each: four blocks a word for the matrix unit, else a float a block.
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
                if constexpr (MODE == EXACT_E8M0) v = __float_as_uint(e8m0_to_f32(static_cast<const uint8_t *>(s)[row * pitch + kb]));
                else v = __float_as_uint(static_cast<const float *>(s)[row * pitch + kb]);
            }
        }
        to[w][r] = v;
    }
}

// 128 x 128 outputs, 4 waves of 64 x 64; a K step is one block of 128, two stages of 32 KiB in LDS, the next one in flight while
// this one is multiplied; two workgroups a CU.
template <int MODE, int OUT_DT>
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
            const int ra = wm + 16 * i + r, rb = wn + 16 * (r >> 2) + 4 * i + (r & 3);
            u32x4 a0 = *reinterpret_cast<const u32x4 *>(la + ra * 128 + 16 * ((2 * g) ^ swz_a(ra)));
            u32x4 a1 = *reinterpret_cast<const u32x4 *>(la + ra * 128 + 16 * ((2 * g + 1) ^ swz_a(ra)));
            u32x4 b0 = *reinterpret_cast<const u32x4 *>(lb + rb * 128 + 16 * ((2 * g) ^ swz_b(rb)));
            u32x4 b1 = *reinterpret_cast<const u32x4 *>(lb + rb * 128 + 16 * ((2 * g + 1) ^ swz_b(rb)));
            if (last) {                                                           // bytes behind column k are not the matrix's
                a0 = first_bytes(a0, tail - 32 * g); a1 = first_bytes(a1, tail - 32 * g - 16);
                b0 = first_bytes(b0, tail - 32 * g); b1 = first_bytes(b1, tail - 32 * g - 16);
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
                kbs[i] = s_b[w][wn + 16 * (r >> 2) + 4 * i + (r & 3)] >> sh;
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int f = 0; f < 4; f++)
                    acc[i][f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa[i], acc[i][f], 0, 0, 0, (int)kbs[f], 0, (int)ka[i]);
        } else {
            const int w = (int)kb & (CH - 1);
            float sa[4];
            f32x4v sb[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sa[i] = __uint_as_float(s_a[w][wm + 16 * i + r]);
                sb[i] = *reinterpret_cast<const f32x4v *>(&s_b[w][wn + 16 * g + 4 * i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int f = 0; f < 4; f++) {
                    f32x4v d = {0, 0, 0, 0};
                    if constexpr (MODE == F32_SCALES) d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa[i], d, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
                    else d = exact_block(fb[f], fa[i], d);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][f][e] = __builtin_fmaf(d[e], sa[i] * sb[f][e], acc[i][f][e]);
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
    const bool vec = p.n % 8 == 0 && mecha_aligned16(p.out) && (p.base == nullptr || mecha_aligned16(p.base));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float row[16];
#pragma unroll
        for (int f = 0; f < 4; f++)
#pragma unroll
            for (int e = 0; e < 4; e++) row[4 * f + e] = acc[i][f][e];
        store_row16<OUT_DT>(p, m0 + wm + 16 * i + r, n0 + wn + 16 * g, row, vec);
    }
}

// 8 contiguous columns of one output row where rows start 16-byte aligned and base has the result's type
template <int OUT_DT, bool BASE>
__device__ __forceinline__ void store_row8(const ProductParams &p, int64_t i, const float (&acc)[8]) {
    float r[8], poison_in = 0.0f;
    if constexpr (BASE) {
        float b[8];
        load8<OUT_DT>(p.base, i, b);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            poison_in = __builtin_fmaf(b[j], 0.0f, poison_in);
            r[j] = __builtin_fmaf(acc[j], p.alpha, b[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = acc[j] * p.alpha;
    }
    store8<OUT_DT>(p.out, i, r);
    if (p.flags) {
        float poison = 0.0f;
        bool nan = poison_in != 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) { poison = __builtin_fmaf(r[j], 0.0f, poison); nan |= r[j] != r[j]; }
        if (nan || poison != 0.0f) atomicOr(p.flags, (nan ? MECHA_FLAG_INPUT_NONFINITE : 0u) | (poison != 0.0f ? MECHA_FLAG_OUTPUT_NONFINITE : 0u));
    }
}

// ---------------------------------------------------------------------------------------------------- large products
// 256 x 256 outputs by 8 waves of 128 x 64, one workgroup a CU that goes on from tile to tile.  A K step is one block of 128: 64 KiB of
// codes in one of two LDS stages, 32 matrix instructions a wave.  The next step's codes -- the next tile's at a tile's end -- are on their
// way while this one is multiplied, also over the epilogue; so are the scales of the next BIG_CH words of blocks.  One barrier a
// step: behind it every wave's part of this stage has landed and the other stage has been read.
// Workgroups go round the 8 XCDs, each with its own L2: an XCD gets a run of tiles, ordered so that the 32 at work at a time are 8 x 4
// tiles (2 MiB of a and 1 MiB of b at k = 1024).
constexpr int BIG = 256, BIG_THREADS = 512, BIG_CH = 4, BIG_CUS = 256, BIG_BAND = 8;
struct BigLds {
    uint8_t stage[2][2][BIG * 128];               // [stage][a, b][row][128]
    uint32_t scale[2][2][BIG_CH][BIG];            // [parity of the chunk][a, b][word][row]
};

__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int MODE, int OUT_DT, bool B_UNIFORM, bool BASE>
__global__ __launch_bounds__(BIG_THREADS, 2) void product_big_kernel(ProductParams p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds_raw[];
    BigLds &lds = *reinterpret_cast<BigLds *>(lds_raw);
    constexpr int PER = MODE == HW_SCALES ? 4 * BIG_CH : BIG_CH;                 // blocks a chunk of scales
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int wm = (wave & 1) * 128, wn = (wave >> 1) * 64;
    const int n_kb = (int)((p.k + SCALE_BLOCK - 1) / SCALE_BLOCK);
    const int tail = (int)(p.k - (int64_t)(n_kb - 1) * SCALE_BLOCK);

    // this workgroup's tiles: every (gridDim / 8)-th of its XCD's run
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    const int xcd = blockIdx.x & 7, per_xcd = gridDim.x >> 3;
    const int64_t run0 = tiles * xcd / 8, run1 = tiles * (xcd + 1) / 8;
    int64_t tile = run0 + (blockIdx.x >> 3);
    if (tile >= run1) return;
    // bands of BIG_BAND rows of tiles, down the band first
    auto place = [&](int64_t i, int64_t &m0, int64_t &n0) {
        const int band_tiles = BIG_BAND * p.tiles_n;
        const int band = (int)(i / band_tiles), in = (int)(i - (int64_t)band * band_tiles);
        const int high = p.tiles_m - band * BIG_BAND < BIG_BAND ? p.tiles_m - band * BIG_BAND : BIG_BAND;
        m0 = (int64_t)(band * BIG_BAND + in % high) * BIG;
        n0 = (int64_t)(in / high) * BIG;
    };

    // DMA: wave w brings rows 32 w .. + 31 of each side, 8 an instruction; rows behind the last one read the last one
    uint32_t oa[4], ob[4];
    const uint8_t *ga, *gb;
    auto aim = [&](int64_t m0, int64_t n0) {
        const int la = p.m - 1 - m0 < BIG ? (int)(p.m - 1 - m0) : BIG, lb = p.n - 1 - n0 < BIG ? (int)(p.n - 1 - n0) : BIG;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = 32 * wave + 8 * i + (lane >> 3), slot = lane & 7;
            oa[i] = (uint32_t)(row < la ? row : la) * (uint32_t)p.a_pitch + 16u * (uint32_t)(slot ^ swz_a(row));
            ob[i] = (uint32_t)(row < lb ? row : lb) * (uint32_t)p.b_pitch + 16u * (uint32_t)(slot ^ swz_b(row));
        }
        ga = p.a + m0 * p.a_pitch;
        gb = p.b + n0 * p.b_pitch;
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_byte *)lds_raw) + (uint32_t)wave * 4096u;
    auto issue = [&](int kb, int to) {
        const uint32_t dst = lds0 + (uint32_t)to * (2 * BIG * 128);
        dma4(ga + (int64_t)kb * SCALE_BLOCK, oa[0], oa[1], oa[2], oa[3], dst);
        dma4(gb + (int64_t)kb * SCALE_BLOCK, ob[0], ob[1], ob[2], ob[3], dst + BIG * 128);
    };
    // scales: thread (side, row) holds the words of a chunk between load and store
    uint32_t held[BIG_CH];
    const int side = __builtin_amdgcn_readfirstlane(t >> 8), srow = t & 255;
    auto load_scales = [&](int64_t m0, int64_t n0, int kb0) {
        const void *s = side ? p.sb : p.sa;
        const int64_t rows = side ? p.n : p.m, pitch = side ? p.sb_pitch : p.sa_pitch;
        int64_t row = (side ? n0 : m0) + srow;
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
            const float *at = static_cast<const float *>(s) + row * pitch;
#pragma unroll
            for (int w = 0; w < BIG_CH; w++) held[w] = __float_as_uint(at[kb0 + w < n_kb ? kb0 + w : n_kb - 1]);
        }
    };
    auto put_scales = [&](int to) {
#pragma unroll
        for (int w = 0; w < BIG_CH; w++) lds.scale[to][side][w][srow] = held[w];
    };

    // fragment addresses inside a stage and a row of scales
    uint32_t fa_at[2], fb_at[2];                                                  // of fragment 0; the others are 16 rows (a), 4 rows (b) on, in the same slots
    const int ra0 = wm + r, rb0 = wn + 16 * (r >> 2) + (r & 3);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        fa_at[h] = (uint32_t)(ra0 * 128 + 16 * ((2 * g + h) ^ swz_a(ra0)));
        fb_at[h] = (uint32_t)(rb0 * 128 + 16 * ((2 * g + h) ^ swz_b(rb0)));
    }

    f32x4v acc[8][4];                                                             // [a fragment][b fragment]
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int f = 0; f < 4; f++) acc[i][f] = f32x4v{0, 0, 0, 0};
    };
    int64_t m0, n0, nm0 = 0, nn0 = 0;
    place(tile, m0, n0);
    aim(m0, n0);
    issue(0, 0);
    load_scales(m0, n0, 0);
    put_scales(0);
    clear();
    wait_vm0();
    int stage = 0, chunk = 0, kb = 0;
#pragma clang loop unroll(disable)
    while (true) {
        const bool last = kb + 1 == n_kb, more = tile + per_xcd < run1;
        lds_barrier();
        if (last && tail < SCALE_BLOCK) {                                         // bytes behind column k are not the matrix's
            const int row = t >> 1;                                               // thread: half of a row of each side
#pragma clang loop unroll(disable)
            for (int c = 0; c < 8; c++) {
                const int sd = c >> 2, piece = 4 * (t & 1) + (c & 3), left = tail - 16 * piece;
                if (left < 16) {
                    u32x4 *at = reinterpret_cast<u32x4 *>(&lds.stage[stage][sd][row * 128 + 16 * (piece ^ (sd ? swz_b(row) : swz_a(row)))]);
                    *at = first_bytes(*at, left);
                }
            }
            lds_barrier();
        }
        if (last && more) {
            place(tile + per_xcd, nm0, nn0);
            aim(nm0, nn0);
        }
        const int next_kb = last ? 0 : kb + 1;
        const bool refill = last ? more : next_kb % PER == 0;
        if (!last || more) issue(next_kb, stage ^ 1);
        if (refill) load_scales(last ? nm0 : m0, last ? nn0 : n0, next_kb);
        {
            const uint8_t *la = &lds.stage[stage][0][0], *lb = &lds.stage[stage][1][0];
            i32x8 fb[4];
#pragma unroll
            for (int f = 0; f < 4; f++)
                fb[f] = join(*reinterpret_cast<const u32x4 *>(lb + fb_at[0] + 512 * f), *reinterpret_cast<const u32x4 *>(lb + fb_at[1] + 512 * f));
            // fragment i + 1 of a is read while fragment i is multiplied
            const int w = MODE == HW_SCALES ? (kb / 4) & (BIG_CH - 1) : kb & (BIG_CH - 1), sh = 8 * (kb & 3);
            auto read_a = [&](int i) { return join(*reinterpret_cast<const u32x4 *>(la + fa_at[0] + 2048 * i), *reinterpret_cast<const u32x4 *>(la + fa_at[1] + 2048 * i)); };
            const uint32_t *sa_row = &lds.scale[chunk][0][w][ra0], *sb_row = &lds.scale[chunk][1][w][0];
            uint32_t sb[4];                                                       // matrix unit's scales of b
            f32x4v sbf[4];
            float sb1 = 0.0f;
            if constexpr (MODE == HW_SCALES) {
#pragma unroll
                for (int f = 0; f < (B_UNIFORM ? 1 : 4); f++) sb[f] = sb_row[B_UNIFORM ? wn : rb0 + 4 * f] >> sh;
            } else if constexpr (B_UNIFORM) sb1 = __uint_as_float(sb_row[wn]);
            else {
#pragma unroll
                for (int f = 0; f < 4; f++) sbf[f] = *reinterpret_cast<const f32x4v *>(&sb_row[wn + 16 * g + 4 * f]);
            }
            i32x8 fa = read_a(0);
            uint32_t sa = sa_row[0];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                i32x8 fa_next = fa;
                uint32_t sa_next = sa;
                if (i < 7) { fa_next = read_a(i + 1); sa_next = sa_row[16 * (i + 1)]; }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (MODE == HW_SCALES) {
                    const uint32_t sah = sa >> sh;
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        acc[i][f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa, acc[i][f], 0, 0, 0, (int)sb[B_UNIFORM ? 0 : f], 0, (int)sah);
                } else {
                    const float sf = __uint_as_float(sa) * (B_UNIFORM ? sb1 : 1.0f);
                    f32x4v d[4];
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        d[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[f], fa, f32x4v{0, 0, 0, 0}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
#pragma unroll
                    for (int f = 0; f < 4; f++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][f][e] = __builtin_fmaf(d[f][e], B_UNIFORM ? sf : sf * sbf[f][e], acc[i][f][e]);
                }
                // (nothing is executed here: the sums of this fragment are made at this point, not sunk to where they are stored)
                asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]));
                __builtin_amdgcn_sched_barrier(0);
                fa = fa_next;
                sa = sa_next;
            }
        }
        wait_vm0();                                                               // the next stage; before the stores, which the same counter counts
        if (refill) { put_scales(chunk ^ 1); chunk ^= 1; }
        stage ^= 1;
        kb = next_kb;
        if (last) {
            const int64_t n = n0 + wn + 16 * g;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int64_t m = m0 + wm + 16 * i + r;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float row[8];
#pragma unroll
                    for (int f = 0; f < 2; f++)
#pragma unroll
                        for (int e = 0; e < 4; e++) row[4 * f + e] = acc[i][2 * h + f][e];
                    if (m < p.m && n + 8 * h < p.n) store_row8<OUT_DT, BASE>(p, m * p.n + n + 8 * h, row);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (!more) break;
            tile += per_xcd; m0 = nm0; n0 = nn0;
            clear();
        }
    }
}

}  // namespace

extern "C" {

int mecha_block_product(const void *a, int64_t a_pitch, const void *a_scales, int64_t a_scale_pitch, int a_tile, const void *b, int64_t b_pitch,
                        const void *b_scales, int64_t b_scale_pitch, int b_tile, int scale_dtype, const void *base, void *out, int64_t m,
                        int64_t n, int64_t k, int base_dtype, int out_dtype, float alpha, uint32_t *flags, void *stream) {
    MECHA_REQUIRE(m >= 0 && n >= 0 && k >= 1, "bad product: %lld x %lld x %lld", (long long)m, (long long)n, (long long)k);
    MECHA_REQUIRE(mecha_valid_dtype(out_dtype) && (base == nullptr || mecha_valid_dtype(base_dtype)), "unknown dtype code (base %d, out %d)", base_dtype, out_dtype);
    MECHA_REQUIRE(scale_dtype == MECHA_SCALE_F32 || scale_dtype == MECHA_SCALE_E8M0, "unknown scale dtype %d", scale_dtype);
    if (m == 0 || n == 0) return MECHA_OK;
    MECHA_REQUIRE(out != nullptr, "out is NULL");
    int st = mecha_check_blocks("a", a, m, k, a_pitch, a_scales, a_scale_pitch);
    if (st) return st;
    st = mecha_check_blocks("b", b, n, k, b_pitch, b_scales, b_scale_pitch);
    if (st) return st;
    MECHA_REQUIRE(a_pitch <= (1 << 24) && b_pitch <= (1 << 24), "rows of more than 2^24 bytes (%lld, %lld)", (long long)a_pitch, (long long)b_pitch);
    const int64_t tm = (m + 127) / 128, tn = (n + 127) / 128;
    MECHA_REQUIRE(tm * tn < (1ll << 24), "%lld x %lld outputs are beyond one launch", (long long)m, (long long)n);
    ProductParams p{static_cast<const uint8_t *>(a), a_pitch, a_scales, a_scale_pitch, a_tile, static_cast<const uint8_t *>(b), b_pitch, b_scales,
                    b_scale_pitch, b_tile, base, out, m, n, k, base_dtype, out_dtype, alpha, flags, (int)tm, (int)tn};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool e8m0 = scale_dtype == MECHA_SCALE_E8M0;
    const int64_t bm = (m + BIG - 1) / BIG, bn = (n + BIG - 1) / BIG;
    const bool big = out_dtype != MECHA_F32 && bm * bn >= 64 && k > 3 * SCALE_BLOCK && n % 8 == 0 && mecha_aligned16(out)
                     && (base == nullptr || (base_dtype == out_dtype && mecha_aligned16(base)));
    if (big) { p.tiles_m = (int)bm; p.tiles_n = (int)bn; }
    int rc = MECHA_OK;
    auto go = [&](auto mode, auto dt) {
        constexpr int MODE = decltype(mode)::value, DT = decltype(dt)::value;
        if constexpr (DT != MECHA_F32) {
            if (big) {
                auto large = [&](auto uniform, auto based) {
                    constexpr bool U = decltype(uniform)::value, B = decltype(based)::value;
                    auto *const kernel = &product_big_kernel<MODE, DT, U, B>;
                    const hipError_t room = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(BigLds));
                    if (room != hipSuccess) { mecha_set_error("%zu bytes of LDS: %s", sizeof(BigLds), hipGetErrorString(room)); rc = MECHA_ERR_HIP; return; }
                    const int64_t grid = bm * bn < BIG_CUS ? (bm * bn + 7) / 8 * 8 : BIG_CUS;
                    MECHA_LAUNCH(MK_BLOCKS_PRODUCT, kernel, dim3((unsigned)grid), dim3(BIG_THREADS), sizeof(BigLds), s, p);
                };
                auto with_base = [&](auto uniform) { if (base) large(uniform, std::true_type{}); else large(uniform, std::false_type{}); };
                if (b_tile) with_base(std::true_type{}); else with_base(std::false_type{});
                return;
            }
        }
        MECHA_LAUNCH(MK_BLOCKS_PRODUCT, (product_kernel<MODE, DT>), dim3((unsigned)(tm * tn)), dim3(MECHA_BLOCK), 0, s, p);
    };
    auto with_mode = [&](auto power, auto real, auto dt) { if (e8m0) go(power, dt); else go(real, dt); };
    typedef std::integral_constant<int, HW_SCALES> Hw;
    typedef std::integral_constant<int, F32_SCALES> F32;
    switch (out_dtype) {
        case MECHA_F32: with_mode(std::integral_constant<int, EXACT_E8M0>{}, std::integral_constant<int, EXACT_F32>{}, std::integral_constant<int, MECHA_F32>{}); break;
        case MECHA_F16: with_mode(Hw{}, F32{}, std::integral_constant<int, MECHA_F16>{}); break;
        default: with_mode(Hw{}, F32{}, std::integral_constant<int, MECHA_BF16>{}); break;
    }
    if (rc) return rc;
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

}  // extern "C"
