// blocks.hip -- 8-bit weights: e4m3 codes with a scale for each block of 128, made from and turned back into 16- and 32-bit keys.
//
// A block-scaled matrix: codes [rows][pitch] (pitch a multiple of 128 bytes, at least the columns rounded up to 128) and scales
// [rows or ceil(rows / 128)][ceil(cols / 128)]: a scale for 128 columns of one row, or of a 128 x 128 square.  value = code * scale.
#include <type_traits>
#include "blocks.h"

namespace {

// ------------------------------------------------------------------------------------------------------------- cast
struct CastParams {
    const void *a;
    int64_t rows, cols, ld;            // elements
    uint8_t *q; int64_t q_pitch;       // bytes; q may be NULL (square kernel)
    uint8_t *s; int64_t s_pitch;
    uint8_t *qt; int64_t qt_pitch;     // transposed, may be NULL
    uint8_t *st; int64_t st_pitch;
    uint32_t *flags;
};

// 8 elements as they lie in memory: maxima are taken on the magnitudes' bits, two 16-bit elements an instruction, and gfx950 converts
// two elements of any of the three types straight to codes of x / 2^e.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
template <int DT> constexpr int WORDS = DT == MECHA_F32 ? 8 : 4;
template <int DT> struct Vec8 { uint32_t w[WORDS<DT>]; };
template <int DT> constexpr uint32_t MAG = DT == MECHA_F32 ? 0x7fffffffu : 0x7fff7fffu;
template <int DT> constexpr uint32_t INF = DT == MECHA_F32 ? 0x7f800000u : DT == MECHA_BF16 ? 0x7f80u : 0x7c00u;

// 8 elements of row `row` from column c; zeros behind the last column
template <int DT>
__device__ __forceinline__ Vec8<DT> load_row8(const CastParams &p, int64_t row, int64_t c) {
    Vec8<DT> v;
    const int64_t i = row * p.ld + c;
    if (c + 8 <= p.cols) {
        const u32x4_any *at = reinterpret_cast<const u32x4_any *>(static_cast<const char *>(p.a) + i * (DT == MECHA_F32 ? 4 : 2));
#pragma unroll
        for (int h = 0; h < WORDS<DT> / 4; h++) {
            // read once, past the caches; but float32's two halves of a line come with two instructions, the second out of the cache (10240 x 1280 both
            // ways 22.2 us past it, 20.6 through it; 8269 x 5120 bfloat16 37.9 us past it, 40.4 through it)
            const u32x4 r = DT == MECHA_F32 ? at[h] : __builtin_nontemporal_load(at + h);
            v.w[4 * h] = r.x; v.w[4 * h + 1] = r.y; v.w[4 * h + 2] = r.z; v.w[4 * h + 3] = r.w;
        }
    } else if constexpr (DT == MECHA_F32) {
#pragma unroll
        for (int j = 0; j < 8; j++) v.w[j] = c + j < p.cols ? static_cast<const uint32_t *>(p.a)[i + j] : 0u;
    } else {
        const uint16_t *at = static_cast<const uint16_t *>(p.a) + i;
#pragma unroll
        for (int j = 0; j < 4; j++) v.w[j] = (c + 2 * j < p.cols ? at[2 * j] : 0u) | (c + 2 * j + 1 < p.cols ? (uint32_t)at[2 * j + 1] << 16 : 0u);
    }
    return v;
}
// element by element, or both halves
template <int DT>
__device__ __forceinline__ uint32_t max_mag(uint32_t a, uint32_t b) {
    if constexpr (DT == MECHA_F32) return a > b ? a : b;
    else return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// the larger half of a word of two
template <int DT>
__device__ __forceinline__ uint32_t one_mag(uint32_t m) {
    if constexpr (DT == MECHA_F32) return m;
    else return max_mag<DT>(m, m >> 16) & 0xffffu;
}
// max over the 16 lanes of a row of lanes, by rotations within it
template <int DT>
__device__ __forceinline__ uint32_t max_mag16(uint32_t m) {
    m = max_mag<DT>(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x128, 0xf, 0xf, true));
    m = max_mag<DT>(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x124, 0xf, 0xf, true));
    m = max_mag<DT>(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x122, 0xf, 0xf, true));
    return max_mag<DT>(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x121, 0xf, 0xf, true));
}
// exponent of a block from its largest magnitude, one of DT's
template <int DT>
__device__ __forceinline__ int exponent_of_mag(uint32_t m) {
    if constexpr (DT == MECHA_F32) return block_exponent(__uint_as_float(m));
    else if constexpr (DT == MECHA_BF16) return block_exponent(__uint_as_float(m << 16));
    else return block_exponent(f16_bits_to_f32(m));
}
// codes of two elements into half `HI` of r
template <int DT, bool HI>
__device__ __forceinline__ s16x2 codes2(s16x2 r, uint32_t lo, uint32_t hi, float scale) {     // 16-bit types: both elements in lo
    if constexpr (DT == MECHA_F32) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __uint_as_float(lo), __uint_as_float(hi), scale, HI);
    else if constexpr (DT == MECHA_BF16) return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, lo), scale, HI);
    else return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, lo), scale, HI);
}
template <int DT>
__device__ __forceinline__ u32x2 codes8(const Vec8<DT> &v, float scale) {
    s16x2 r0 = {0, 0}, r1 = {0, 0};
    if constexpr (DT == MECHA_F32) {
        r0 = codes2<DT, false>(r0, v.w[0], v.w[1], scale); r0 = codes2<DT, true>(r0, v.w[2], v.w[3], scale);
        r1 = codes2<DT, false>(r1, v.w[4], v.w[5], scale); r1 = codes2<DT, true>(r1, v.w[6], v.w[7], scale);
    } else {
        r0 = codes2<DT, false>(r0, v.w[0], 0, scale); r0 = codes2<DT, true>(r0, v.w[1], 0, scale);
        r1 = codes2<DT, false>(r1, v.w[2], 0, scale); r1 = codes2<DT, true>(r1, v.w[3], 0, scale);
    }
    return u32x2{__builtin_bit_cast(uint32_t, r0), __builtin_bit_cast(uint32_t, r1)};
}
template <int DT>
__device__ __forceinline__ uint32_t mag8(const Vec8<DT> &v) {
    uint32_t m = v.w[0] & MAG<DT>;
#pragma unroll
    for (int j = 1; j < WORDS<DT>; j++) m = max_mag<DT>(m, v.w[j] & MAG<DT>);
    return m;
}
// inf and NaN out of 8 elements: they become 0 and their bits are set (rare)
template <int DT>
__device__ __forceinline__ uint32_t take_out(Vec8<DT> &v) {
    uint32_t out = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t w = DT == MECHA_F32 ? v.w[j % WORDS<DT>] : (v.w[j / 2] >> (16 * (j & 1))) & 0xffffu;
        if ((w & INF<DT>) == INF<DT>) {
            out |= 1u << j;
            if constexpr (DT == MECHA_F32) v.w[j] = 0u;
            else v.w[j / 2] &= j & 1 ? 0xffffu : 0xffff0000u;
        }
    }
    return out;
}
__device__ __forceinline__ u32x2 with_nan(u32x2 codes, uint32_t bits) {
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (bits & (1u << j)) codes[j / 4] = (codes[j / 4] & ~(0xffu << (8 * (j & 3)))) | (0x7fu << (8 * (j & 3)));
    return codes;
}

// Codes of float32 keys leave past the caches (10240 x 1280 both ways 20.6 -> 18.7 us, 8269 x 2560 rows 20.3 -> 19.6); of 16-bit keys, whose
// loads go past them already, that costs 36.0 -> 37.4 us at 8269 x 5120 both ways.
template <int DT>
__device__ __forceinline__ void store_codes(uint8_t *at, u32x2 codes) {
    if constexpr (DT == MECHA_F32) __builtin_nontemporal_store(codes, reinterpret_cast<u32x2 *>(at));
    else *reinterpret_cast<u32x2 *>(at) = codes;
}

// Rows form, codes of the matrix as it lies: 16 lanes own a block of 128, 8 elements each; one pass over memory, the block's
// maximum goes round the 16 lanes.  Dividing by a power of two is exact, the only rounding is the code's.  Bound by memory: 8269 x 5120
// bfloat16 25 us (5.1 TB/s), 77 x 768 2.6 us, which is a launch and one trip to memory.
template <int DT>
__global__ __launch_bounds__(MECHA_BLOCK) void cast_rows_kernel(CastParams p, int64_t n_groups, int64_t blocks_per_row) {
    const int64_t group = (int64_t)blockIdx.x * (MECHA_BLOCK / 16) + (threadIdx.x >> 4);
    if (group >= n_groups) return;
    const int64_t row = n_groups < (1ll << 31) ? (int64_t)((uint32_t)group / (uint32_t)blocks_per_row) : group / blocks_per_row;
    const int64_t kb = group - row * blocks_per_row;
    const int l = threadIdx.x & 15;
    const int64_t c = kb * SCALE_BLOCK + 8 * l;
    Vec8<DT> v = load_row8<DT>(p, row, c);
    uint32_t m = one_mag<DT>(mag8<DT>(v)), nan = 0;
    if (m >= INF<DT>) {
        nan = take_out<DT>(v);
        m = one_mag<DT>(mag8<DT>(v));
    }
    const int e = exponent_of_mag<DT>(max_mag16<DT>(m));
    u32x2 codes = codes8<DT>(v, scale_bits(e + 127));
    if (nan) codes = with_nan(codes, nan);
    store_codes<DT>(p.q + row * p.q_pitch + c, codes);
    if (l == 0) p.s[row * p.s_pitch + kb] = (uint8_t)(e + 127);
    if (nan && p.flags) atomicOr(p.flags, MECHA_FLAG_INPUT_NONFINITE);
}

// 128 x 128 squares: tile scales and / or codes of the transposed matrix.  Thread (t / 16, t % 16) holds rows 8 (t / 16) .. + 7 and
// columns 8 (t % 16) .. + 7 in registers, so that a row's maximum stays within 16 lanes, a column's takes one exchange between the
// waves, and an 8 x 8 square of codes turns over in registers; transposed codes go through 16 KiB of LDS to leave as whole
// 128-byte lines.  Bound by memory, one pass over the key for both matrices: 10240 x 1280 float32 both ways 19 us (4.2 TB/s, 14 us with the key in
// the last-level cache; a grid of all
// the squares at once, which first all read and then all write), 8269 x 5120 bfloat16 both ways with scales of their own 36 us (4.7 TB/s).
template <int DT, bool TILE>
__global__ __launch_bounds__(MECHA_BLOCK, DT == MECHA_F32 ? 3 : 5) void cast_square_kernel(CastParams p, int64_t squares_per_row) {
    constexpr int W = WORDS<DT>;
    __shared__ uint32_t wave_max[4][16][W];
    __shared__ u32x2 turned[SCALE_BLOCK][16];
    const int t = threadIdx.x, tr = t >> 4, tc = t & 15, lane = t & 63, wave = t >> 6;
    const int64_t sr = blockIdx.x / squares_per_row, sc = blockIdx.x - sr * squares_per_row;
    const int64_t row0 = sr * SCALE_BLOCK + 8 * tr, c = sc * SCALE_BLOCK + 8 * tc;
    Vec8<DT> v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (row0 + i < p.rows) v[i] = load_row8<DT>(p, row0 + i, c);
        else {
#pragma unroll
            for (int j = 0; j < W; j++) v[i].w[j] = 0u;
        }
    }
    // columns first: over this thread's rows, and from there whether anything is inf or NaN
    uint32_t cmax[W], nan[2] = {0, 0}, all = 0;      // nan: 8 bits a row
    auto columns = [&]() {
        all = 0;
#pragma unroll
        for (int j = 0; j < W; j++) {
            cmax[j] = v[0].w[j] & MAG<DT>;
#pragma unroll
            for (int i = 1; i < 8; i++) cmax[j] = max_mag<DT>(cmax[j], v[i].w[j] & MAG<DT>);
            all = max_mag<DT>(all, cmax[j]);
        }
    };
    columns();
    const bool bad = one_mag<DT>(all) >= INF<DT>;
    if (bad) {
#pragma unroll
        for (int i = 0; i < 8; i++) nan[i >> 2] |= take_out<DT>(v[i]) << (8 * (i & 3));
        columns();
        if (p.flags) atomicOr(p.flags, MECHA_FLAG_INPUT_NONFINITE);
    }
    int tile_e = 0;
    if constexpr (TILE) {
        const uint32_t m = max_mag16<DT>(one_mag<DT>(all));
        if (tc == 0) wave_max[wave][tr & 3][0] = m;
        lds_barrier();
        uint32_t o = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) o = o > wave_max[i >> 2][i & 3][0] ? o : wave_max[i >> 2][i & 3][0];
        tile_e = exponent_of_mag<DT>(o);
        if (t == 0) {
            if (p.q) p.s[sr * p.s_pitch + sc] = (uint8_t)(tile_e + 127);
            if (p.qt) p.st[sc * p.st_pitch + sr] = (uint8_t)(tile_e + 127);
        }
    } else {
        // a column's maximum: the wave's 4 row groups (lanes 16 and 32 apart) here, the 4 waves behind the barrier
#pragma unroll
        for (int j = 0; j < W; j++) {
            const auto x = __builtin_amdgcn_permlane32_swap(cmax[j], cmax[j], false, false);
            const uint32_t m = max_mag<DT>(x[0], x[1]);
            const auto y = __builtin_amdgcn_permlane16_swap(m, m, false, false);
            cmax[j] = max_mag<DT>(y[0], y[1]);
        }
        if (lane < 16) {
#pragma unroll
            for (int j = 0; j < W; j++) wave_max[wave][lane][j] = cmax[j];
        }
    }
    // the straight codes leave while the columns' maxima meet
    if (p.q) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            int e[2] = {tile_e, tile_e};
            if constexpr (!TILE) {
                if constexpr (DT == MECHA_F32) {
                    e[0] = exponent_of_mag<DT>(max_mag16<DT>(mag8<DT>(v[i])));
                    e[1] = exponent_of_mag<DT>(max_mag16<DT>(mag8<DT>(v[i + 1])));
                } else {                             // two rows a word go round the lanes together
                    const uint32_t m = max_mag16<DT>(one_mag<DT>(mag8<DT>(v[i])) | one_mag<DT>(mag8<DT>(v[i + 1])) << 16);
                    e[0] = exponent_of_mag<DT>(m & 0xffffu);
                    e[1] = exponent_of_mag<DT>(m >> 16);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int64_t row = row0 + i + h;
                u32x2 codes = codes8<DT>(v[i + h], scale_bits(e[h] + 127));
                if (bad) codes = with_nan(codes, nan[(i + h) >> 2] >> (8 * ((i + h) & 3)));
                if (row < p.rows) {
                    store_codes<DT>(p.q + row * p.q_pitch + c, codes);
                    if (!TILE && tc == 0) p.s[row * p.s_pitch + sc] = (uint8_t)(e[h] + 127);
                }
            }
        }
    }
    int ce[8];                                       // exponents of this thread's columns
    if constexpr (TILE) {
#pragma unroll
        for (int j = 0; j < 8; j++) ce[j] = tile_e;
    } else {
        lds_barrier();
#pragma unroll
        for (int j = 0; j < W; j++) {
            uint32_t m = wave_max[0][tc][j];
#pragma unroll
            for (int i = 1; i < 4; i++) m = max_mag<DT>(m, wave_max[i][tc][j]);
            if constexpr (DT == MECHA_F32) ce[j] = exponent_of_mag<DT>(m);
            else { ce[2 * j] = exponent_of_mag<DT>(m & 0xffffu); ce[2 * j + 1] = exponent_of_mag<DT>(m >> 16); }
        }
        if (tr == 0) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < p.cols) p.st[(c + j) * p.st_pitch + sr] = (uint8_t)(ce[j] + 127);
        }
    }
    if (p.qt) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float scale = scale_bits(ce[j] + 127);
            u32x2 codes;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                s16x2 r = {0, 0};
                const int i = 4 * h;
                if constexpr (DT == MECHA_F32) {
                    r = codes2<DT, false>(r, v[i].w[j], v[i + 1].w[j], scale);
                    r = codes2<DT, true>(r, v[i + 2].w[j], v[i + 3].w[j], scale);
                } else {                         // the column's halves of two rows
                    const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
                    r = codes2<DT, false>(r, __builtin_amdgcn_perm(v[i + 1].w[j / 2], v[i].w[j / 2], pick), 0, scale);
                    r = codes2<DT, true>(r, __builtin_amdgcn_perm(v[i + 3].w[j / 2], v[i + 2].w[j / 2], pick), 0, scale);
                }
                codes[h] = __builtin_bit_cast(uint32_t, r);
            }
            if (bad) {
                uint32_t column = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) column |= ((nan[i >> 2] >> (8 * (i & 3) + j)) & 1u) << i;
                codes = with_nan(codes, column);
            }
            // slot XOR the column's group: 16 lanes (columns 8 apart, 1 KiB) write to 16 different slots
            turned[8 * tc + j][tr ^ tc] = codes;
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int col = 16 * i + tr;
            const u32x2 w = turned[col][tc ^ (col >> 3)];
            const int64_t oc = sc * SCALE_BLOCK + col;
            if (oc < p.cols) store_codes<DT>(p.qt + oc * p.qt_pitch + sr * SCALE_BLOCK + 8 * tc, w);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ uncast
// 8 codes a thread, one scale for them.  Bound by memory: 5120 x 2816 to bfloat16 9.8 us (4.4 TB/s).
template <int OUT_DT, bool E8M0, bool VEC>
__global__ __launch_bounds__(MECHA_BLOCK) void uncast_kernel(const uint8_t *q, int64_t q_pitch, const void *s, int64_t s_pitch, int tile,
                                                             int64_t rows, int64_t cols, int64_t vec_per_row, void *out, uint32_t *flags) {
    const int64_t i = (int64_t)blockIdx.x * MECHA_BLOCK + threadIdx.x;
    if (i >= rows * vec_per_row) return;
    const int64_t row = rows * vec_per_row < (1ll << 31) ? (int64_t)((uint32_t)i / (uint32_t)vec_per_row) : i / vec_per_row;
    const int64_t c = 8 * (i - row * vec_per_row);
    const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(q + row * q_pitch + c));
    const int64_t si = (tile ? row / SCALE_BLOCK : row) * s_pitch + c / SCALE_BLOCK;
    float scale;
    if constexpr (E8M0) scale = e8m0_to_f32(static_cast<const uint8_t *>(s)[si]);
    else scale = static_cast<const float *>(s)[si];
    float v[8];
    unpack_e4m3x4(w.x, v);
    unpack_e4m3x4(w.y, v + 4);
    bool bad_in = nonfinite_f32(scale), bad_out = false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        bad_in |= c + j < cols && nonfinite_f32(v[j]);
        v[j] *= scale;
        if constexpr (OUT_DT == MECHA_F16) asm volatile("" : "+v"(v[j]));    // (or the product and its conversion become one instruction with one rounding)
        bad_out |= c + j < cols && !(fabsf(v[j]) < stored_as_inf(OUT_DT));
    }
    if (VEC) store8<OUT_DT, true>(out, row * cols + c, v);
    else if (c + 8 <= cols) {
        if constexpr (OUT_DT == MECHA_F32) {
            u32x4_any *at = reinterpret_cast<u32x4_any *>(static_cast<float *>(out) + row * cols + c);
#pragma unroll
            for (int h = 0; h < 2; h++)
                at[h] = u32x4{__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])};
        } else {
            u32x4 x;
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] = OUT_DT == MECHA_BF16 ? f32_to_bf16_bits(v[2 * j]) | f32_to_bf16_bits(v[2 * j + 1]) << 16 : f32_to_f16_bits(v[2 * j]) | f32_to_f16_bits(v[2 * j + 1]) << 16;
            *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(out) + row * cols + c) = x;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c + j < cols) store1<OUT_DT>(out, row * cols + c + j, v[j]);
    }
    if ((bad_in || bad_out) && flags) atomicOr(flags, (bad_in ? MECHA_FLAG_INPUT_NONFINITE : 0u) | (bad_out ? MECHA_FLAG_OUTPUT_NONFINITE : 0u));
}

}  // namespace

extern "C" {

int mecha_cast_blocks(const void *a, int64_t row_stride, int in_dtype, const mecha_block_matrix *straight, const mecha_block_matrix *transposed,
                      uint32_t *flags, void *stream) {
    MECHA_REQUIRE(straight != nullptr || transposed != nullptr, "neither codes nor transposed codes are asked for");
    MECHA_REQUIRE(mecha_valid_dtype(in_dtype), "unknown dtype code %d", in_dtype);
    const int64_t rows = straight ? straight->rows : transposed->cols, cols = straight ? straight->cols : transposed->rows;
    const int tile = straight ? straight->tile : transposed->tile;
    for (const mecha_block_matrix *q : {straight, transposed}) {
        if (!q) continue;
        const int st = mecha_check_blocks(q == straight ? "codes" : "transposed codes", *q);
        if (st) return st;
        MECHA_REQUIRE(q->scale_dtype == MECHA_SCALE_E8M0, "a cast makes power-of-two scales");
    }
    if (straight && transposed)
        MECHA_REQUIRE(transposed->rows == cols && transposed->cols == rows && !transposed->tile == !tile, "the transposed matrix is %lld x %lld, not %lld x %lld of the same form",
                      (long long)transposed->rows, (long long)transposed->cols, (long long)cols, (long long)rows);
    if (rows == 0 || cols == 0) return MECHA_OK;
    MECHA_REQUIRE(a != nullptr && row_stride >= cols, "a is NULL or its rows overlap (stride %lld, %lld columns)", (long long)row_stride, (long long)cols);
    const size_t a_bytes = ((size_t)(rows - 1) * row_stride + cols) * mecha_dtype_size(in_dtype);
    for (const mecha_block_matrix *q : {straight, transposed}) {
        if (!q) continue;
        const size_t codes = mecha_codes_bytes(*q), scales = mecha_scales_bytes(*q);
        MECHA_REQUIRE(!mecha_overlap(a, a_bytes, q->codes, codes) && !mecha_overlap(a, a_bytes, q->scales, scales) && !mecha_overlap(q->codes, codes, q->scales, scales),
                      "a cast's codes or scales share memory with the key or with each other");
    }
    if (straight && transposed)
        MECHA_REQUIRE(!mecha_codes_overlap(*straight, *transposed) && !mecha_overlap(straight->codes, mecha_codes_bytes(*straight), transposed->scales, mecha_scales_bytes(*transposed))
                      && !mecha_overlap(straight->scales, mecha_scales_bytes(*straight), transposed->codes, mecha_codes_bytes(*transposed))
                      && !mecha_overlap(straight->scales, mecha_scales_bytes(*straight), transposed->scales, mecha_scales_bytes(*transposed)),
                      "a cast's two matrices share memory");
    CastParams p{a, rows, cols, row_stride, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, flags};
    if (straight) { p.q = static_cast<uint8_t *>(straight->codes); p.q_pitch = straight->pitch; p.s = static_cast<uint8_t *>(straight->scales); p.s_pitch = straight->scale_pitch; }
    if (transposed) { p.qt = static_cast<uint8_t *>(transposed->codes); p.qt_pitch = transposed->pitch; p.st = static_cast<uint8_t *>(transposed->scales); p.st_pitch = transposed->scale_pitch; }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t bc = (cols + SCALE_BLOCK - 1) / SCALE_BLOCK, br = (rows + SCALE_BLOCK - 1) / SCALE_BLOCK;
    const bool flat = transposed == nullptr && !tile;
    const int64_t blocks = flat ? (rows * bc + MECHA_BLOCK / 16 - 1) / (MECHA_BLOCK / 16) : br * bc;
    MECHA_REQUIRE(blocks * MECHA_BLOCK < (1ll << 32), "%lld x %lld is beyond one launch", (long long)rows, (long long)cols);
    dim3 grid((unsigned)blocks), block(MECHA_BLOCK);
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (flat) MECHA_LAUNCH(MK_BLOCKS_CAST, (cast_rows_kernel<DT>), grid, block, 0, s, p, rows * bc, bc);
        else if (tile) MECHA_LAUNCH(MK_BLOCKS_CAST, (cast_square_kernel<DT, true>), grid, block, 0, s, p, bc);
        else MECHA_LAUNCH(MK_BLOCKS_CAST, (cast_square_kernel<DT, false>), grid, block, 0, s, p, bc);
    };
    switch (in_dtype) {
        case MECHA_F32: go(std::integral_constant<int, MECHA_F32>{}); break;
        case MECHA_F16: go(std::integral_constant<int, MECHA_F16>{}); break;
        default: go(std::integral_constant<int, MECHA_BF16>{}); break;
    }
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

int mecha_uncast_blocks(const mecha_block_matrix *q, void *out, int out_dtype, uint32_t *flags, void *stream) {
    MECHA_REQUIRE(q != nullptr && mecha_valid_dtype(out_dtype), "no matrix, or unknown dtype code %d", out_dtype);
    const int st = mecha_check_blocks("codes", *q);
    if (st) return st;
    const int64_t rows = q->rows, cols = q->cols;
    if (rows == 0 || cols == 0) return MECHA_OK;
    MECHA_REQUIRE(out != nullptr, "out is NULL");
    const size_t out_bytes = (size_t)rows * cols * mecha_dtype_size(out_dtype);
    MECHA_REQUIRE(!mecha_overlap(out, out_bytes, q->codes, mecha_codes_bytes(*q)) && !mecha_overlap(out, out_bytes, q->scales, mecha_scales_bytes(*q)), "out shares memory with the codes or scales");
    const int64_t vec_per_row = (cols + 7) / 8, blocks = (rows * vec_per_row + MECHA_BLOCK - 1) / MECHA_BLOCK;
    MECHA_REQUIRE(blocks * MECHA_BLOCK < (1ll << 32), "%lld x %lld is beyond one launch", (long long)rows, (long long)cols);
    const bool vec = mecha_aligned16(out) && cols % 8 == 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto dt, auto e8, auto v) {
        MECHA_LAUNCH(MK_BLOCKS_CAST, (uncast_kernel<decltype(dt)::value, decltype(e8)::value, decltype(v)::value>), dim3((unsigned)blocks), dim3(MECHA_BLOCK), 0, s,
                     static_cast<const uint8_t *>(q->codes), q->pitch, q->scales, q->scale_pitch, q->tile, rows, cols, vec_per_row, out, flags);
    };
    auto with_vec = [&](auto dt, auto e8) { if (vec) go(dt, e8, std::true_type{}); else go(dt, e8, std::false_type{}); };
    auto with_scale = [&](auto dt) { if (q->scale_dtype == MECHA_SCALE_E8M0) with_vec(dt, std::true_type{}); else with_vec(dt, std::false_type{}); };
    switch (out_dtype) {
        case MECHA_F32: with_scale(std::integral_constant<int, MECHA_F32>{}); break;
        case MECHA_F16: with_scale(std::integral_constant<int, MECHA_F16>{}); break;
        default: with_scale(std::integral_constant<int, MECHA_BF16>{}); break;
    }
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

}  // extern "C"
