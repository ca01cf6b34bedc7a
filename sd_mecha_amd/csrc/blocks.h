// blocks.h -- e4m3 codes and the power-of-two scale of a block of 128, shared by blocks.hip and adamw.hip.
#pragma once
#include "common.h"

constexpr int SCALE_BLOCK = MECHA_SCALE_BLOCK;      // 128
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Rows need not be whole 16 bytes long: gfx950 loads and stores vectors at any element's address.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(2)));
// the first `bytes` of 16 (a multiple of 2, from 2 to 14), for a row's last elements
__device__ __forceinline__ void store_part(void *to, u32x4 v, int bytes) {
    char *at = static_cast<char *>(to);
    u32x2 w = {v.x, v.y};
    if (bytes & 8) { *reinterpret_cast<u32x2_any *>(at) = w; at += 8; w = u32x2{v.z, v.w}; }
    uint32_t x = w.x;
    if (bytes & 4) { *reinterpret_cast<u32_any *>(at) = x; at += 4; x = w.y; }
    if (bytes & 2) *reinterpret_cast<uint16_t *>(at) = (uint16_t)x;
}
__device__ __forceinline__ u32x4 load_part(const void *from, int bytes) {     // zeros behind them
    const char *at = static_cast<const char *>(from);
    u32x2 a = {0, 0}, w = {0, 0};
    if (bytes & 8) { a = *reinterpret_cast<const u32x2_any *>(at); at += 8; }
    if (bytes & 4) { w.x = *reinterpret_cast<const u32_any *>(at); at += 4; }
    if (bytes & 2) { const uint32_t x = *reinterpret_cast<const uint16_t *>(at); if (bytes & 4) w.y = x; else w.x = x; }
    return bytes & 8 ? u32x4{a.x, a.y, w.x, w.y} : u32x4{w.x, w.y, 0u, 0u};
}

// The smallest e >= -127 with amax <= 448 * 2^e, from the bits of amax (finite, >= 0): 448 = 1.75 * 2^8, so e is amax's exponent
// less 8, one more where its mantissa is over 1.75.  Zero and subnormal amax end at the clamp.
__device__ __forceinline__ int block_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -127 ? -127 : e;
}
// 2^(byte - 127) as gfx950's scaled conversions take it: only the exponent's byte counts, 0 being 2^-127 and 255 NaN
__device__ __forceinline__ float scale_bits(uint32_t byte) { return __uint_as_float(byte << 23); }
// 2^(byte - 127); byte 0 is 2^-127, a subnormal; byte 255 is NaN
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
    return byte == 0u ? __uint_as_float(0x00400000u) : byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

__device__ __forceinline__ void unpack_e4m3x4(uint32_t w, float *v) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}

// max over the 16 lanes that share a block of 128 (8 elements each), by rotations within a row of lanes; every lane gets it.  NaN is left out.
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x128, 0xf, 0xf, true)));
    v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x124, 0xf, 0xf, true)));
    v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x122, 0xf, 0xf, true)));
    return fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x121, 0xf, 0xf, true)));
}

// The smallest magnitude that a type stores as infinity: half a step over its largest number (the tie goes to the even side, infinity).  Output
// flags are about what is stored: !(|x| < this), which NaN sets as well.
__host__ __device__ constexpr float stored_as_inf(int dt) { return dt == MECHA_F16 ? 65520.0f : dt == MECHA_BF16 ? 0x1.ffp127f : __builtin_inff(); }

// A barrier for what the waves exchange through LDS: unlike __syncthreads() it does not wait for stores to memory.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

static inline bool mecha_overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a != nullptr && b != nullptr && x < y + b_bytes && y < x + a_bytes;
}
// from a matrix's first code or scale to behind its last
static inline size_t mecha_codes_bytes(const mecha_block_matrix &q) {
    return q.rows && q.cols ? (size_t)(q.rows - 1) * q.pitch + (q.cols + SCALE_BLOCK - 1) / SCALE_BLOCK * SCALE_BLOCK : 0;
}
static inline size_t mecha_scales_bytes(const mecha_block_matrix &q) {
    const int64_t rows = q.tile ? (q.rows + SCALE_BLOCK - 1) / SCALE_BLOCK : q.rows;
    return rows && q.cols ? ((size_t)(rows - 1) * q.scale_pitch + (q.cols + SCALE_BLOCK - 1) / SCALE_BLOCK) * (q.scale_dtype == MECHA_SCALE_F32 ? 4 : 1) : 0;
}

// whether two matrices' codes share memory; rows of one pitch may lie side by side
static inline bool mecha_codes_overlap(const mecha_block_matrix &a, const mecha_block_matrix &b) {
    if (!mecha_overlap(a.codes, mecha_codes_bytes(a), b.codes, mecha_codes_bytes(b))) return false;
    if (a.pitch != b.pitch) return true;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.codes), y = reinterpret_cast<uintptr_t>(b.codes);
    const mecha_block_matrix &low = x < y ? a : b, &high = x < y ? b : a;
    auto width = [](const mecha_block_matrix &q) { return (q.cols + SCALE_BLOCK - 1) / SCALE_BLOCK * SCALE_BLOCK; };
    const int64_t apart = (int64_t)((x < y ? y - x : x - y) % (uintptr_t)a.pitch);
    return apart < width(low) || apart + width(high) > a.pitch;
}

// the layout of include/mecha_hip.h for one matrix; an error message and code where it is not kept
static inline int mecha_check_blocks(const char *what, const mecha_block_matrix &q) {
    const int64_t blocks = (q.cols + SCALE_BLOCK - 1) / SCALE_BLOCK;
    MECHA_REQUIRE(q.rows >= 0 && q.cols >= 0, "%s: bad matrix %lld x %lld", what, (long long)q.rows, (long long)q.cols);
    MECHA_REQUIRE(q.scale_dtype == MECHA_SCALE_F32 || q.scale_dtype == MECHA_SCALE_E8M0, "%s: unknown scale dtype %d", what, q.scale_dtype);
    if (q.rows == 0 || q.cols == 0) return MECHA_OK;
    MECHA_REQUIRE(q.codes != nullptr && q.scales != nullptr, "%s: codes or scales are NULL", what);
    MECHA_REQUIRE(mecha_aligned16(q.codes), "%s: codes must be 16-byte aligned", what);
    MECHA_REQUIRE(q.pitch % SCALE_BLOCK == 0 && q.pitch >= blocks * SCALE_BLOCK, "%s: the row pitch %lld must be a multiple of 128 and hold %lld columns rounded up to 128",
                  what, (long long)q.pitch, (long long)q.cols);
    MECHA_REQUIRE(q.scale_pitch >= blocks, "%s: a row of scales holds %lld, %lld are needed", what, (long long)q.scale_pitch, (long long)blocks);
    return MECHA_OK;
}
