// adamw.hip -- one AdamW step for every key of an arena in one launch, states in 32 or in 8 bits.
//
//   g = grad * clip;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd[key]) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in float32, whatever the storage types.
//
// HBM-bound: 28 bytes an element with float32 throughout, 10 with 16-bit weights and gradients and 8-bit states: 174 M float32 elements with
// bfloat16 gradients and a bfloat16 copy 810 us (6.0 TB/s, what a flat copy reaches is 6.2), 348 M bfloat16 ones with 8-bit states 605 to 690 us
// (5.1 to 5.8 TB/s, by the weights' and states' values; 59 vector instructions an element take four fifths of it, the conversions' hashes most of them).  One vector a
// thread on a flat grid, 4 elements with float32 states and 8 with 8-bit ones; a vector lies in one key (offsets are multiples of
// 8), its key is found by a search over the segment table that a wave does once, behind the loads.
//
// 8-bit states: e4m3 codes and a power-of-two scale for every 128 elements of the arena; 16 lanes own a block, also one that several
// keys share.  The second moment is kept as its ROOT: e4m3 spans 2^18 between its largest and its
// smallest code, which squared would be only 2^9 of gradient magnitudes.  A code's distance is up to 1/8 of its value and a moving mean
// changes by (1 - b2) of itself a step, so rounding to nearest would never move it: |x| is rounded up with probability equal
// to its part of the distance, by 16 bits of a hash of (offset, step, seed).  A root that is not zero never becomes zero: the
// next step would divide by eps alone.  A gradient over 1.8e19 has a square over float32's largest number: its element takes no part in its
// block's scales and keeps the NaN code for its root, which the next step reads as an infinite one: that weight only decays from then on, as
// with float32 states, and the other 127 of its block move as they would without it.
#include <math.h>
#include <type_traits>
#include "blocks.h"

namespace {

struct AdamParams {
    void *p;
    const void *g;
    void *m, *v;                       // float32, or e4m3 codes
    uint8_t *ms, *vs;                  // scales of 8-bit states
    void *copy;                        // may be NULL
    int copy_dt;
    const mecha_segment *segs;
    int n_segs;
    const float *decay;                // weight decay per key, may be NULL
    float decay_all;
    int64_t total;
    float lr, b1, b2, c1, c2, eps;     // c1 = 1 - b1, c2 = 1 - b2, rounded from double
    float size, root_size;             // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t key;                      // of the hash
    const float *clip;                 // device [norm, coefficient], may be NULL
    const int64_t *step_dev;           // may be NULL; then size, root_size and key are made here
    double b1d, b2d, lrd;
    uint32_t seed;
    uint32_t *seg_flags;
    float over;                        // a weight of this size is stored as infinity, in the arena or in the copy
};

// index of the last segment with offset <= elem, or -1: the 64 lanes look at 64 offsets at once (wave-uniform elem)
__device__ __forceinline__ int find_segment_wave(const mecha_segment *segs, int n, int64_t elem) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;                                      // first segment with offset > elem is in [lo, hi]
    while (hi - lo > 0) {
        const int stride = (hi - lo + 63) >> 6;
        const int at = lo + lane * stride;
        const bool le = at < hi && segs[at].offset <= elem;
        const int c = __popcll(__ballot(le));                // lanes 0 .. c - 1
        if (c == 0) { hi = lo; break; }
        const int nlo = lo + (c - 1) * stride + 1;
        const int nhi = lo + c * stride;
        hi = nhi < hi ? nhi : hi;
        lo = nlo;
    }
    return lo - 1;
}

// (segment or -1, elements of [i, i + N) inside it, elements from i to its end); a vector of N lies in one key.  Every lane of the wave
// calls this.
template <int N>
__device__ __forceinline__ int locate(const mecha_segment *segs, int n, int64_t total, int64_t i, int64_t wave_i, int &valid, int64_t &left) {
    int s = find_segment_wave(segs, n, wave_i);
    while (s + 1 < n && segs[s + 1].offset <= i) s++;
    valid = 0;
    left = INT64_MIN;
    if (s >= 0) {
        left = segs[s].offset + segs[s].numel - i;
        left = left < total - i ? left : total - i;
        valid = left >= N ? N : left > 0 ? (int)left : 0;
    }
    return s;
}

// N consecutive elements of any type as float32: 4 (16 bytes of float32) or 8 (16 bytes of the 16-bit types), read or written once
template <int DT, int N>
__device__ __forceinline__ void load_n(const void *base, int64_t i, float (&v)[N]) {
    if constexpr (N == 8) load8<DT, true>(base, i, v);
    else if constexpr (DT == MECHA_F32) {
        const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(static_cast<const float *>(base) + i));
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(base) + i));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t h = j & 1 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu;
            v[j] = DT == MECHA_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
        }
    }
}
template <int DT, int N>
__device__ __forceinline__ void store_n(void *base, int64_t i, const float (&v)[N]) {
    if constexpr (N == 8) store8<DT, true>(base, i, v);
    else if constexpr (DT == MECHA_F32)
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4 *>(static_cast<float *>(base) + i));
    else {
        u32x2 x;
#pragma unroll
        for (int j = 0; j < 2; j++)
            x[j] = DT == MECHA_BF16 ? f32_to_bf16_bits(v[2 * j]) | f32_to_bf16_bits(v[2 * j + 1]) << 16 : f32_to_f16_bits(v[2 * j]) | f32_to_f16_bits(v[2 * j + 1]) << 16;
        __builtin_nontemporal_store(x, reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(base) + i));
    }
}

// The square root to one unit in the last place, v_sqrt_f32's own error, and the reciprocal below likewise: with the rounded root and division 348 M
// elements with 8-bit states take 685 us, 625 without, and what comes of them is no nearer to float64: 4.75e-7 of the roots' codes are another's
// than float64 would take here, 4.89e-7 there; weights are off by 3.88e-8 either way.  Under 2^-96 (where the instruction would take subnormals
// for zeros) the root of 2^64 v.
__device__ __forceinline__ float root_of(float v) {
    const bool small = v < 1.262177448e-29f;
    const float r = __builtin_amdgcn_sqrtf(small ? v * 18446744073709551616.0f : v);
    return small ? r * 2.3283064365386963e-10f : r;
}

// bit 7 of every byte whose code is NaN
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// 32 bits for an element: multiplications by odd constants (the first 32 fractional bits of the golden ratio and of the square roots
// of 2, 3 and 5) and right shifts, modulo 2^32
__device__ __forceinline__ uint32_t dither32(int64_t i, uint32_t key) {
    uint32_t x = (uint32_t)i * 0x9E3779B9u;
    x ^= x >> 16;
    x = x * 0x6A09E667u + key + (uint32_t)(i >> 32) * 0xBB67AE85u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t dither_key(uint32_t step, uint32_t seed) { return step * 0x3C6EF373u + seed * 0x6A09E667u; }

template <int P_DT, int G_DT, bool BITS8, bool VEC>
__global__ __launch_bounds__(MECHA_BLOCK) void adamw_kernel(AdamParams a) {
    constexpr int N = BITS8 ? 8 : 4;                          // elements a thread: 16 bytes of the arrays that weigh most
    const int64_t i = ((int64_t)blockIdx.x * MECHA_BLOCK + threadIdx.x) * N;
    const int64_t wave_i = i - N * (int)(threadIdx.x & 63);
    if (wave_i >= a.total) return;
    float p[N], g[N], m[N], v[N];
    u32x2 mc = {0, 0}, vc = {0, 0};
    uint32_t ms = 0, vs = 0;
    // what a whole vector of the arenas holds is on its way before the segment is known
    const bool inside = i + N <= a.total;
    if (VEC && inside) {
        load_n<P_DT, N>(a.p, i, p);
        load_n<G_DT, N>(a.g, i, g);
        if constexpr (!BITS8) {
            load_n<MECHA_F32, N>(a.m, i, m);
            load_n<MECHA_F32, N>(a.v, i, v);
        }
    }
    if constexpr (BITS8) {
        if (inside) {                                         // (always: total is a multiple of 128)
            mc = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(a.m) + i));
            vc = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(a.v) + i));
            ms = a.ms[i >> 7];
            vs = a.vs[i >> 7];
        }
    }
    int valid;
    int64_t left;
    const int s = locate<N>(a.segs, a.n_segs, a.total, i, wave_i, valid, left);
    const float keep = 1.0f - a.lr * (a.decay ? (s >= 0 ? a.decay[s] : 0.0f) : a.decay_all);
    const float clip = a.clip ? a.clip[1] : 1.0f;
    float size = a.size, root_size = a.root_size;
    uint32_t key = a.key;
    if (a.step_dev) {
        const int64_t t = *a.step_dev < 1 ? 1 : *a.step_dev;
        double w1 = 1.0, w2 = 1.0, q1 = a.b1d, q2 = a.b2d;
        for (int64_t e = t; e > 0; e >>= 1) {
            if (e & 1) { w1 *= q1; w2 *= q2; }
            q1 *= q1; q2 *= q2;
        }
        size = (float)(a.lrd / (1.0 - w1));
        root_size = (float)(1.0 / sqrt(1.0 - w2));
        key = dither_key((uint32_t)t, a.seed);
    }
    if (!BITS8 && valid == 0) return;
    const bool whole = VEC && valid == N;
    if (!VEC || !inside) {                                    // arenas that are not 16-byte aligned, an arena's last elements
#pragma unroll
        for (int j = 0; j < N; j++) {
            const bool in = j < valid;
            p[j] = in ? load1<P_DT>(a.p, i + j) : 0.0f;
            g[j] = in ? load1<G_DT>(a.g, i + j) : 0.0f;
            if constexpr (!BITS8) {
                m[j] = in ? load1<MECHA_F32>(a.m, i + j) : 0.0f;
                v[j] = in ? load1<MECHA_F32>(a.v, i + j) : 0.0f;
            }
        }
    }
    float poison_in = 0.0f, root[N];                          // fma(x, 0, poison) stays 0 while every x is finite
    bool bad_out = false;
    if (a.seg_flags) {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < valid) poison_in = __builtin_fmaf(g[j], 0.0f, __builtin_fmaf(p[j], 0.0f, poison_in));
    }
    if (!(clip >= 0.0f)) {                                    // the gradients' norm is inf or NaN: the step is left out
        if (a.seg_flags && valid && poison_in != 0.0f) atomicOr(a.seg_flags + s, MECHA_FLAG_INPUT_NONFINITE);
        return;
    }
    auto store = [&](auto dt, void *to, const float (&from)[N]) {
        constexpr int DT = decltype(dt)::value;
        if (whole) store_n<DT, N>(to, i, from);
        else {
#pragma unroll
            for (int j = 0; j < N; j++)
                if (j < valid) store1<DT>(to, i + j, from[j]);
        }
    };
    if constexpr (BITS8) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {                      // two codes an instruction, the scale with them
            const uint32_t mw = mc[j / 4], vw = vc[j / 4];
            const f32x2 x = j & 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(mw, scale_bits(ms), true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(mw, scale_bits(ms), false);
            const f32x2 y = j & 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(vw, scale_bits(vs), true) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(vw, scale_bits(vs), false);
            m[j] = x.x; m[j + 1] = x.y;
            v[j] = y.x * y.x; v[j + 1] = y.y * y.y;
        }
        if (nan_codes(vc.x) | nan_codes(vc.y)) {              // a root over the largest number (rare)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if ((nan_codes(vc[j / 4]) >> (8 * (j & 3))) & 0x80u) v[j] = INFINITY;
        }
        if (valid < 8) {                                      // what lies between the keys takes no part in a scale, and its codes become 0
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j >= valid) m[j] = v[j] = g[j] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float gj = g[j] * clip;
        m[j] = __builtin_fmaf(gj, a.c1, m[j] * a.b1);
        v[j] = __builtin_fmaf(gj * gj, a.c2, v[j] * a.b2);
        root[j] = root_of(v[j]);
        const float den = __builtin_fmaf(root[j], root_size, a.eps);
        p[j] = __builtin_fmaf(m[j] * __builtin_amdgcn_rcpf(den), -size, p[j] * keep);
    }
    if (a.seg_flags) {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < valid) bad_out |= !(fabsf(p[j]) < a.over) || !(root[j] < INFINITY);
    }
    if (valid) {
        store(std::integral_constant<int, P_DT>{}, a.p, p);
        if (a.copy) {
            if (a.copy_dt == MECHA_BF16) store(std::integral_constant<int, MECHA_BF16>{}, a.copy, p);
            else if (a.copy_dt == MECHA_F16) store(std::integral_constant<int, MECHA_F16>{}, a.copy, p);
            else store(std::integral_constant<int, MECHA_F32>{}, a.copy, p);
        }
    }
    if constexpr (BITS8) {
        float mm = 0.0f, vm = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) { mm = fmaxf(mm, fabsf(m[j])); vm = fmaxf(vm, root[j]); }
        if (!(fmaxf(mm, vm) < INFINITY)) {                    // (NaN takes no part in the maxima)
            mm = vm = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (!(root[j] < INFINITY)) { m[j] = fabsf(m[j]) < INFINITY ? 0.0f : NAN; root[j] = NAN; }
                mm = fmaxf(mm, fabsf(m[j]));
                vm = fmaxf(vm, root[j]);
            }
        }
        const int em = block_exponent(max16(mm)), ev = block_exponent(max16(vm));
        const float sm = scale_bits(em + 127), sv = scale_bits(ev + 127);
        int mw[2] = {0, 0}, vw[2] = {0, 0};
#pragma unroll
        for (int w = 0; w < 2; w++) {
            // gfx950's stochastic conversion of x / 2^e: floor(|x| / distance + random / 2^32) for every code, subnormal ones too (checked on
            // 2^22 numbers against the definition)
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; j++) u[j] = dither32(i + 4 * w + j, key);
            mw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(mw[w], m[4 * w], u[0] << 16, sm, 0);
            mw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(mw[w], m[4 * w + 1], u[1] << 16, sm, 1);
            mw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(mw[w], m[4 * w + 2], u[2] << 16, sm, 2);
            mw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(mw[w], m[4 * w + 3], u[3] << 16, sm, 3);
            // no root that is not zero goes under the smallest code: under it, it is raised to it, and not a random part further
            const float least = sv * 0.001953125f;
            float rr[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = root[4 * w + j];
                const bool tiny = x > 0.0f && x < least;
                rr[j] = tiny ? least : x;
                u[j] = tiny ? 0u : u[j] & 0xffff0000u;
            }
            vw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(vw[w], rr[0], u[0], sv, 0);
            vw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(vw[w], rr[1], u[1], sv, 1);
            vw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(vw[w], rr[2], u[2], sv, 2);
            vw[w] = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(vw[w], rr[3], u[3], sv, 3);
        }
        if (left > -(i & 127)) {                              // the key reaches into this block: its codes are all written
            __builtin_nontemporal_store(u32x2{(uint32_t)mw[0], (uint32_t)mw[1]}, reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.m) + i));
            __builtin_nontemporal_store(u32x2{(uint32_t)vw[0], (uint32_t)vw[1]}, reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.v) + i));
        }
        // (the block's first lane may lie in front of its first key)
        const bool any = (__ballot(valid) >> (threadIdx.x & 48)) & 0xffffull;
        if ((threadIdx.x & 15) == 0 && any) { a.ms[i >> 7] = (uint8_t)(em + 127); a.vs[i >> 7] = (uint8_t)(ev + 127); }
    } else {
        store(std::integral_constant<int, MECHA_F32>{}, a.m, m);
        store(std::integral_constant<int, MECHA_F32>{}, a.v, v);
    }
    if (a.seg_flags && valid && (poison_in != 0.0f || bad_out))
        atomicOr(a.seg_flags + s, (poison_in != 0.0f ? MECHA_FLAG_INPUT_NONFINITE : 0u) | (bad_out ? MECHA_FLAG_OUTPUT_NONFINITE : 0u));
}

// ------------------------------------------------------------------------------------------------------- gradient norm
// Sum of squares over the keys' elements: fixed runs of the arena per block, float64 partials in a fixed order (no atomics, the same
// sum every time), folded by one block into [norm, min(1, max_norm / (norm + 1e-6))]; NaN where an element is inf or NaN.  One read of the
// gradients: 174 M bfloat16 ones 65 us (5.4 TB/s) and 4.5 for the fold.
constexpr int NORM_GRID = 2048;

template <int G_DT, bool VEC>
__global__ __launch_bounds__(MECHA_BLOCK) void norm_partial_kernel(const void *g, const mecha_segment *segs, int n_segs, int64_t total, int64_t per_wave,
                                                                   double *partial) {
    __shared__ double fold[MECHA_BLOCK];
    constexpr int AHEAD = 4;                                  // vectors in flight a lane
    const int lane = threadIdx.x & 63;
    const int64_t begin = ((int64_t)blockIdx.x * (MECHA_BLOCK / 64) + (threadIdx.x >> 6)) * per_wave;
    const int64_t end = begin + per_wave < total ? begin + per_wave : total;
    double sum = 0.0;
    int64_t key_begin = 0, key_end = 0;                       // a key's elements, the same for the whole wave
    for (int64_t at = begin; at < end; at += 512 * AHEAD) {
        float v[AHEAD][8];
        const bool fast = VEC && at + 512 * AHEAD <= end;
        if (fast) {
#pragma unroll
            for (int x = 0; x < AHEAD; x++) load8<G_DT, true>(g, at + 512 * x + 8 * lane, v[x]);
        }
#pragma unroll
        for (int x = 0; x < AHEAD; x++) {
            const int64_t wave_i = at + 512 * x, i = wave_i + 8 * lane;
            if (wave_i >= end) break;
            int valid = 8;
            if (wave_i < key_begin || wave_i + 512 > key_end) {
                int s = find_segment_wave(segs, n_segs, wave_i);
                key_begin = s >= 0 ? segs[s].offset : 0;
                key_end = s >= 0 ? segs[s].offset + segs[s].numel : 0;
                key_end = key_end < total ? key_end : total;
                int64_t left;
                if (wave_i + 512 > key_end) locate<8>(segs, n_segs, total, i, wave_i, valid, left);
                if (i >= end) valid = 0;
            }
            if (!fast) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[x][j] = j < valid && i < end ? load1<G_DT>(g, i + j) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const double d = j < valid ? (double)v[x][j] : 0.0;
                sum = __builtin_fma(d, d, sum);
            }
        }
    }
    fold[threadIdx.x] = sum;
    __syncthreads();
    for (int d = MECHA_BLOCK / 2; d > 0; d >>= 1) {
        if (threadIdx.x < d) fold[threadIdx.x] += fold[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) partial[blockIdx.x] = fold[0];
}

__global__ __launch_bounds__(MECHA_BLOCK) void norm_finish_kernel(const double *partial, int n, double max_norm, float *out) {
    __shared__ double fold[MECHA_BLOCK];
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += MECHA_BLOCK) sum += partial[i];
    fold[threadIdx.x] = sum;
    __syncthreads();
    for (int d = MECHA_BLOCK / 2; d > 0; d >>= 1) {
        if (threadIdx.x < d) fold[threadIdx.x] += fold[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(fold[0]);
        const float coef = (float)max_norm / (norm + 1e-6f);
        out[0] = norm;
        out[1] = nonfinite_f32(norm) ? __uint_as_float(0x7fc00000u) : coef < 1.0f ? coef : 1.0f;
    }
}

int check_arena(const mecha_segment *segs, int n_segs, int64_t total) {
    MECHA_REQUIRE(n_segs > 0 && segs != nullptr, "batched call needs a device segment table");
    MECHA_REQUIRE(total >= 0, "total_elems must be >= 0 (got %lld)", (long long)total);
    MECHA_REQUIRE((total + 3) / 4 < (1ll << 32) - MECHA_BLOCK, "total_elems %lld is beyond one launch (2^34)", (long long)total);
    return MECHA_OK;
}

template <typename F>
void with_dtype(int dt, F &&f) {
    switch (dt) {
        case MECHA_F32: f(std::integral_constant<int, MECHA_F32>{}); break;
        case MECHA_F16: f(std::integral_constant<int, MECHA_F16>{}); break;
        default: f(std::integral_constant<int, MECHA_BF16>{}); break;
    }
}

}  // namespace

extern "C" {

size_t mecha_batched_grad_norm_workspace_bytes(int64_t total_elems) {
    (void)total_elems;
    return NORM_GRID * sizeof(double);
}

int mecha_batched_grad_norm(const void *grad_arena, const mecha_segment *segments, int n_segments, int64_t total_elems, int grad_dtype,
                            double max_norm, float *norm_out, void *workspace, size_t workspace_bytes, void *stream) {
    const int st = check_arena(segments, n_segments, total_elems);
    if (st) return st;
    MECHA_REQUIRE(mecha_valid_dtype(grad_dtype), "unknown dtype code %d", grad_dtype);
    MECHA_REQUIRE(norm_out != nullptr && (grad_arena != nullptr || total_elems == 0), "grad_arena or norm_out is NULL");
    MECHA_REQUIRE(max_norm >= 0.0, "max_norm must be >= 0 (got %g)", max_norm);
    if (workspace == nullptr || workspace_bytes < mecha_batched_grad_norm_workspace_bytes(total_elems)) {
        mecha_set_error("grad_norm workspace: %zu bytes given, %zu needed", workspace_bytes, mecha_batched_grad_norm_workspace_bytes(total_elems));
        return MECHA_ERR_WORKSPACE;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t waves = NORM_GRID * (MECHA_BLOCK / 64), units = (total_elems + 2047) / 2048;
    const int64_t per_wave = (units + waves - 1) / waves * 2048;                  // whole rounds of a wave
    const int grid = per_wave ? (int)((total_elems + 4 * per_wave - 1) / (4 * per_wave)) : 0;
    double *partial = static_cast<double *>(workspace);
    const bool vec = mecha_aligned16(grad_arena);
    if (grid > 0)
        with_dtype(grad_dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            if (vec) MECHA_LAUNCH(MK_ADAMW, (norm_partial_kernel<DT, true>), dim3(grid), dim3(MECHA_BLOCK), 0, s, grad_arena, segments, n_segments, total_elems, per_wave, partial);
            else MECHA_LAUNCH(MK_ADAMW, (norm_partial_kernel<DT, false>), dim3(grid), dim3(MECHA_BLOCK), 0, s, grad_arena, segments, n_segments, total_elems, per_wave, partial);
        });
    MECHA_LAUNCH(MK_ADAMW, norm_finish_kernel, dim3(1), dim3(MECHA_BLOCK), 0, s, partial, grid, max_norm, norm_out);
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

int mecha_batched_adamw(const mecha_adamw *args, void *stream) {
    MECHA_REQUIRE(args != nullptr, "no arguments");
    const mecha_adamw &x = *args;
    const int st = check_arena(x.segments, x.n_segments, x.total_elems);
    if (st) return st;
    MECHA_REQUIRE(mecha_valid_dtype(x.param_dtype) && mecha_valid_dtype(x.grad_dtype) && (x.copy == nullptr || mecha_valid_dtype(x.copy_dtype)),
                  "unknown dtype code (param %d, grad %d, copy %d)", x.param_dtype, x.grad_dtype, x.copy_dtype);
    MECHA_REQUIRE(x.state_bits == 32 || x.state_bits == 8, "states are held in 32 or 8 bits (got %d)", x.state_bits);
    MECHA_REQUIRE(x.beta1 >= 0.0 && x.beta1 < 1.0 && x.beta2 >= 0.0 && x.beta2 < 1.0, "betas must be in [0, 1) (got %g, %g)", x.beta1, x.beta2);
    MECHA_REQUIRE(x.eps >= 0.0 && x.lr >= 0.0, "lr and eps must be >= 0 (got %g, %g)", x.lr, x.eps);
    MECHA_REQUIRE(x.step_dev != nullptr || x.step >= 1, "steps count from 1 (got %lld)", (long long)x.step);
    if (x.total_elems == 0) return MECHA_OK;
    MECHA_REQUIRE(x.params && x.grads && x.exp_avg && x.exp_avg_sq, "an arena is NULL");
    if (x.state_bits == 8) {
        MECHA_REQUIRE(x.exp_avg_scales && x.exp_avg_sq_scales, "8-bit states need their scales");
        MECHA_REQUIRE(x.total_elems % SCALE_BLOCK == 0, "8-bit states: total_elems %lld must be a multiple of 128", (long long)x.total_elems);
        MECHA_REQUIRE((reinterpret_cast<uintptr_t>(x.exp_avg) & 7u) == 0 && (reinterpret_cast<uintptr_t>(x.exp_avg_sq) & 7u) == 0, "8-bit states must be 8-byte aligned");
    }
    const size_t n = (size_t)x.total_elems, state_bytes = x.state_bits == 8 ? n : 4 * n, scale_bytes = x.state_bits == 8 ? n / SCALE_BLOCK : 0;
    const struct { const void *at; size_t bytes; } arenas[] = {
        {x.params, n * mecha_dtype_size(x.param_dtype)}, {x.grads, n * mecha_dtype_size(x.grad_dtype)}, {x.exp_avg, state_bytes}, {x.exp_avg_sq, state_bytes},
        {x.copy, x.copy ? n * mecha_dtype_size(x.copy_dtype) : 0}, {x.exp_avg_scales, scale_bytes}, {x.exp_avg_sq_scales, scale_bytes}};
    for (int i = 0; i < 7; i++)
        for (int j = 0; j < i; j++)
            MECHA_REQUIRE(arenas[i].bytes == 0 || !mecha_overlap(arenas[i].at, arenas[i].bytes, arenas[j].at, arenas[j].bytes), "two arenas share memory");
    AdamParams a{};
    a.p = x.params; a.g = x.grads; a.m = x.exp_avg; a.v = x.exp_avg_sq;
    a.ms = static_cast<uint8_t *>(x.exp_avg_scales); a.vs = static_cast<uint8_t *>(x.exp_avg_sq_scales);
    a.copy = x.copy; a.copy_dt = x.copy_dtype;
    a.segs = x.segments; a.n_segs = x.n_segments; a.total = x.total_elems;
    a.decay = x.key_weight_decay; a.decay_all = (float)x.weight_decay;
    a.lr = (float)x.lr; a.b1 = (float)x.beta1; a.b2 = (float)x.beta2; a.c1 = (float)(1.0 - x.beta1); a.c2 = (float)(1.0 - x.beta2); a.eps = (float)x.eps;
    a.lrd = x.lr; a.b1d = x.beta1; a.b2d = x.beta2; a.seed = x.seed; a.step_dev = x.step_dev; a.clip = x.clip; a.seg_flags = x.seg_flags;
    a.over = fminf(stored_as_inf(x.param_dtype), x.copy ? stored_as_inf(x.copy_dtype) : INFINITY);
    if (x.step_dev == nullptr) {
        a.size = (float)(x.lr / (1.0 - pow(x.beta1, (double)x.step)));
        a.root_size = (float)(1.0 / sqrt(1.0 - pow(x.beta2, (double)x.step)));
        a.key = dither_key((uint32_t)x.step, x.seed);
    }
    const bool vec = mecha_aligned16(x.params) && mecha_aligned16(x.grads) && (x.state_bits == 8 || (mecha_aligned16(x.exp_avg) && mecha_aligned16(x.exp_avg_sq)))
                     && (x.copy == nullptr || mecha_aligned16(x.copy));
    const int64_t each = (x.state_bits == 8 ? 8 : 4) * MECHA_BLOCK, blocks = (x.total_elems + each - 1) / each;
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(x.param_dtype, [&](auto pd) {
        with_dtype(x.grad_dtype, [&](auto gd) {
            auto go = [&](auto b8, auto v) {
                MECHA_LAUNCH(MK_ADAMW, (adamw_kernel<decltype(pd)::value, decltype(gd)::value, decltype(b8)::value, decltype(v)::value>),
                             dim3((unsigned)blocks), dim3(MECHA_BLOCK), 0, s, a);
            };
            if (x.state_bits == 8) { if (vec) go(std::true_type{}, std::true_type{}); else go(std::true_type{}, std::false_type{}); }
            else { if (vec) go(std::false_type{}, std::true_type{}); else go(std::false_type{}, std::false_type{}); }
        });
    });
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

}  // extern "C"
