// adamw.hip -- one AdamW step for every key of an arena in one launch, states in 32 or in 8 bits.
//
//   g = grad * clip;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd[key]) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in float32, every product, sum, quotient and root rounded by itself, whatever the storage types.
//
// HBM-bound: 28 bytes an element with float32 throughout, 10 with 16-bit weights and gradients and 8-bit states.  One vector of
// 8 elements a thread on a flat grid; a vector lies in one key (offsets are multiples of 8), its key is found by a search
// over the segment table that a wave does once.
//
// 8-bit states: e4m3 codes and a power-of-two scale for every 128 elements of the arena (segment offsets are multiples of 128, so
// a block belongs to one key; 16 lanes own it).  The second moment is kept as its ROOT: e4m3 spans 2^18 between its largest and its
// smallest code, which squared would be only 2^9 of gradient magnitudes.  A code's distance is up to 1/8 of its value and a moving mean
// changes by (1 - b2) of itself a step, so rounding to nearest would never move it: |x| is rounded up with probability equal
// to its part of the distance, by 16 bits of a hash of (offset, step, seed).  A root that is not zero never becomes zero: the
// next step would divide by eps alone.
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

// (segment or -1, elements of [i, i + 8) inside it).  i is a multiple of 8; every lane of the wave calls this.
__device__ __forceinline__ int locate8(const mecha_segment *segs, int n, int64_t total, int64_t i, int64_t wave_i, int &valid) {
    int s = find_segment_wave(segs, n, wave_i);
    while (s + 1 < n && segs[s + 1].offset <= i) s++;
    valid = 0;
    if (s >= 0) {
        int64_t left = segs[s].offset + segs[s].numel - i;
        left = left < total - i ? left : total - i;
        valid = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    }
    return s;
}

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
__device__ __forceinline__ uint32_t dither_key(uint32_t step, uint32_t seed) { return step * 0x3C6EF373u + seed * 0x6A09E667u; }

// |y| <= 448 down to a code or up to the next one: floor(|y| / distance + u / 2^16).  A float's top 12 bits below the sign are its
// e4m3 code but for the exponent's bias, and the 20 below them its part of the distance: adding u << 4 carries with the right
// probability.  Under 2^-6 the codes are 2^-9 apart like those of the next binade, so |y| + 2^-6 is rounded there instead.
__device__ __forceinline__ uint32_t dithered_code(float y, uint32_t u) {
    const float size = fabsf(y);
    const bool small = size < 0.015625f;
    const uint32_t bits = __float_as_uint(small ? size + 0.015625f : size);
    uint32_t code = ((bits + (u << 4)) >> 20) - (small ? 968u : 960u);
    code = nonfinite_f32(y) ? 0x7fu : code;
    return code | ((__float_as_uint(y) >> 24) & 0x80u);
}

template <int P_DT, int G_DT, bool BITS8, bool VEC>
__global__ __launch_bounds__(MECHA_BLOCK) void adamw_kernel(AdamParams a) {
    const int64_t i = ((int64_t)blockIdx.x * MECHA_BLOCK + threadIdx.x) * 8;
    const int64_t wave_i = i - 8 * (threadIdx.x & 63);
    if (wave_i >= a.total) return;
    float clip = 1.0f;
    if (a.clip) {
        clip = a.clip[1];
        if (!(clip >= 0.0f)) return;                          // a gradient is inf or NaN: the step is left out
    }
    int valid;
    const int s = locate8(a.segs, a.n_segs, a.total, i, wave_i, valid);
    if constexpr (!BITS8) { if (valid == 0) return; }
    const bool whole = VEC && valid == 8;
    float p[8], g[8], m[8], v[8];
    auto load = [&](auto dt, const void *from, float (&to)[8]) {
        constexpr int DT = decltype(dt)::value;
        if (whole) load8<DT, true>(from, i, to);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++) to[j] = j < valid ? load1<DT>(from, i + j) : 0.0f;
        }
    };
    auto store = [&](auto dt, void *to, const float (&from)[8]) {
        constexpr int DT = decltype(dt)::value;
        if (whole) store8<DT, true>(to, i, from);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < valid) store1<DT>(to, i + j, from[j]);
        }
    };
    load(std::integral_constant<int, P_DT>{}, a.p, p);
    load(std::integral_constant<int, G_DT>{}, a.g, g);
    if constexpr (BITS8) {
        if (valid) {                                          // a block's codes are all there, also behind its key's last element
            const u32x2 mc = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(a.m) + i);
            const u32x2 vc = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(a.v) + i);
            const float sm = e8m0_to_f32(a.ms[i >> 7]), sv = e8m0_to_f32(a.vs[i >> 7]);
            unpack_e4m3x4(mc.x, m); unpack_e4m3x4(mc.y, m + 4);
            unpack_e4m3x4(vc.x, v); unpack_e4m3x4(vc.y, v + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                m[j] = j < valid ? m[j] * sm : 0.0f;
                const float root = j < valid ? v[j] * sv : 0.0f;
                v[j] = root * root;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) m[j] = v[j] = 0.0f;
        }
    } else {
        load(std::integral_constant<int, MECHA_F32>{}, a.m, m);
        load(std::integral_constant<int, MECHA_F32>{}, a.v, v);
    }
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
    const float keep = 1.0f - a.lr * (a.decay ? (s >= 0 ? a.decay[s] : 0.0f) : a.decay_all);
    bool bad_in = false, bad_out = false;
    float root[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        bad_in |= nonfinite_f32(g[j]) || nonfinite_f32(p[j]);
        const float gj = g[j] * clip;
        m[j] = m[j] * a.b1 + gj * a.c1;
        v[j] = v[j] * a.b2 + gj * gj * a.c2;
        root[j] = __builtin_sqrtf(v[j]);
        p[j] = p[j] * keep - m[j] / (root[j] * root_size + a.eps) * size;
        bad_out |= nonfinite_f32(p[j]);
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
        for (int j = 0; j < 8; j++) {
            mm = fmaxf(mm, nonfinite_f32(m[j]) ? 0.0f : fabsf(m[j]));
            vm = fmaxf(vm, nonfinite_f32(root[j]) ? 0.0f : root[j]);
        }
        const int em = block_exponent(max16(mm)), ev = block_exponent(max16(vm));
        const float im = pow2f(-em), iv = pow2f(-ev);
        uint32_t mc[8], vc[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t u = dither32(i + j, key);
            mc[j] = dithered_code(m[j] * im, u & 0xffffu);
            const float y = root[j] * iv;
            const uint32_t c = dithered_code(y, u >> 16);
            vc[j] = y > 0.0f && c == 0u ? 1u : c;
        }
        if (valid) {
            auto pack = [](const uint32_t (&c)[8]) {
                return u32x2{c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
            };
            *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.m) + i) = pack(mc);
            *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(a.v) + i) = pack(vc);
            if ((threadIdx.x & 15) == 0) { a.ms[i >> 7] = (uint8_t)(em + 127); a.vs[i >> 7] = (uint8_t)(ev + 127); }
        }
    } else {
        store(std::integral_constant<int, MECHA_F32>{}, a.m, m);
        store(std::integral_constant<int, MECHA_F32>{}, a.v, v);
    }
    if ((bad_in || bad_out) && valid && a.seg_flags)
        atomicOr(a.seg_flags + s, (bad_in ? MECHA_FLAG_INPUT_NONFINITE : 0u) | (bad_out ? MECHA_FLAG_OUTPUT_NONFINITE : 0u));
}

// ------------------------------------------------------------------------------------------------------- gradient norm
// Sum of squares over the keys' elements: fixed runs of the arena per block, float64 partials in a fixed order (no atomics, the same
// sum every time), folded by one block into [norm, min(1, max_norm / (norm + 1e-6))]; NaN where an element is inf or NaN.
constexpr int NORM_GRID = 2048;

template <int G_DT, bool VEC>
__global__ __launch_bounds__(MECHA_BLOCK) void norm_partial_kernel(const void *g, const mecha_segment *segs, int n_segs, int64_t total, int64_t per_block,
                                                                   double *partial) {
    __shared__ double fold[MECHA_BLOCK];
    const int64_t begin = blockIdx.x * per_block, end = begin + per_block < total ? begin + per_block : total;
    double sum = 0.0;
    for (int64_t at = begin; at < end; at += 8 * MECHA_BLOCK) {
        const int64_t i = at + 8 * threadIdx.x, wave_i = i - 8 * (threadIdx.x & 63);
        if (wave_i >= end) break;
        int valid;
        locate8(segs, n_segs, total, i, wave_i, valid);
        if (i >= end) valid = 0;
        float v[8];
        if (VEC && valid == 8) load8<G_DT, true>(g, i, v);
        else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = j < valid ? load1<G_DT>(g, i + j) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) sum += (double)v[j] * (double)v[j];
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
    MECHA_REQUIRE((total + 7) / 8 < (1ll << 32) - MECHA_BLOCK, "total_elems %lld is beyond one launch (2^35)", (long long)total);
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
    const int64_t unit = 8 * MECHA_BLOCK, units = (total_elems + unit - 1) / unit;
    const int64_t per_block = (units + NORM_GRID - 1) / NORM_GRID * unit;
    const int grid = per_block ? (int)((total_elems + per_block - 1) / per_block) : 0;
    double *partial = static_cast<double *>(workspace);
    const bool vec = mecha_aligned16(grad_arena);
    if (grid > 0)
        with_dtype(grad_dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            if (vec) MECHA_LAUNCH(MK_ADAMW, (norm_partial_kernel<DT, true>), dim3(grid), dim3(MECHA_BLOCK), 0, s, grad_arena, segments, n_segments, total_elems, per_block, partial);
            else MECHA_LAUNCH(MK_ADAMW, (norm_partial_kernel<DT, false>), dim3(grid), dim3(MECHA_BLOCK), 0, s, grad_arena, segments, n_segments, total_elems, per_block, partial);
        });
    MECHA_LAUNCH(MK_ADAMW, norm_finish_kernel, dim3(1), dim3(MECHA_BLOCK), 0, s, partial, grid, max_norm, norm_out);
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

int mecha_batched_adamw(void *param_arena, const void *grad_arena, void *exp_avg, void *exp_avg_sq, void *exp_avg_scales,
                        void *exp_avg_sq_scales, void *copy_arena, const mecha_segment *segments, int n_segments, int64_t total_elems,
                        int param_dtype, int grad_dtype, int copy_dtype, int state_bits, double lr, double beta1, double beta2, double eps,
                        double weight_decay, const float *key_weight_decay, int64_t step, const int64_t *step_dev, uint32_t seed,
                        const float *clip, uint32_t *seg_flags, void *stream) {
    const int st = check_arena(segments, n_segments, total_elems);
    if (st) return st;
    MECHA_REQUIRE(mecha_valid_dtype(param_dtype) && mecha_valid_dtype(grad_dtype) && (copy_arena == nullptr || mecha_valid_dtype(copy_dtype)),
                  "unknown dtype code (param %d, grad %d, copy %d)", param_dtype, grad_dtype, copy_dtype);
    MECHA_REQUIRE(state_bits == 32 || state_bits == 8, "states are held in 32 or 8 bits (got %d)", state_bits);
    MECHA_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "betas must be in [0, 1) (got %g, %g)", beta1, beta2);
    MECHA_REQUIRE(eps >= 0.0 && lr >= 0.0, "lr and eps must be >= 0 (got %g, %g)", lr, eps);
    MECHA_REQUIRE(step_dev != nullptr || step >= 1, "steps count from 1 (got %lld)", (long long)step);
    if (total_elems == 0) return MECHA_OK;
    MECHA_REQUIRE(param_arena && grad_arena && exp_avg && exp_avg_sq, "an arena is NULL");
    if (state_bits == 8) {
        MECHA_REQUIRE(exp_avg_scales && exp_avg_sq_scales, "8-bit states need their scales");
        MECHA_REQUIRE(total_elems % SCALE_BLOCK == 0, "8-bit states: total_elems %lld must be a multiple of 128", (long long)total_elems);
        MECHA_REQUIRE((reinterpret_cast<uintptr_t>(exp_avg) & 7u) == 0 && (reinterpret_cast<uintptr_t>(exp_avg_sq) & 7u) == 0, "8-bit states must be 8-byte aligned");
    }
    AdamParams a{};
    a.p = param_arena; a.g = grad_arena; a.m = exp_avg; a.v = exp_avg_sq;
    a.ms = static_cast<uint8_t *>(exp_avg_scales); a.vs = static_cast<uint8_t *>(exp_avg_sq_scales);
    a.copy = copy_arena; a.copy_dt = copy_dtype;
    a.segs = segments; a.n_segs = n_segments; a.total = total_elems;
    a.decay = key_weight_decay; a.decay_all = (float)weight_decay;
    a.lr = (float)lr; a.b1 = (float)beta1; a.b2 = (float)beta2; a.c1 = (float)(1.0 - beta1); a.c2 = (float)(1.0 - beta2); a.eps = (float)eps;
    a.lrd = lr; a.b1d = beta1; a.b2d = beta2; a.seed = seed; a.step_dev = step_dev; a.clip = clip; a.seg_flags = seg_flags;
    if (step_dev == nullptr) {
        a.size = (float)(lr / (1.0 - pow(beta1, (double)step)));
        a.root_size = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
        a.key = (uint32_t)step * 0x3C6EF373u + seed * 0x6A09E667u;
    }
    const bool vec = mecha_aligned16(param_arena) && mecha_aligned16(grad_arena) && (state_bits == 8 || (mecha_aligned16(exp_avg) && mecha_aligned16(exp_avg_sq)))
                     && (copy_arena == nullptr || mecha_aligned16(copy_arena));
    const int64_t blocks = ((total_elems + 7) / 8 + MECHA_BLOCK - 1) / MECHA_BLOCK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(param_dtype, [&](auto pd) {
        with_dtype(grad_dtype, [&](auto gd) {
            auto go = [&](auto b8, auto v) {
                MECHA_LAUNCH(MK_ADAMW, (adamw_kernel<decltype(pd)::value, decltype(gd)::value, decltype(b8)::value, decltype(v)::value>),
                             dim3((unsigned)blocks), dim3(MECHA_BLOCK), 0, s, a);
            };
            if (state_bits == 8) { if (vec) go(std::true_type{}, std::true_type{}); else go(std::true_type{}, std::false_type{}); }
            else { if (vec) go(std::false_type{}, std::true_type{}); else go(std::false_type{}, std::false_type{}); }
        });
    });
    MECHA_CHECK_HIP(hipGetLastError());
    return MECHA_OK;
}

}  // extern "C"
