// gs_adamw.hip -- AdamW over many tensors with moments in 32 or 8 bits, the norm of gradients, the reading of 8-bit moments.
//
// All of it is streaming: per element a step reads and writes parameter, gradient and moments once (28 bytes for float
// tensors with 32-bit moments, 16.06 with 8-bit ones) and computes 20 to 60 instructions, so HBM bounds the large cases and
// launches the small ones.  Hence: one launch for many tensors (their addresses travel as kernel arguments: no table to
// upload, nothing to keep, capturable), a workgroup finds its tensor from its block index.
//
// A tensor is cut into units: a row (1..64 elements) or 64 consecutive elements.  GROUP lanes (1, 4 or 16, the least that
// hold a unit at four elements a lane) work on a unit, so the largest value of a block -- the 8-bit moments' exponent -- is
// a reduction inside a DPP row: no shared memory, no barrier.
#include "gs_common.h"

#include <stdlib.h>

namespace {

typedef unsigned long long u64;
constexpr int UNIT = 64;            // elements of a block where blocks are not rows
constexpr int MAX_TENSORS = 30;     // a batch's table is 3.9 KB of kernel arguments
constexpr int MAX_NORM_TENSORS = 80;
constexpr int NORM_PARTIALS = 4096; // most workgroups that the norm's first pass aims at, beyond one for each tensor

struct AdamwScalars {
    float rate, root, keep, one_minus_beta1, beta2, one_minus_beta2, eps, beta1;   // rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
    uint32_t key;
    int step;
};

struct AdamwTensor {
    void *param;
    const void *grad;
    void *exp_avg, *exp_avg_sq;
    uint8_t *exponents;
    float *master;
    const int8_t *row_mask;
    int32_t *last_step;
    long long numel;
    AdamwScalars k;
    int row_len;
};

struct AdamwBatch {
    const float *grad_scale;
    const AdamwScalars *device_scalars;     // null: each tensor's own k
    int n_tensors;
    unsigned first_chunk[MAX_TENSORS + 1];
    AdamwTensor t[MAX_TENSORS];
};
static_assert(sizeof(AdamwBatch) <= 4096, "a batch's table has to fit the kernel arguments");

// ------------------------------------------------------------------ random bits of the rounding
// Two rounds of xor-shift and multiplication (the multipliers are the first 32 bits of the fractions of sqrt 2 and sqrt 3,
// both odd): every input bit reaches every output bit.
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

__host__ __device__ __forceinline__ uint32_t tensor_key(uint32_t seed, uint32_t tensor, uint32_t step) {
    return mix32(mix32(seed + 0x9E3779B1u * tensor) + step);
}

// One hash serves four consecutive elements, each with another rotation of it; of an element's 32 bits the lower half
// rounds the first moment, the upper half the second.
__device__ __forceinline__ uint32_t element_bits(uint32_t hash, int j) { return __builtin_rotateleft32(hash, 8 * j); }

// ------------------------------------------------------------------ elements
template <int DT>
__device__ __forceinline__ float load_one(const void *p, long long i) {
    if (DT == GS_DTYPE_F32) return ((const float *)p)[i];
    if (DT == GS_DTYPE_BF16) return (float)((const __bf16 *)p)[i];
    return (float)((const _Float16 *)p)[i];
}
template <int DT>
__device__ __forceinline__ void store_one(void *p, long long i, float x) {
    if (DT == GS_DTYPE_F32) ((float *)p)[i] = x;
    else if (DT == GS_DTYPE_BF16) ((__bf16 *)p)[i] = (__bf16)x;      // both round to nearest, ties to even
    else ((_Float16 *)p)[i] = (_Float16)x;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ f32x4 load_four(const void *p, long long i) {
    if (DT == GS_DTYPE_F32) return *(const f32x4 *)((const float *)p + i);
    if (DT == GS_DTYPE_BF16) return __builtin_convertvector(*(const bf16x4 *)((const __bf16 *)p + i), f32x4);
    return __builtin_convertvector(*(const f16x4 *)((const _Float16 *)p + i), f32x4);
}
template <int DT>
__device__ __forceinline__ void store_four(void *p, long long i, f32x4 x) {
    if (DT == GS_DTYPE_F32) *(f32x4 *)((float *)p + i) = x;
    else if (DT == GS_DTYPE_BF16) *(bf16x4 *)((__bf16 *)p + i) = __builtin_convertvector(x, bf16x4);
    else *(f16x4 *)((_Float16 *)p + i) = __builtin_convertvector(x, f16x4);
}

// ------------------------------------------------------------------ 8-bit moments
__device__ __forceinline__ float from_bits(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t to_bits(float x) { return __builtin_bit_cast(uint32_t, x); }

// 2^(X - 127 + shift) for an exponent byte; NaN for 255
__device__ __forceinline__ float exponent_scale(int x, int low, int shift) {
    const int e = x < low ? low : x;
    return x == 255 ? __builtin_nanf("") : from_bits((uint32_t)(e + shift) << 23);
}

__device__ __forceinline__ float decode_m(uint32_t c, float scale) {
    const uint32_t a = c & 127u;
    const float size = a < 8u ? (float)a * 0x1p-9f : from_bits((a + 960u) << 20);
    return (c & 128u ? -size : size) * scale;
}
__device__ __forceinline__ float decode_v(uint32_t c, float scale) {
    return c == 0u ? 0.f * scale : from_bits((c << 20) + (127u << 23)) * scale;
}

// Exponent byte of a block from the bits of its largest magnitude (positive floats order like their bits, NaN above all):
// `carry` moves values whose mantissa is over the largest code's to the next power, so that rounding up stays in range.
__device__ __forceinline__ int block_exponent(uint32_t largest, uint32_t carry, int low) {
    if (largest >= 0x7F800000u) return 255;
    const int x = (int)((largest + carry) >> 23);
    return x < low ? low : (x > 254 ? 254 : x);
}

// |m| 2^(135 - X) to sign, 4 exponent and 3 mantissa bits.  The 20 bits below the third mantissa bit meet 20 random ones
// (16 of them, and a half): the carry into the code has the chance that keeps the mean.  Below 2^-6 the codes are evenly
// spaced: there 2^-6 is added first, so that the same bits are the ones below the code.
__device__ __forceinline__ uint32_t encode_m(float m, float unscale, uint32_t bits) {
    const float t = fabsf(m) * unscale;
    const bool tiny = t < 0x1p-6f;
    const uint32_t u = to_bits(tiny ? t + 0x1p-6f : t) + ((bits & 0xFFFFu) << 4) + 8u;
    uint32_t a = (u >> 20) - (tiny ? 968u : 960u);
    a = a > 126u ? 126u : a;
    return a | (m < 0.f ? 128u : 0u);
}
// v 2^(158 - X) to 5 exponent and 3 mantissa bits; a value over zero stays over zero (it is a divisor's square).
__device__ __forceinline__ uint32_t encode_v(float v, float unscale, uint32_t bits) {
    const int u = (int)(to_bits(v * unscale) - (127u << 23)) ;
    // (u is within +-2^30 except for zero and tiny values, which are the negative ones: the sum does not pass 2^31)
    int c = (u + (int)((bits >> 16) << 4) + 8) >> 20;
    c = c < 1 ? 1 : (c > 255 ? 255 : c);
    return v > 0.f ? (uint32_t)c : 0u;
}

// Largest of GROUP consecutive lanes, in all of them (GROUP = 4: quad permutations, 16: rotations of a DPP row)
template <int GROUP>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
    if (GROUP == 4) {
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
    } else if (GROUP == 16) {
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xF, 0xF, true));
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xF, 0xF, true));
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xF, 0xF, true));
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xF, 0xF, true));
    }
    return x;
}

// Which tensor of a batch a chunk belongs to: every lane compares one entry of the table.
template <int MAX>
__device__ __forceinline__ int find_tensor(const unsigned *first_chunk, int n_tensors, unsigned chunk) {
    static_assert(MAX <= 2 * GS_WAVE, "two entries a lane");
    const int lane = gs_lane();
    int t = __popcll(__ballot(lane < n_tensors && first_chunk[lane < n_tensors ? lane : 0] <= chunk)) - 1;
    if (MAX > GS_WAVE) {
        const int l = lane + GS_WAVE;
        t += __popcll(__ballot(l < n_tensors && first_chunk[l < n_tensors ? l : 0] <= chunk));
    }
    return t;
}

// ------------------------------------------------------------------ the step
// The gradient times the clipping coefficient, rounded to float: clipping on the way gives the bits of a step whose
// gradients were scaled before (contracted into g - m it would not).
__device__ __forceinline__ float scaled(float g, float scale) {
#pragma clang fp contract(off)
    return g * scale;
}

__device__ __forceinline__ float update_one(float p, float g, float &m, float &v, const AdamwScalars &k) {
    m = fmaf(k.one_minus_beta1, g - m, m);
    v = fmaf(k.one_minus_beta2 * g, g, k.beta2 * v);
    const float denom = sqrtf(v) * k.root + k.eps;
    return p * k.keep - k.rate * (m / denom);
}

template <int GROUP>
constexpr int units_per_chunk() { return GS_BLOCK / GROUP; }

// GROUP lanes a unit; VEC: four consecutive elements a lane in one access (aligned buffers, unit lengths that are multiples
// of four), else elements GROUP apart.
template <int GROUP, bool VEC, int DT, bool MASTER, bool STATE8, bool MASKED>
__global__ __launch_bounds__(GS_BLOCK) void adamw_kernel(AdamwBatch b) {
    const int ti = find_tensor<MAX_TENSORS>(b.first_chunk, b.n_tensors, blockIdx.x);
    const AdamwTensor &t = b.t[ti];
    const AdamwScalars k = b.device_scalars ? b.device_scalars[ti] : t.k;
    const float scale = b.grad_scale ? *b.grad_scale : 1.f;
    const int unit_len = t.row_len > 0 ? t.row_len : UNIT;
    const int sub = threadIdx.x % GROUP;
    const long long unit = (long long)(blockIdx.x - b.first_chunk[ti]) * units_per_chunk<GROUP>() + threadIdx.x / GROUP;
    const long long base = unit * unit_len;
    const long long left = t.numel - base;
    const int len = left <= 0 ? 0 : (left < unit_len ? (int)left : unit_len);   // (rows are whole: only a flat tail is shorter)

    bool live = len > 0;
    float decay_m = 1.f, decay_v = 1.f;
    if (MASKED && live) {
        live = t.row_mask[unit] == 0;
        if (live) {
            const int gap = k.step - 1 - t.last_step[unit];
            if (gap > 0) {
                decay_m = powf(k.beta1, (float)gap);
                decay_v = powf(k.beta2, (float)gap);
            }
        }
    }
    const int count = !live ? 0 : (VEC ? max(0, min(4, len - 4 * sub)) : max(0, (len - sub + GROUP - 1) / GROUP));
    // element j of this lane; count of them exist
    const long long lane_base = base + (VEC ? 4 * sub : sub);
    constexpr int STRIDE = VEC ? 1 : GROUP;

    float p[4], g[4], m[4], v[4];
    float scale_m = 1.f, scale_v = 1.f;
    if (STATE8 && live) {
        const uint8_t *e = t.exponents + 2 * unit;
        scale_m = exponent_scale(e[0], 9, -8);
        scale_v = exponent_scale(e[1], 32, -31);
    }
    const void *source = MASTER ? (const void *)t.master : (const void *)t.param;
    constexpr int SOURCE_DT = MASTER ? GS_DTYPE_F32 : DT;
    if (VEC && count == 4) {
        const f32x4 p4 = load_four<SOURCE_DT>(source, lane_base), g4 = load_four<DT>(t.grad, lane_base);
        f32x4 m4, v4;
        if (STATE8) {
            const uint32_t mc = *(const uint32_t *)((const uint8_t *)t.exp_avg + lane_base);
            const uint32_t vc = *(const uint32_t *)((const uint8_t *)t.exp_avg_sq + lane_base);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                m4[j] = decode_m((mc >> (8 * j)) & 255u, scale_m);
                v4[j] = decode_v((vc >> (8 * j)) & 255u, scale_v);
            }
        } else {
            m4 = load_four<GS_DTYPE_F32>(t.exp_avg, lane_base);
            v4 = load_four<GS_DTYPE_F32>(t.exp_avg_sq, lane_base);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { p[j] = p4[j]; g[j] = g4[j]; m[j] = m4[j]; v[j] = v4[j]; }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = g[j] = m[j] = v[j] = 0.f;
            if (j < count) {
                const long long i = lane_base + j * STRIDE;
                p[j] = load_one<SOURCE_DT>(source, i);
                g[j] = load_one<DT>(t.grad, i);
                if (STATE8) {
                    m[j] = decode_m(((const uint8_t *)t.exp_avg)[i], scale_m);
                    v[j] = decode_v(((const uint8_t *)t.exp_avg_sq)[i], scale_v);
                } else {
                    m[j] = ((const float *)t.exp_avg)[i];
                    v[j] = ((const float *)t.exp_avg_sq)[i];
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (MASKED) { m[j] *= decay_m; v[j] *= decay_v; }
        p[j] = update_one(p[j], scaled(g[j], scale), m[j], v[j], k);
        // (a 16-bit parameter is its master copy rounded: without the stop the conversion may join the last operation)
        if (MASTER) asm volatile("" : "+v"(p[j]));
    }

    uint32_t mc[4], vc[4];
    if (STATE8) {
        uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            top_m = j < count ? max(top_m, to_bits(m[j]) & 0x7FFFFFFFu) : top_m;
            top_v = j < count ? max(top_v, to_bits(v[j]) & 0x7FFFFFFFu) : top_v;
        }
        const int xm = block_exponent(group_max<GROUP>(top_m), 0x1FFFFFu, 9);
        const int xv = block_exponent(group_max<GROUP>(top_v), 0x0FFFFFu, 32);
        const float unscale_m = from_bits((uint32_t)(xm == 255 ? 0 : 262 - xm) << 23);
        const float unscale_v = from_bits((uint32_t)(xv == 255 ? 0 : min(285 - xv, 254)) << 23);
        uint32_t hash = mix32((uint32_t)(lane_base >> 2) ^ k.key);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long i = lane_base + j * STRIDE;
            if (!VEC) hash = mix32((uint32_t)(i >> 2) ^ k.key);
            const uint32_t bits = element_bits(hash, VEC ? j : (int)(i & 3));
            mc[j] = xm == 255 ? 0u : encode_m(m[j], unscale_m, bits);
            vc[j] = xv == 255 ? 0u : encode_v(v[j], unscale_v, bits);
        }
        if (live && sub == 0) {
            t.exponents[2 * unit] = (uint8_t)xm;
            t.exponents[2 * unit + 1] = (uint8_t)xv;
        }
    }
    if (MASKED && live && sub == 0) t.last_step[unit] = k.step;

    if (VEC && count == 4) {
        const f32x4 p4 = {p[0], p[1], p[2], p[3]};
        if (MASTER) store_four<GS_DTYPE_F32>(t.master, lane_base, p4);
        store_four<DT>(t.param, lane_base, p4);
        if (STATE8) {
            *(uint32_t *)((uint8_t *)t.exp_avg + lane_base) = mc[0] | mc[1] << 8 | mc[2] << 16 | mc[3] << 24;
            *(uint32_t *)((uint8_t *)t.exp_avg_sq + lane_base) = vc[0] | vc[1] << 8 | vc[2] << 16 | vc[3] << 24;
        } else {
            store_four<GS_DTYPE_F32>(t.exp_avg, lane_base, f32x4{m[0], m[1], m[2], m[3]});
            store_four<GS_DTYPE_F32>(t.exp_avg_sq, lane_base, f32x4{v[0], v[1], v[2], v[3]});
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < count) {
                const long long i = lane_base + j * STRIDE;
                if (MASTER) t.master[i] = p[j];
                store_one<DT>(t.param, i, p[j]);
                if (STATE8) {
                    ((uint8_t *)t.exp_avg)[i] = (uint8_t)mc[j];
                    ((uint8_t *)t.exp_avg_sq)[i] = (uint8_t)vc[j];
                } else {
                    ((float *)t.exp_avg)[i] = m[j];
                    ((float *)t.exp_avg_sq)[i] = v[j];
                }
            }
        }
    }
}

// Scalars of tensors whose step count or learning rate lives on the device.  1 - beta^t is taken as -expm1(t log beta) in
// double precision: for beta2 = 0.999 and t = 1 the difference of two floats would keep three digits.
struct PrepareArgs {
    int n;
    uint32_t seed;
    struct { const long long *step; const float *lr; double lr_host, beta1, beta2, eps, weight_decay; long long step_host; uint32_t tensor; } t[MAX_TENSORS];
};
static_assert(sizeof(PrepareArgs) <= 4096, "kernel arguments");

__host__ __device__ AdamwScalars adamw_scalars(double lr, double beta1, double beta2, double eps, double weight_decay, long long step,
                                               uint32_t seed, uint32_t tensor) {
    AdamwScalars k;
    const double t = (double)step;
    const double bc1 = beta1 > 0.0 ? -expm1(t * log(beta1)) : 1.0, bc2 = beta2 > 0.0 ? -expm1(t * log(beta2)) : 1.0;
    k.rate = (float)(lr / bc1);
    k.root = (float)(1.0 / sqrt(bc2));
    k.keep = (float)(1.0 - lr * weight_decay);
    k.one_minus_beta1 = (float)(1.0 - beta1);
    k.beta2 = (float)beta2;
    k.one_minus_beta2 = (float)(1.0 - beta2);
    k.eps = (float)eps;
    k.beta1 = (float)beta1;
    k.key = tensor_key(seed, tensor, (uint32_t)step);
    k.step = (int)step;
    return k;
}

__global__ void adamw_prepare_kernel(PrepareArgs a, AdamwScalars *out) {
    const int i = threadIdx.x;
    if (i >= a.n) return;
    const auto &t = a.t[i];
    out[i] = adamw_scalars(t.lr ? (double)*t.lr : t.lr_host, t.beta1, t.beta2, t.eps, t.weight_decay, t.step ? *t.step : t.step_host,
                           a.seed, t.tensor);
}

// ------------------------------------------------------------------ reading 8-bit moments
struct MomentsTensor {
    const uint8_t *m, *v, *exponents;
    void *m_out, *v_out;
    long long numel;
    int row_len;
};
struct MomentsBatch {
    int n_tensors;
    unsigned first_chunk[MAX_TENSORS + 1];
    MomentsTensor t[MAX_TENSORS];
};
static_assert(sizeof(MomentsBatch) <= 4096, "kernel arguments");

template <int GROUP, bool VEC, int DT>
__global__ __launch_bounds__(GS_BLOCK) void read_moments_kernel(MomentsBatch b) {
    const int ti = find_tensor<MAX_TENSORS>(b.first_chunk, b.n_tensors, blockIdx.x);
    const MomentsTensor &t = b.t[ti];
    const int unit_len = t.row_len > 0 ? t.row_len : UNIT;
    const int sub = threadIdx.x % GROUP;
    const long long unit = (long long)(blockIdx.x - b.first_chunk[ti]) * units_per_chunk<GROUP>() + threadIdx.x / GROUP;
    const long long base = unit * unit_len;
    const long long left = t.numel - base;
    const int len = left <= 0 ? 0 : (left < unit_len ? (int)left : unit_len);
    if (len == 0) return;
    const float scale_m = exponent_scale(t.exponents[2 * unit], 9, -8), scale_v = exponent_scale(t.exponents[2 * unit + 1], 32, -31);
    if (VEC && 4 * sub + 4 <= len) {
        const long long i = base + 4 * sub;
        const uint32_t mc = *(const uint32_t *)(t.m + i), vc = *(const uint32_t *)(t.v + i);
        f32x4 m4, v4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m4[j] = decode_m((mc >> (8 * j)) & 255u, scale_m);
            v4[j] = decode_v((vc >> (8 * j)) & 255u, scale_v);
        }
        store_four<DT>(t.m_out, i, m4);
        store_four<DT>(t.v_out, i, v4);
    } else {
        for (int j = 0; j < 4; ++j) {
            const int e = VEC ? 4 * sub + j : sub + j * GROUP;
            if (e < len) {
                store_one<DT>(t.m_out, base + e, decode_m(t.m[base + e], scale_m));
                store_one<DT>(t.v_out, base + e, decode_v(t.v[base + e], scale_v));
            }
        }
    }
}

// ------------------------------------------------------------------ norm of gradients
// First pass: each workgroup adds the squares of one chunk in double precision (a float's square is exact there, so the
// result does not depend on the order to within 1e-16) and leaves a partial sum; the second adds the partial sums in a
// fixed order.
struct NormTensor {
    const void *grad;
    const int8_t *row_mask;
    long long numel;
    int row_len, dtype;
    unsigned first_partial;
};
struct NormBatch {
    int n_tensors;
    unsigned chunk;             // elements, a multiple of 1024
    unsigned first_block[MAX_NORM_TENSORS + 1];
    NormTensor t[MAX_NORM_TENSORS];
};
static_assert(sizeof(NormBatch) <= 4096, "kernel arguments");

__device__ __forceinline__ double block_sum(double x) {
    __shared__ double red[GS_BLOCK / GS_WAVE];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, GS_WAVE);
    __syncthreads();
    if (gs_lane() == 0) red[threadIdx.x / GS_WAVE] = x;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < GS_BLOCK / GS_WAVE; ++i) s += red[i];
    return s;
}

template <int DT>
__device__ double sum_of_squares(const NormTensor &t, long long begin, long long end) {
    constexpr int BYTES = DT == GS_DTYPE_F32 ? 4 : 2;
    double s = 0.0;
    if (t.row_mask) {
        for (long long i = begin + threadIdx.x; i < end; i += GS_BLOCK)
            if (t.row_mask[i / t.row_len] == 0) {
                const double g = (double)load_one<DT>(t.grad, i);
                s = fma(g, g, s);
            }
        return s;
    }
    // (begin is a multiple of 1024 elements: the chunk is aligned where the tensor is)
    const bool aligned = ((uintptr_t)t.grad & (4 * BYTES - 1)) == 0;
    const long long fours = aligned ? (end - begin) / 4 : 0;
    for (long long q = threadIdx.x; q < fours; q += GS_BLOCK) {
        const f32x4 g = load_four<DT>(t.grad, begin + 4 * q);
#pragma unroll
        for (int j = 0; j < 4; ++j) s = fma((double)g[j], (double)g[j], s);
    }
    for (long long i = begin + 4 * fours + threadIdx.x; i < end; i += GS_BLOCK) {
        const double g = (double)load_one<DT>(t.grad, i);
        s = fma(g, g, s);
    }
    return s;
}

__global__ __launch_bounds__(GS_BLOCK) void norm_partial_kernel(NormBatch b, int tensor_offset, double *__restrict__ partials,
                                                                unsigned *__restrict__ first_partial) {
    const int ti = find_tensor<MAX_NORM_TENSORS>(b.first_block, b.n_tensors, blockIdx.x);
    const NormTensor &t = b.t[ti];
    const unsigned part = blockIdx.x - b.first_block[ti];
    const long long begin = (long long)part * b.chunk;
    const long long end = min(t.numel, begin + (long long)b.chunk);
    double s = 0.0;
    if (t.dtype == GS_DTYPE_F32) s = sum_of_squares<GS_DTYPE_F32>(t, begin, end);
    else if (t.dtype == GS_DTYPE_BF16) s = sum_of_squares<GS_DTYPE_BF16>(t, begin, end);
    else s = sum_of_squares<GS_DTYPE_F16>(t, begin, end);
    s = block_sum(s);
    if (threadIdx.x == 0) {
        partials[t.first_partial + part] = s;
        if (part == 0) first_partial[tensor_offset + ti] = t.first_partial;
    }
}

__device__ __forceinline__ float clip_of(double sq_sum, double max_norm) {
    if (max_norm <= 0.0) return 1.f;
    const double c = max_norm / (sqrt(sq_sum) + 1e-6);
    return c > 1.0 ? 1.f : (float)c;        // (a norm that is NaN stays visible: the comparison fails)
}

// Block 0 adds up all partial sums, block 1 + i those of tensor i.
__global__ __launch_bounds__(GS_BLOCK) void norm_finish_kernel(const double *__restrict__ partials,
                                                               const unsigned *__restrict__ first_partial, unsigned n_partials,
                                                               int n_tensors, double max_norm, double *sq_sum, float *norm, float *clip,
                                                               float *each) {
    unsigned begin = 0, end = n_partials;
    if (blockIdx.x > 0) {
        const int i = (int)blockIdx.x - 1;
        begin = first_partial[i];
        end = i + 1 < n_tensors ? first_partial[i + 1] : n_partials;
    }
    double s = 0.0;
    for (unsigned i = begin + threadIdx.x; i < end; i += GS_BLOCK) s += partials[i];
    s = block_sum(s);
    if (threadIdx.x != 0) return;
    if (blockIdx.x > 0) {
        each[blockIdx.x - 1] = (float)sqrt(s);
        return;
    }
    *sq_sum = s;
    *norm = (float)sqrt(s);
    *clip = clip_of(s, max_norm);
}

__global__ void clip_coefficient_kernel(const double *sq_sum, double max_norm, float *norm, float *clip) {
    *norm = (float)sqrt(*sq_sum);
    *clip = clip_of(*sq_sum, max_norm);
}

// ------------------------------------------------------------------ host side
struct Range { u64 begin, end; int written; };
int by_begin(const void *a, const void *b) {
    const u64 x = ((const Range *)a)->begin, y = ((const Range *)b)->begin;
    return x < y ? -1 : (x > y ? 1 : 0);
}
// whether a written range meets any other
bool ranges_meet(Range *r, size_t n) {
    qsort(r, n, sizeof(Range), by_begin);
    u64 written_to = 0, any_to = 0;
    for (size_t i = 0; i < n; ++i) {
        if (r[i].begin == r[i].end) continue;
        if (r[i].begin < (r[i].written ? any_to : written_to)) return true;
        any_to = r[i].end > any_to ? r[i].end : any_to;
        if (r[i].written) written_to = r[i].end > written_to ? r[i].end : written_to;
    }
    return false;
}

int element_bytes(int dtype) { return dtype == GS_DTYPE_F32 ? 4 : 2; }
int group_of(int row_len) { return row_len == 0 || row_len > 16 ? 16 : (row_len > 4 ? 4 : 1); }
bool aligned_to(u64 p, u64 bytes) { return p % bytes == 0; }

// The form of the kernel that a tensor takes
struct Variant {
    int group, vec, dtype, master, state8, masked;
    int code() const { return group | vec << 5 | dtype << 6 | master << 8 | state8 << 9 | masked << 10; }
};

template <int GROUP, bool VEC, int DT, bool MASTER, bool STATE8, bool MASKED>
void launch(const AdamwBatch &b, hipStream_t s) {
    hipLaunchKernelGGL((adamw_kernel<GROUP, VEC, DT, MASTER, STATE8, MASKED>), dim3(b.first_chunk[b.n_tensors]), dim3(GS_BLOCK), 0, s, b);
}
template <int GROUP, bool VEC, bool STATE8>
void launch_type(const Variant &v, const AdamwBatch &b, hipStream_t s) {
    if (v.masked) return launch<GROUP, VEC, GS_DTYPE_F32, false, STATE8, true>(b, s);
    if constexpr (STATE8 || GROUP == 16) {      // (moments in 32 bits without a mask: units of 64 whatever the shape)
        if (v.dtype == GS_DTYPE_F32) launch<GROUP, VEC, GS_DTYPE_F32, false, STATE8, false>(b, s);
        else if (v.dtype == GS_DTYPE_BF16 && v.master) launch<GROUP, VEC, GS_DTYPE_BF16, true, STATE8, false>(b, s);
        else if (v.dtype == GS_DTYPE_BF16) launch<GROUP, VEC, GS_DTYPE_BF16, false, STATE8, false>(b, s);
        else if (v.master) launch<GROUP, VEC, GS_DTYPE_F16, true, STATE8, false>(b, s);
        else launch<GROUP, VEC, GS_DTYPE_F16, false, STATE8, false>(b, s);
    }
}
template <int GROUP, bool VEC>
void launch_state(const Variant &v, const AdamwBatch &b, hipStream_t s) {
    if (v.state8) launch_type<GROUP, VEC, true>(v, b, s);
    else launch_type<GROUP, VEC, false>(v, b, s);
}
template <int GROUP>
void launch_group(const Variant &v, const AdamwBatch &b, hipStream_t s) {
    if (v.vec) launch_state<GROUP, true>(v, b, s);
    else launch_state<GROUP, false>(v, b, s);
}
void launch_variant(const Variant &v, const AdamwBatch &b, hipStream_t s) {
    if (v.group == 16) launch_group<16>(v, b, s);
    else if (v.group == 4) launch_group<4>(v, b, s);
    else launch_group<1>(v, b, s);
}

template <int GROUP, bool VEC>
void launch_moments_type(int dtype, const MomentsBatch &b, hipStream_t s) {
    const dim3 grid(b.first_chunk[b.n_tensors]), block(GS_BLOCK);
    if (dtype == GS_DTYPE_F32) hipLaunchKernelGGL((read_moments_kernel<GROUP, VEC, GS_DTYPE_F32>), grid, block, 0, s, b);
    else hipLaunchKernelGGL((read_moments_kernel<GROUP, VEC, GS_DTYPE_BF16>), grid, block, 0, s, b);
}
void launch_moments(int group, bool vec, int dtype, const MomentsBatch &b, hipStream_t s) {
    if (group == 16) vec ? launch_moments_type<16, true>(dtype, b, s) : launch_moments_type<16, false>(dtype, b, s);
    else if (group == 4) vec ? launch_moments_type<4, true>(dtype, b, s) : launch_moments_type<4, false>(dtype, b, s);
    else vec ? launch_moments_type<1, true>(dtype, b, s) : launch_moments_type<1, false>(dtype, b, s);
}

long long units_of(long long numel, int row_len) { return row_len > 0 ? numel / row_len : (numel + UNIT - 1) / UNIT; }
long long chunks_of(long long numel, int row_len) {
    const int per = GS_BLOCK / group_of(row_len);
    return (units_of(numel, row_len) + per - 1) / per;
}

}  // namespace

extern "C" long long gs_adamw_workspace_bytes(int n_tensors) { return n_tensors < 0 ? 0 : (long long)n_tensors * (long long)sizeof(AdamwScalars); }

extern "C" int gs_adamw_step(int n_tensors, const uint64_t *host_param, const uint64_t *host_grad, const uint64_t *host_exp_avg,
                             const uint64_t *host_exp_avg_sq, const uint64_t *host_exponents, const uint64_t *host_master,
                             const uint64_t *host_row_mask, const uint64_t *host_last_step, const int64_t *host_numel,
                             const int32_t *host_row_len, const int32_t *host_dtype, const int32_t *host_tensor_id,
                             const double *host_hyper, const int64_t *host_step, const uint64_t *host_step_device,
                             const uint64_t *host_lr_device, const float *grad_scale, uint32_t seed, void *workspace, void *stream) {
    GS_REQUIRE(n_tensors >= 0 && n_tensors <= (1 << 20), "gs_adamw_step: 0 to 2^20 tensors");
    if (n_tensors == 0) return 0;
    GS_REQUIRE(host_param && host_grad && host_exp_avg && host_exp_avg_sq && host_numel && host_row_len && host_dtype &&
                   host_tensor_id && host_hyper && host_step, "gs_adamw_step: null array");
    GS_REQUIRE((host_row_mask == nullptr) == (host_last_step == nullptr), "gs_adamw_step: row masks come with last steps");
    const bool on_device = host_step_device || host_lr_device;
    GS_REQUIRE(!on_device || workspace, "gs_adamw_step: a step count or learning rate on the device needs the workspace");
    for (int i = 0; i < n_tensors; ++i) {
        const long long n = host_numel[i];
        const int row = host_row_len[i], dt = host_dtype[i];
        const double *h = host_hyper + 5 * (size_t)i;
        GS_REQUIRE(n >= 0 && n < (1LL << 46) && row >= 0 && row <= UNIT && (row == 0 || n % row == 0),
                   "gs_adamw_step: numel in [0, 2^46), too large else, rows of 1..64 elements");
        GS_REQUIRE(dt == GS_DTYPE_F32 || dt == GS_DTYPE_BF16 || dt == GS_DTYPE_F16, "gs_adamw_step: unknown dtype");
        GS_REQUIRE(chunks_of(n, row) < 0x7fffffffLL, "gs_adamw_step: tensor too large");
        GS_REQUIRE(n == 0 || (host_param[i] && host_grad[i] && host_exp_avg[i] && host_exp_avg_sq[i] && (!host_exponents || host_exponents[i])),
                   "gs_adamw_step: null tensor");
        const bool masked = host_row_mask && host_row_mask[i];
        GS_REQUIRE(!masked || (row > 0 && dt == GS_DTYPE_F32 && host_last_step[i]), "gs_adamw_step: a row mask needs float rows and last steps");
        GS_REQUIRE(!(host_master && host_master[i]) || dt != GS_DTYPE_F32, "gs_adamw_step: a master copy belongs to a 16-bit parameter");
        GS_REQUIRE((host_step[i] >= 1 && host_step[i] < 0x7fffffffLL) || (host_step_device && host_step_device[i]), "gs_adamw_step: step >= 1");
        GS_REQUIRE(h[1] >= 0.0 && h[1] < 1.0 && h[2] >= 0.0 && h[2] < 1.0 && h[3] >= 0.0, "gs_adamw_step: betas in [0, 1), eps >= 0");
        GS_REQUIRE(aligned_to(host_param[i] | host_grad[i], element_bytes(dt)) &&
                       aligned_to((host_exponents ? 0 : host_exp_avg[i] | host_exp_avg_sq[i]) | (host_master ? host_master[i] : 0), 4),
                   "gs_adamw_step: an address is no multiple of its type's size");
    }
    {
        Range *r = (Range *)malloc((size_t)n_tensors * 7 * sizeof(Range));
        GS_REQUIRE(r != nullptr, "gs_adamw_step: out of host memory");
        size_t k = 0;
        for (int i = 0; i < n_tensors; ++i) {
            const u64 n = (u64)host_numel[i], pe = n * element_bytes(host_dtype[i]), se = n * (host_exponents ? 1 : 4);
            r[k++] = {host_param[i], host_param[i] + pe, 1};
            r[k++] = {host_grad[i], host_grad[i] + pe, 0};
            r[k++] = {host_exp_avg[i], host_exp_avg[i] + se, 1};
            r[k++] = {host_exp_avg_sq[i], host_exp_avg_sq[i] + se, 1};
            if (host_exponents) r[k++] = {host_exponents[i], host_exponents[i] + 2 * (u64)units_of(host_numel[i], host_row_len[i]), 1};
            if (host_master && host_master[i]) r[k++] = {host_master[i], host_master[i] + 4 * n, 1};
            if (host_row_mask && host_row_mask[i]) r[k++] = {host_last_step[i], host_last_step[i] + 4 * (u64)units_of(host_numel[i], host_row_len[i]), 1};
        }
        const bool meet = ranges_meet(r, k);
        free(r);
        GS_REQUIRE(!meet, "gs_adamw_step: buffers overlap");
    }
    hipStream_t s = (hipStream_t)stream;
    unsigned char *done = (unsigned char *)calloc((size_t)n_tensors, 1);
    GS_REQUIRE(done != nullptr, "gs_adamw_step: out of host memory");
    AdamwScalars *device_scalars = on_device ? (AdamwScalars *)workspace : nullptr;
    AdamwBatch b;
    PrepareArgs prep;
    b.grad_scale = grad_scale;
    // Tensors that take the same form of the kernel go together, in batches of MAX_TENSORS.
    for (int first = 0; first < n_tensors; ++first) {
        if (done[first]) continue;
        int form = -1;
        Variant variant = {};
        b.n_tensors = 0;
        b.first_chunk[0] = 0;
        for (int i = first; i < n_tensors; ++i) {
            if (done[i]) continue;
            if (host_numel[i] == 0) { done[i] = 1; continue; }
            const int dt = host_dtype[i];
            Variant v;
            v.masked = host_row_mask && host_row_mask[i];
            v.state8 = host_exponents != nullptr;
            v.master = host_master && host_master[i];
            v.dtype = dt;
            const int row = v.masked || v.state8 ? host_row_len[i] : 0;
            v.group = group_of(row);
            v.vec = row % 4 == 0 && aligned_to(host_param[i] | host_grad[i], 4 * element_bytes(dt)) &&
                    aligned_to(host_exp_avg[i] | host_exp_avg_sq[i], v.state8 ? 4 : 16) && aligned_to(v.master ? host_master[i] : 0, 16);
            if (form >= 0 && v.code() != form) continue;
            const long long chunks = chunks_of(host_numel[i], row);
            if (b.n_tensors == MAX_TENSORS || (long long)b.first_chunk[b.n_tensors] + chunks >= 0x7fffffffLL) break;
            form = v.code();
            variant = v;
            done[i] = 1;
            AdamwTensor &t = b.t[b.n_tensors];
            t.param = (void *)host_param[i];
            t.grad = (const void *)host_grad[i];
            t.exp_avg = (void *)host_exp_avg[i];
            t.exp_avg_sq = (void *)host_exp_avg_sq[i];
            t.exponents = v.state8 ? (uint8_t *)host_exponents[i] : nullptr;
            t.master = v.master ? (float *)host_master[i] : nullptr;
            t.row_mask = v.masked ? (const int8_t *)host_row_mask[i] : nullptr;
            t.last_step = v.masked ? (int32_t *)host_last_step[i] : nullptr;
            t.numel = host_numel[i];
            t.row_len = row;
            const double *h = host_hyper + 5 * (size_t)i;
            if (on_device) {
                auto &q = prep.t[b.n_tensors];
                q.step = host_step_device ? (const long long *)host_step_device[i] : nullptr;
                q.lr = host_lr_device ? (const float *)host_lr_device[i] : nullptr;
                q.lr_host = h[0]; q.beta1 = h[1]; q.beta2 = h[2]; q.eps = h[3]; q.weight_decay = h[4];
                q.step_host = host_step[i];
                q.tensor = (uint32_t)host_tensor_id[i];
            } else {
                t.k = adamw_scalars(h[0], h[1], h[2], h[3], h[4], host_step[i], seed, (uint32_t)host_tensor_id[i]);
            }
            b.first_chunk[b.n_tensors + 1] = b.first_chunk[b.n_tensors] + (unsigned)chunks;
            ++b.n_tensors;
        }
        if (b.n_tensors == 0) continue;
        b.device_scalars = device_scalars;
        if (on_device) {
            prep.n = b.n_tensors;
            prep.seed = seed;
            hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(GS_WAVE), 0, s, prep, device_scalars);
            device_scalars += b.n_tensors;      // (every batch has its own part: at most n_tensors in all)
        }
        launch_variant(variant, b, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            free(done);
            gs_set_error("gs_adamw_step: kernel launch failed: %s", hipGetErrorString(e));
            return -3;
        }
    }
    free(done);
    return 0;
}

extern "C" int gs_read_moments(int n_tensors, const uint64_t *host_exp_avg, const uint64_t *host_exp_avg_sq,
                               const uint64_t *host_exponents, const uint64_t *host_m_out, const uint64_t *host_v_out,
                               const int64_t *host_numel, const int32_t *host_row_len, int out_dtype, void *stream) {
    GS_REQUIRE(n_tensors >= 0 && n_tensors <= (1 << 20), "gs_read_moments: 0 to 2^20 tensors");
    if (n_tensors == 0) return 0;
    GS_REQUIRE(host_exp_avg && host_exp_avg_sq && host_exponents && host_m_out && host_v_out && host_numel && host_row_len,
               "gs_read_moments: null array");
    GS_REQUIRE(out_dtype == GS_DTYPE_F32 || out_dtype == GS_DTYPE_BF16, "gs_read_moments: values in float or bfloat16");
    for (int i = 0; i < n_tensors; ++i) {
        const long long n = host_numel[i];
        const int row = host_row_len[i];
        GS_REQUIRE(n >= 0 && n < (1LL << 46) && row >= 0 && row <= UNIT && (row == 0 || n % row == 0),
                   "gs_read_moments: numel in [0, 2^46), rows of 1..64 elements");
        GS_REQUIRE(chunks_of(n, row) < 0x7fffffffLL, "gs_read_moments: tensor too large");
        GS_REQUIRE(n == 0 || (host_exp_avg[i] && host_exp_avg_sq[i] && host_exponents[i] && host_m_out[i] && host_v_out[i]),
                   "gs_read_moments: null tensor");
        GS_REQUIRE(aligned_to(host_m_out[i] | host_v_out[i], element_bytes(out_dtype)), "gs_read_moments: misaligned output");
    }
    unsigned char *done = (unsigned char *)calloc((size_t)n_tensors, 1);
    GS_REQUIRE(done != nullptr, "gs_read_moments: out of host memory");
    MomentsBatch b;
    for (int first = 0; first < n_tensors; ++first) {
        if (done[first]) continue;
        int form = -1;
        b.n_tensors = 0;
        b.first_chunk[0] = 0;
        for (int i = first; i < n_tensors; ++i) {
            if (done[i]) continue;
            if (host_numel[i] == 0) { done[i] = 1; continue; }
            const int row = host_row_len[i];
            const bool vec = row % 4 == 0 && aligned_to(host_exp_avg[i] | host_exp_avg_sq[i], 4) &&
                             aligned_to(host_m_out[i] | host_v_out[i], 4 * element_bytes(out_dtype));
            const int code = group_of(row) | (int)vec << 5;
            if (form >= 0 && code != form) continue;
            const long long chunks = chunks_of(host_numel[i], row);
            if (b.n_tensors == MAX_TENSORS || (long long)b.first_chunk[b.n_tensors] + chunks >= 0x7fffffffLL) break;
            form = code;
            done[i] = 1;
            b.t[b.n_tensors] = {(const uint8_t *)host_exp_avg[i], (const uint8_t *)host_exp_avg_sq[i], (const uint8_t *)host_exponents[i],
                                (void *)host_m_out[i], (void *)host_v_out[i], host_numel[i], row};
            b.first_chunk[b.n_tensors + 1] = b.first_chunk[b.n_tensors] + (unsigned)chunks;
            ++b.n_tensors;
        }
        if (b.n_tensors == 0) continue;
        launch_moments(form & 31, form >> 5, out_dtype, b, (hipStream_t)stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            free(done);
            gs_set_error("gs_read_moments: kernel launch failed: %s", hipGetErrorString(e));
            return -3;
        }
    }
    free(done);
    return 0;
}

extern "C" long long gs_grad_norm_workspace_bytes(int n_tensors) {
    return n_tensors < 0 ? 0 : ((long long)NORM_PARTIALS + n_tensors) * 8 + (long long)n_tensors * 4;
}

extern "C" int gs_grad_norm(int n_tensors, const uint64_t *host_grad, const uint64_t *host_row_mask, const int64_t *host_numel,
                            const int32_t *host_row_len, const int32_t *host_dtype, double max_norm, double *sq_sum, float *norm,
                            float *clip, float *each, void *workspace, void *stream) {
    GS_REQUIRE(n_tensors >= 1 && n_tensors <= (1 << 20), "gs_grad_norm: 1 to 2^20 tensors");
    GS_REQUIRE(host_grad && host_numel && host_row_len && host_dtype && sq_sum && norm && clip && workspace, "gs_grad_norm: null pointer");
    GS_REQUIRE(((uintptr_t)workspace & 7) == 0, "gs_grad_norm: the workspace must be 8-byte aligned");
    long long total = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const long long n = host_numel[i];
        const int dt = host_dtype[i];
        GS_REQUIRE(n >= 0 && n < (1LL << 46), "gs_grad_norm: numel >= 0");
        GS_REQUIRE(dt == GS_DTYPE_F32 || dt == GS_DTYPE_BF16 || dt == GS_DTYPE_F16, "gs_grad_norm: unknown dtype");
        GS_REQUIRE(n == 0 || (host_grad[i] && aligned_to(host_grad[i], element_bytes(dt))), "gs_grad_norm: null or misaligned tensor");
        GS_REQUIRE(!(host_row_mask && host_row_mask[i]) || (host_row_len[i] > 0 && n % host_row_len[i] == 0), "gs_grad_norm: a row mask needs rows");
        total += n;
    }
    // chunks of a multiple of 1024 elements, so that there are at most NORM_PARTIALS of them and one more for each tensor
    long long chunk = (total + NORM_PARTIALS - 1) / NORM_PARTIALS;
    chunk = chunk < 4096 ? 4096 : (chunk + 1023) / 1024 * 1024;
    GS_REQUIRE(chunk < 0x7fffffffLL, "gs_grad_norm: too many elements");
    hipStream_t s = (hipStream_t)stream;
    double *partials = (double *)workspace;
    unsigned *first_partial = (unsigned *)(partials + NORM_PARTIALS + n_tensors);
    unsigned n_partials = 0;
    NormBatch b;
    b.chunk = (unsigned)chunk;
    for (int first = 0; first < n_tensors; first += MAX_NORM_TENSORS) {
        b.n_tensors = n_tensors - first < MAX_NORM_TENSORS ? n_tensors - first : MAX_NORM_TENSORS;
        b.first_block[0] = 0;
        for (int j = 0; j < b.n_tensors; ++j) {
            const int i = first + j;
            // (a tensor without elements has one partial sum too: zero)
            const unsigned parts = host_numel[i] == 0 ? 1u : (unsigned)((host_numel[i] + chunk - 1) / chunk);
            b.t[j] = {(const void *)host_grad[i], host_row_mask ? (const int8_t *)host_row_mask[i] : nullptr, host_numel[i],
                      host_row_len[i], host_dtype[i], n_partials};
            n_partials += parts;
            b.first_block[j + 1] = b.first_block[j] + parts;
        }
        hipLaunchKernelGGL(norm_partial_kernel, dim3(b.first_block[b.n_tensors]), dim3(GS_BLOCK), 0, s, b, first, partials, first_partial);
        GS_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(norm_finish_kernel, dim3(each ? 1 + n_tensors : 1), dim3(GS_BLOCK), 0, s, partials, first_partial, n_partials,
                       n_tensors, max_norm, sq_sum, norm, clip, each);
    GS_CHECK_LAUNCH();
    return 0;
}

extern "C" int gs_clip_coefficient(const double *sq_sum, double max_norm, float *norm, float *clip, void *stream) {
    GS_REQUIRE(sq_sum && norm && clip, "gs_clip_coefficient: null pointer");
    hipLaunchKernelGGL(clip_coefficient_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, sq_sum, max_norm, norm, clip);
    GS_CHECK_LAUNCH();
    return 0;
}
