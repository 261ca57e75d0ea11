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
#include <string.h>

#include <algorithm>

namespace {

typedef unsigned long long u64;
constexpr int UNIT = 64;            // elements of a block where blocks are not rows
constexpr int MAX_TENSORS = 48;     // a batch's table is 3.9 KB of kernel arguments
constexpr int MAX_SETS = 4;         // different (learning rate, step, ...) in a batch
constexpr int MAX_NORM_TENSORS = 160, MAX_NORM_MASKED = 64;
constexpr int NORM_PARTIALS = 4096; // most workgroups that the norm's first pass aims at, beyond one for each tensor

// What a step needs besides the tensors; key and step belong to one tensor
struct AdamwScalars {
    float rate, root, keep, one_minus_beta1, beta2, one_minus_beta2, eps, beta1;   // rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
    int step;
    uint32_t key;
};

// How a tensor is cut among lanes
enum Form : int {
    FOURS,          // units of 64, or rows of 20, 24 .. 64 elements: 16 lanes a unit, four consecutive elements a lane
    FOURS_MASKED,   // the same rows under a mask: a wave packs the live ones of 64 rows
    NARROW,         // float rows of 1 to 4 elements: four rows a lane
    ELEMENTS        // anything else, unaligned tensors: element by element
};

struct AdamwTensor {
    void *param;
    const void *grad;
    void *exp_avg, *exp_avg_sq;
    uint8_t *exponents;
    void *master_or_mask;       // float master copy of a 16-bit parameter, or the row mask of a float one
    int32_t *last_step;
    long long numel;
    uint32_t key;
    uint8_t row_len, form, masked, set;
};

struct AdamwBatch {
    const float *grad_scale;
    const AdamwScalars *device_scalars;     // null: scalars[t.set] and t.key
    int n_tensors;
    unsigned first_chunk[MAX_TENSORS + 1];
    AdamwScalars scalars[MAX_SETS];
    AdamwTensor t[MAX_TENSORS];
};
static_assert(sizeof(AdamwBatch) <= 4000, "a batch's table has to fit the kernel arguments");

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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <int DT> struct Four;
template <> struct Four<GS_DTYPE_F32> { typedef f32x4 type; };
template <> struct Four<GS_DTYPE_BF16> { typedef bf16x4 type; };
template <> struct Four<GS_DTYPE_F16> { typedef f16x4 type; };

// sixteen bytes
template <int DT> struct Wide;
template <> struct Wide<GS_DTYPE_F32> { typedef f32x4 type; };
template <> struct Wide<GS_DTYPE_BF16> { typedef bf16x8 type; };
template <> struct Wide<GS_DTYPE_F16> { typedef f16x8 type; };

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

// Four codes of each moment (the first in the lowest byte) under the exponent bytes X_m | X_v << 8
__device__ __forceinline__ void decode_four(uint32_t mc, uint32_t vc, uint32_t x, f32x4 &m, f32x4 &v) {
    const float scale_m = exponent_scale((int)(x & 255u), 9, -8), scale_v = exponent_scale((int)(x >> 8 & 255u), 32, -31);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = decode_m((mc >> (8 * j)) & 255u, scale_m);
        v[j] = decode_v((vc >> (8 * j)) & 255u, scale_v);
    }
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
__device__ __forceinline__ uint32_t encode_m(float m, int x, uint32_t bits) {
    if (x == 255) return 0u;
    const float unscale = from_bits((uint32_t)(262 - x) << 23);
    const float t = fabsf(m) * unscale;
    const bool tiny = t < 0x1p-6f;
    const uint32_t u = to_bits(tiny ? t + 0x1p-6f : t) + ((bits & 0xFFFFu) << 4) + 8u;
    uint32_t a = (u >> 20) - (tiny ? 968u : 960u);
    a = a > 126u ? 126u : a;
    return a | (m < 0.f ? 128u : 0u);
}
// v 2^(158 - X) to 5 exponent and 3 mantissa bits; a value over zero stays over zero (it is a divisor's square).
__device__ __forceinline__ uint32_t encode_v(float v, int x, uint32_t bits) {
    if (x == 255) return 0u;
    const float unscale = from_bits((uint32_t)(285 - x) << 23);
    const int u = (int)(to_bits(v * unscale) - (127u << 23));
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

// Which tensor of a batch a chunk belongs to: every lane compares entries of the table.
template <int MAX>
__device__ __forceinline__ int find_tensor(const unsigned *first_chunk, int n_tensors, unsigned chunk) {
    int t = -1;
#pragma unroll
    for (int l = 0; l < MAX; l += GS_WAVE) {
        const int i = l + gs_lane();
        t += __popcll(__ballot(i < n_tensors && first_chunk[i < n_tensors ? i : 0] <= chunk));
    }
    return __builtin_amdgcn_readfirstlane(t);
}

// ------------------------------------------------------------------ the step
// The gradient times the clipping coefficient, rounded to float: clipping on the way gives the bits of a step whose
// gradients were scaled before (contracted into g - m it would not).
__device__ __forceinline__ float scaled(float g, float scale) {
#pragma clang fp contract(off)
    return g * scale;
}

// The moments in 32 bits take the correctly rounded square root and division (they are hidden behind 28 bytes an element);
// with 8 bits hardware's own, one unit in the last place each, are as good: the moments' codes do not depend on them.
template <bool FAST, bool MASTER>
__device__ __forceinline__ float update_one(float p, float g, float &m, float &v, const AdamwScalars &k) {
    m = fmaf(k.one_minus_beta1, g - m, m);
    v = fmaf(k.one_minus_beta2 * g, g, k.beta2 * v);
    float change;
    if (FAST) change = m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * k.root + k.eps);
    else change = m / (sqrtf(v) * k.root + k.eps);
    p = p * k.keep - k.rate * change;
    // (a 16-bit parameter is its master copy rounded: without the stop the conversion may join the last operation)
    if (MASTER) asm volatile("" : "+v"(p));
    return p;
}

// What a row that was last stepped at `last` has to be multiplied with before this step
__device__ __forceinline__ void row_decay(const AdamwScalars &k, int last, float &decay_m, float &decay_v) {
    const int gap = k.step - 1 - last;
    if (gap > 0) {
        decay_m = powf(k.beta1, (float)gap);
        decay_v = powf(k.beta2, (float)gap);
    }
}

// Codes and exponents of a block from the lanes that share it: four elements a lane
template <int GROUP>
__device__ __forceinline__ uint32_t encode_four(const f32x4 &m, const f32x4 &v, uint32_t hash, uint32_t &mc, uint32_t &vc) {
    uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        top_m = max(top_m, to_bits(m[j]) & 0x7FFFFFFFu);
        top_v = max(top_v, to_bits(v[j]) & 0x7FFFFFFFu);
    }
    const int xm = block_exponent(group_max<GROUP>(top_m), 0x1FFFFFu, 9), xv = block_exponent(group_max<GROUP>(top_v), 0x0FFFFFu, 32);
    mc = vc = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t bits = element_bits(hash, j);
        mc |= encode_m(m[j], xm, bits) << (8 * j);
        vc |= encode_v(v[j], xv, bits) << (8 * j);
    }
    return (uint32_t)(xm | xv << 8);
}

template <bool FAST, bool MASTER>
__device__ __forceinline__ void update_four(f32x4 &p, const f32x4 &g, f32x4 &m, f32x4 &v, float scale, const AdamwScalars &k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float mj = m[j], vj = v[j];
        p[j] = update_one<FAST, MASTER>(p[j], scaled(g[j], scale), mj, vj, k);
        m[j] = mj;
        v[j] = vj;
    }
}

// Four consecutive elements a lane: what a lane reads before the step and writes after it
template <int DT, bool MASTER, bool STATE8>
struct Quad {
    typename Four<MASTER ? GS_DTYPE_F32 : DT>::type p;
    typename Four<DT>::type g;
    f32x4 m, v;
    uint32_t mc, vc;

    __device__ __forceinline__ void clear() {
        p = {};
        g = {};
        m = v = f32x4{0.f, 0.f, 0.f, 0.f};
        mc = vc = 0u;
    }
    __device__ __forceinline__ void load(const AdamwTensor &t, long long i) {
        p = *(const decltype(p) *)((const char *)(MASTER ? t.master_or_mask : t.param) + i * (long long)(sizeof(p) / 4));
        g = *(const decltype(g) *)((const char *)t.grad + i * (long long)(sizeof(g) / 4));
        if (STATE8) {
            mc = *(const uint32_t *)((const uint8_t *)t.exp_avg + i);
            vc = *(const uint32_t *)((const uint8_t *)t.exp_avg_sq + i);
        } else {
            m = *(const f32x4 *)((const float *)t.exp_avg + i);
            v = *(const f32x4 *)((const float *)t.exp_avg_sq + i);
        }
    }
    // The step; returns the exponent bytes of the block that GROUP lanes share
    template <int GROUP>
    __device__ __forceinline__ uint32_t step(f32x4 &out, uint32_t x, float decay_m, float decay_v, long long i, float scale, const AdamwScalars &k) {
        out = __builtin_convertvector(p, f32x4);
        if (STATE8) decode_four(mc, vc, x, m, v);
        m *= decay_m;
        v *= decay_v;
        update_four<STATE8, MASTER>(out, __builtin_convertvector(g, f32x4), m, v, scale, k);
        return STATE8 ? encode_four<GROUP>(m, v, mix32((uint32_t)(i >> 2) ^ k.key), mc, vc) : 0u;
    }
    __device__ __forceinline__ void store(const AdamwTensor &t, long long i, const f32x4 &out) const {
        if (MASTER) *(f32x4 *)((float *)t.master_or_mask + i) = out;
        *(decltype(g) *)((char *)t.param + i * (long long)(sizeof(g) / 4)) = __builtin_convertvector(out, decltype(g));
        if (STATE8) {
            *(uint32_t *)((uint8_t *)t.exp_avg + i) = mc;
            *(uint32_t *)((uint8_t *)t.exp_avg_sq + i) = vc;
        } else {
            *(f32x4 *)((float *)t.exp_avg + i) = m;
            *(f32x4 *)((float *)t.exp_avg_sq + i) = v;
        }
    }
};

// The element-wise form: GROUP lanes take a unit, elements GROUP apart.
template <int GROUP, int DT, bool MASTER, bool STATE8>
__device__ __forceinline__ void step_unit(const AdamwTensor &t, const AdamwScalars &k, float scale, long long unit, int unit_len) {
    const int sub = threadIdx.x % GROUP;
    const long long base = unit * unit_len;
    const long long left = t.numel - base;
    const int len = left <= 0 ? 0 : (left < unit_len ? (int)left : unit_len);   // (rows are whole: only a flat tail is shorter)
    bool live = len > 0;
    float decay_m = 1.f, decay_v = 1.f;
    const bool masked = DT == GS_DTYPE_F32 && t.masked;
    if (masked && live) {
        live = ((const int8_t *)t.master_or_mask)[unit] == 0;
        if (live) row_decay(k, t.last_step[unit], decay_m, decay_v);
    }
    const int count = live ? max(0, (len - sub + GROUP - 1) / GROUP) : 0;     // element j of this lane exists for j < count
    float p[4], m[4], v[4];
    float scale_m = 1.f, scale_v = 1.f;
    if (STATE8 && live) {
        scale_m = exponent_scale(t.exponents[2 * unit], 9, -8);
        scale_v = exponent_scale(t.exponents[2 * unit + 1], 32, -31);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float g = 0.f;
        p[j] = m[j] = v[j] = 0.f;
        if (j < count) {
            const long long i = base + sub + j * GROUP;
            p[j] = MASTER ? ((const float *)t.master_or_mask)[i] : load_one<DT>(t.param, i);
            g = load_one<DT>(t.grad, i);
            if (STATE8) {
                m[j] = decode_m(((const uint8_t *)t.exp_avg)[i], scale_m);
                v[j] = decode_v(((const uint8_t *)t.exp_avg_sq)[i], scale_v);
            } else {
                m[j] = ((const float *)t.exp_avg)[i];
                v[j] = ((const float *)t.exp_avg_sq)[i];
            }
        }
        m[j] *= decay_m;
        v[j] *= decay_v;
        p[j] = update_one<STATE8, MASTER>(p[j], scaled(g, scale), m[j], v[j], k);
    }
    int xm = 0, xv = 0;
    if (STATE8) {
        uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            top_m = j < count ? max(top_m, to_bits(m[j]) & 0x7FFFFFFFu) : top_m;
            top_v = j < count ? max(top_v, to_bits(v[j]) & 0x7FFFFFFFu) : top_v;
        }
        xm = block_exponent(group_max<GROUP>(top_m), 0x1FFFFFu, 9);
        xv = block_exponent(group_max<GROUP>(top_v), 0x0FFFFFu, 32);
        if (live && sub == 0) {
            t.exponents[2 * unit] = (uint8_t)xm;
            t.exponents[2 * unit + 1] = (uint8_t)xv;
        }
    }
    if (masked && live && sub == 0) t.last_step[unit] = k.step;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j < count) {
            const long long i = base + sub + j * GROUP;
            if (MASTER) ((float *)t.master_or_mask)[i] = p[j];
            store_one<DT>(t.param, i, p[j]);
            if (STATE8) {
                const uint32_t bits = element_bits(mix32((uint32_t)(i >> 2) ^ k.key), (int)(i & 3));
                ((uint8_t *)t.exp_avg)[i] = (uint8_t)encode_m(m[j], xm, bits);
                ((uint8_t *)t.exp_avg_sq)[i] = (uint8_t)encode_v(v[j], xv, bits);
            } else {
                ((float *)t.exp_avg)[i] = m[j];
                ((float *)t.exp_avg_sq)[i] = v[j];
            }
        }
    }
}

// A workgroup's share in units is 16 (of 16 lanes) times UNROLL; a lane asks for all its units' data before it uses any.
template <int UNROLL, int DT, bool MASTER, bool STATE8>
__device__ __forceinline__ void step_fours(const AdamwTensor &t, const AdamwScalars &k, float scale, unsigned chunk) {
    constexpr int GROUP = 16, PER_PASS = GS_BLOCK / GROUP;
    const int unit_len = t.row_len > 0 ? t.row_len : UNIT;
    const long long chunk_unit = (long long)chunk * (PER_PASS * UNROLL);
    const long long unit0 = chunk_unit + threadIdx.x / GROUP;
    const long long whole = t.numel / unit_len;         // units of full length
    const int sub = threadIdx.x % GROUP;
    Quad<DT, MASTER, STATE8> q[UNROLL];
    uint32_t x[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long unit = unit0 + u * PER_PASS;
        q[u].clear();
        x[u] = 0u;
        if (unit < whole && 4 * sub < unit_len) {
            q[u].load(t, unit * unit_len + 4 * sub);
            if (STATE8) x[u] = *(const uint16_t *)(t.exponents + 2 * unit);
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long unit = unit0 + u * PER_PASS;
        const long long i = unit * unit_len + 4 * sub;
        f32x4 p;
        // (a lane past its row's end holds zeros, and NaN only where the clipping coefficient makes NaN of all)
        const uint32_t new_x = q[u].template step<GROUP>(p, x[u], 1.f, 1.f, i, scale, k);
        if (unit < whole && 4 * sub < unit_len) {
            q[u].store(t, i, p);
            if (STATE8 && sub == 0) *(uint16_t *)(t.exponents + 2 * unit) = (uint16_t)new_x;
        }
    }
    // the last unit of a flat tensor, where it is shorter
    if (whole * unit_len < t.numel && whole >= chunk_unit && whole < chunk_unit + PER_PASS * UNROLL && threadIdx.x < GS_WAVE)
        step_unit<GROUP, DT, MASTER, STATE8>(t, k, scale, whole + threadIdx.x / GROUP, unit_len);
}

// Rows under a mask: a wave reads the mask and the stamps of 64 rows, packs the live ones and steps them four at a time, so
// that no lane waits beside a row without a point and none of such a row's data is asked for.
template <int UNROLL, bool STATE8>
__device__ __forceinline__ void step_fours_masked(const AdamwTensor &t, const AdamwScalars &k, float scale, unsigned chunk) {
    constexpr int GROUP = 16;
    const int row_len = t.row_len, lane = gs_lane(), sub = lane % GROUP;
    const long long row0 = ((long long)chunk * (GS_BLOCK / GS_WAVE) + threadIdx.x / GS_WAVE) * GS_WAVE;
    const long long mine = row0 + lane, rows = t.numel / row_len;
    const bool live = mine < rows && ((const int8_t *)t.master_or_mask)[mine < rows ? mine : 0] == 0;
    const u64 lives = __ballot(live);
    if (lives == 0) return;
    float decay_m = 1.f, decay_v = 1.f;
    int x = 0;
    if (live) {
        row_decay(k, t.last_step[mine], decay_m, decay_v);
        t.last_step[mine] = k.step;
        if (STATE8) x = *(const uint16_t *)(t.exponents + 2 * mine);
    }
    // lane i learns which lane has the i-th live row
    const int rank = __popcll(lives & ((1ull << lane) - 1ull)), n_live = __popcll(lives);
    const int order = __builtin_amdgcn_ds_permute(4 * (live ? rank : 63 - __popcll(~lives & ((1ull << lane) - 1ull))), lane);
    const bool any_late = __ballot(decay_m != 1.f || decay_v != 1.f) != 0;
    for (int at = 0; at < n_live; at += 4 * UNROLL) {
        Quad<GS_DTYPE_F32, false, STATE8> q[UNROLL];
        int from[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = at + 4 * u + lane / GROUP;
            from[u] = __shfl(order, i < n_live ? i : 0, GS_WAVE);
            q[u].clear();
            if (i < n_live && 4 * sub < row_len) q[u].load(t, (row0 + from[u]) * row_len + 4 * sub);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long long i = (row0 + from[u]) * row_len + 4 * sub;
            const uint32_t old_x = STATE8 ? (uint32_t)__shfl(x, from[u], GS_WAVE) : 0u;
            const float dm = any_late ? __shfl(decay_m, from[u], GS_WAVE) : 1.f, dv = any_late ? __shfl(decay_v, from[u], GS_WAVE) : 1.f;
            f32x4 p;
            const uint32_t new_x = q[u].template step<GROUP>(p, old_x, dm, dv, i, scale, k);
            if (at + 4 * u + lane / GROUP < n_live && 4 * sub < row_len) {
                q[u].store(t, i, p);
                if (STATE8 && sub == 0) *(uint16_t *)(t.exponents + 2 * (row0 + from[u])) = (uint16_t)new_x;
            }
        }
    }
}

// Float rows of L elements, four rows (L quads) a lane: every access is 16 bytes (4 for codes, 8 for exponents) although a row
// is not.  Of rows under a mask the lane writes back what it read.
template <int L, bool STATE8>
__device__ __forceinline__ void step_narrow(const AdamwTensor &t, const AdamwScalars &k, float scale, unsigned chunk) {
    const long long rows = t.numel / L, row0 = 4 * ((long long)chunk * GS_BLOCK + threadIdx.x);
    if (row0 >= rows) return;
    if (row0 + 4 > rows) {
        for (long long r = row0; r < rows; ++r) step_unit<1, GS_DTYPE_F32, false, STATE8>(t, k, scale, r, L);
        return;
    }
    bool live[4] = {true, true, true, true};
    float decay_m[4] = {1.f, 1.f, 1.f, 1.f}, decay_v[4] = {1.f, 1.f, 1.f, 1.f};
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    if (t.masked) {
        const uint32_t mask = *(const uint32_t *)((const int8_t *)t.master_or_mask + row0);
        i32x4 last = *(const i32x4 *)(t.last_step + row0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            live[r] = (mask >> (8 * r) & 255u) == 0u;
            if (live[r]) {
                row_decay(k, last[r], decay_m[r], decay_v[r]);
                last[r] = k.step;
            }
        }
        if (!(live[0] || live[1] || live[2] || live[3])) return;
        *(i32x4 *)(t.last_step + row0) = last;
    }
    const long long base = row0 * L;
    Quad<GS_DTYPE_F32, false, STATE8> q[L];
    u16x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < L; ++c) q[c].load(t, base + 4 * c);
    if (STATE8) x = *(const u16x4 *)(t.exponents + 2 * row0);
    f32x4 p[L];
    float m[4 * L], v[4 * L];
#pragma unroll
    for (int e = 0; e < 4 * L; ++e) {
        const int r = e / L, c = e / 4, j = e % 4;
        if (STATE8) {
            m[e] = decode_m((q[c].mc >> (8 * j)) & 255u, exponent_scale(x[r] & 255, 9, -8));
            v[e] = decode_v((q[c].vc >> (8 * j)) & 255u, exponent_scale(x[r] >> 8, 32, -31));
        } else {
            m[e] = q[c].m[j];
            v[e] = q[c].v[j];
        }
        const float old_p = q[c].p[j], old_m = m[e], old_v = v[e];
        m[e] *= decay_m[r];
        v[e] *= decay_v[r];
        p[c][j] = update_one<STATE8, false>(old_p, scaled(q[c].g[j], scale), m[e], v[e], k);
        if (!live[r]) {
            p[c][j] = old_p;
            m[e] = old_m;
            v[e] = old_v;
        }
    }
    if (STATE8) {
        uint32_t hash[L];
#pragma unroll
        for (int c = 0; c < L; ++c) hash[c] = mix32((uint32_t)((base + 4 * c) >> 2) ^ k.key);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
            for (int e = r * L; e < r * L + L; ++e) {
                top_m = max(top_m, to_bits(m[e]) & 0x7FFFFFFFu);
                top_v = max(top_v, to_bits(v[e]) & 0x7FFFFFFFu);
            }
            const int xm = block_exponent(top_m, 0x1FFFFFu, 9), xv = block_exponent(top_v, 0x0FFFFFu, 32);
            if (live[r]) x[r] = (uint16_t)(xm | xv << 8);
#pragma unroll
            for (int e = r * L; e < r * L + L; ++e) {
                const int c = e / 4, j = e % 4;
                const uint32_t bits = element_bits(hash[c], j), keep = ~(255u << (8 * j));
                const uint32_t mc = (q[c].mc & keep) | encode_m(m[e], xm, bits) << (8 * j), vc = (q[c].vc & keep) | encode_v(v[e], xv, bits) << (8 * j);
                q[c].mc = live[r] ? mc : q[c].mc;
                q[c].vc = live[r] ? vc : q[c].vc;
            }
        }
        *(u16x4 *)(t.exponents + 2 * row0) = x;
    }
#pragma unroll
    for (int c = 0; c < L; ++c) {
        if (!STATE8) {
            q[c].m = f32x4{m[4 * c], m[4 * c + 1], m[4 * c + 2], m[4 * c + 3]};
            q[c].v = f32x4{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
        }
        q[c].store(t, base + 4 * c, p[c]);
    }
}

// Chunks that a form makes of a tensor (a workgroup each)
__host__ __device__ inline long long form_chunks(int form, long long numel, int row_len, int unroll) {
    const long long units = row_len > 0 ? numel / row_len : (numel + UNIT - 1) / UNIT;
    const int group = row_len == 0 || row_len > 16 ? 16 : (row_len > 4 ? 4 : 1);
    const int per = form == FOURS ? GS_BLOCK / 16 * unroll : form == FOURS_MASKED ? GS_BLOCK : form == NARROW ? 4 * GS_BLOCK : GS_BLOCK / group;
    return (units + per - 1) / per;
}

// All tensors of one parameter type and one form of moments, whatever their shapes: the branches on `form` are uniform in a
// workgroup, and one launch costs less than the idle lanes' registers.
template <int UNROLL, int DT, bool MASTER, bool STATE8>
__global__ __launch_bounds__(GS_BLOCK) void adamw_kernel(AdamwBatch b) {
    const int ti = find_tensor<MAX_TENSORS>(b.first_chunk, b.n_tensors, blockIdx.x);
    const AdamwTensor &t = b.t[ti];
    AdamwScalars k = b.device_scalars ? b.device_scalars[ti] : b.scalars[t.set];
    if (!b.device_scalars) k.key = t.key;
    const float scale = b.grad_scale ? *b.grad_scale : 1.f;
    const unsigned chunk = blockIdx.x - b.first_chunk[ti];
    if (t.form == FOURS) return step_fours<UNROLL, DT, MASTER, STATE8>(t, k, scale, chunk);
    if constexpr (DT == GS_DTYPE_F32) {
        if (t.form == FOURS_MASKED) return step_fours_masked<UNROLL, STATE8>(t, k, scale, chunk);
        if (t.form == NARROW) {
            if (t.row_len == 3) return step_narrow<3, STATE8>(t, k, scale, chunk);
            if (t.row_len == 1) return step_narrow<1, STATE8>(t, k, scale, chunk);
            if (t.row_len == 2) return step_narrow<2, STATE8>(t, k, scale, chunk);
            return step_narrow<4, STATE8>(t, k, scale, chunk);
        }
    }
    const int row_len = t.row_len > 0 ? t.row_len : UNIT;
    if (row_len > 16) step_unit<16, DT, MASTER, STATE8>(t, k, scale, (long long)chunk * (GS_BLOCK / 16) + threadIdx.x / 16, row_len);
    else if (row_len > 4) step_unit<4, DT, MASTER, STATE8>(t, k, scale, (long long)chunk * (GS_BLOCK / 4) + threadIdx.x / 4, row_len);
    else step_unit<1, DT, MASTER, STATE8>(t, k, scale, (long long)chunk * GS_BLOCK + threadIdx.x, row_len);
}

// Scalars of tensors whose step count or learning rate lives on the device.  1 - beta^t is taken as -expm1(t log beta) in
// double precision: for beta2 = 0.999 and t = 1 the difference of two floats would keep three digits.
struct PrepareArgs {
    int n;
    uint32_t seed;
    struct { const long long *step; const float *lr; double lr_host, beta1, beta2, eps, weight_decay; long long step_host; uint32_t tensor; } t[MAX_TENSORS];   // 72 bytes each
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
    int row_len, form;
};
struct MomentsBatch {
    int n_tensors;
    unsigned first_chunk[MAX_TENSORS + 1];
    MomentsTensor t[MAX_TENSORS];
};
static_assert(sizeof(MomentsBatch) <= 4000, "kernel arguments");

template <int GROUP, int DT>
__device__ __forceinline__ void read_unit(const MomentsTensor &t, long long unit, int unit_len) {
    const long long base = unit * unit_len, left = t.numel - base;
    const int len = left <= 0 ? 0 : (left < unit_len ? (int)left : unit_len);
    if (len == 0) return;
    const float scale_m = exponent_scale(t.exponents[2 * unit], 9, -8), scale_v = exponent_scale(t.exponents[2 * unit + 1], 32, -31);
    for (int e = threadIdx.x % GROUP; e < len; e += GROUP) {
        store_one<DT>(t.m_out, base + e, decode_m(t.m[base + e], scale_m));
        store_one<DT>(t.v_out, base + e, decode_v(t.v[base + e], scale_v));
    }
}

template <int UNROLL, int DT>
__device__ __forceinline__ void read_fours(const MomentsTensor &t, unsigned chunk) {
    constexpr int GROUP = 16, PER_PASS = GS_BLOCK / GROUP;
    const int unit_len = t.row_len > 0 ? t.row_len : UNIT;
    const long long chunk_unit = (long long)chunk * (PER_PASS * UNROLL), unit0 = chunk_unit + threadIdx.x / GROUP;
    const long long whole = t.numel / unit_len;
    const int sub = threadIdx.x % GROUP;
    uint32_t mc[UNROLL], vc[UNROLL], x[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long unit = unit0 + u * PER_PASS;
        mc[u] = vc[u] = x[u] = 0u;
        if (unit < whole && 4 * sub < unit_len) {
            mc[u] = *(const uint32_t *)(t.m + unit * unit_len + 4 * sub);
            vc[u] = *(const uint32_t *)(t.v + unit * unit_len + 4 * sub);
            x[u] = *(const uint16_t *)(t.exponents + 2 * unit);
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const long long unit = unit0 + u * PER_PASS;
        f32x4 m, v;
        decode_four(mc[u], vc[u], x[u], m, v);
        if (unit < whole && 4 * sub < unit_len) {
            store_four<DT>(t.m_out, unit * unit_len + 4 * sub, m);
            store_four<DT>(t.v_out, unit * unit_len + 4 * sub, v);
        }
    }
    if (whole * unit_len < t.numel && whole >= chunk_unit && whole < chunk_unit + PER_PASS * UNROLL && threadIdx.x < GROUP)
        read_unit<GROUP, DT>(t, whole, unit_len);
}

template <int L, int DT>
__device__ __forceinline__ void read_narrow(const MomentsTensor &t, unsigned chunk) {
    const long long rows = t.numel / L, row0 = 4 * ((long long)chunk * GS_BLOCK + threadIdx.x);
    if (row0 >= rows) return;
    if (row0 + 4 > rows) {
        for (long long r = row0; r < rows; ++r) read_unit<1, DT>(t, r, L);
        return;
    }
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    const u16x4 x = *(const u16x4 *)(t.exponents + 2 * row0);
#pragma unroll
    for (int c = 0; c < L; ++c) {
        const uint32_t mc = *(const uint32_t *)(t.m + row0 * L + 4 * c), vc = *(const uint32_t *)(t.v + row0 * L + 4 * c);
        f32x4 m, v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = (4 * c + j) / L;
            m[j] = decode_m((mc >> (8 * j)) & 255u, exponent_scale(x[r] & 255, 9, -8));
            v[j] = decode_v((vc >> (8 * j)) & 255u, exponent_scale(x[r] >> 8, 32, -31));
        }
        store_four<DT>(t.m_out, row0 * L + 4 * c, m);
        store_four<DT>(t.v_out, row0 * L + 4 * c, v);
    }
}

template <int UNROLL, int DT>
__global__ __launch_bounds__(GS_BLOCK) void read_moments_kernel(MomentsBatch b) {
    const int ti = find_tensor<MAX_TENSORS>(b.first_chunk, b.n_tensors, blockIdx.x);
    const MomentsTensor &t = b.t[ti];
    const unsigned chunk = blockIdx.x - b.first_chunk[ti];
    if (t.form == FOURS) return read_fours<UNROLL, DT>(t, chunk);
    if (t.form == NARROW) {
        if (t.row_len == 3) return read_narrow<3, DT>(t, chunk);
        if (t.row_len == 1) return read_narrow<1, DT>(t, chunk);
        if (t.row_len == 2) return read_narrow<2, DT>(t, chunk);
        return read_narrow<4, DT>(t, chunk);
    }
    const int row_len = t.row_len > 0 ? t.row_len : UNIT;
    if (row_len > 16) read_unit<16, DT>(t, (long long)chunk * (GS_BLOCK / 16) + threadIdx.x / 16, row_len);
    else if (row_len > 4) read_unit<4, DT>(t, (long long)chunk * (GS_BLOCK / 4) + threadIdx.x / 4, row_len);
    else read_unit<1, DT>(t, (long long)chunk * GS_BLOCK + threadIdx.x, row_len);
}

// ------------------------------------------------------------------ norm of gradients
// First pass: each workgroup adds the squares of one chunk in double precision (a float's square is exact there, so the
// result does not depend on the order to within 1e-16) and leaves a partial sum; the second adds the partial sums in a
// fixed order.
struct NormTensor {
    const void *grad;
    u64 numel_type;             // numel * 4 + type
};
struct NormBatch {              // tensors without a row mask
    int n_tensors;
    unsigned chunk;             // elements, a multiple of 1024
    unsigned first_block[MAX_NORM_TENSORS + 1];
    int id[MAX_NORM_TENSORS];   // place in the caller's list
    NormTensor t[MAX_NORM_TENSORS];
};
struct NormMaskedTensor {
    const void *grad;
    const int8_t *row_mask;
    long long numel;
    int row_len, dtype;
};
struct NormMaskedBatch {
    int n_tensors;
    unsigned chunk;
    unsigned first_block[MAX_NORM_MASKED + 1];
    int id[MAX_NORM_MASKED];
    NormMaskedTensor t[MAX_NORM_MASKED];
};
static_assert(sizeof(NormBatch) <= 4000 && sizeof(NormMaskedBatch) <= 4000, "kernel arguments");

// Rows of a masked tensor that a workgroup of the first pass takes: at least a chunk's elements, so that there are no more
// parts than without a mask; whole waves' worth of rows
__host__ __device__ __forceinline__ long long norm_rows(long long chunk, int row_len) {
    return ((chunk + row_len - 1) / row_len + 63) / 64 * 64;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, GS_WAVE);
    return x;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double red[THREADS / GS_WAVE];
    x = wave_sum(x);
    if (gs_lane() == 0) red[threadIdx.x / GS_WAVE] = x;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < THREADS / GS_WAVE; ++i) s += red[i];
    return s;
}

template <int N, typename V>
__device__ __forceinline__ double add_squares(double s, V x) {
#pragma unroll
    for (int j = 0; j < N; ++j) s = fma((double)(float)x[j], (double)(float)x[j], s);
    return s;
}

// Elements begin..end (begin is a multiple of 1024: the chunk is aligned where the tensor is): 16 bytes a lane, four requests
// in flight.
template <int DT>
__device__ __forceinline__ double flat_squares(const void *grad, long long begin, long long end) {
    typedef typename Wide<DT>::type V;
    constexpr int N = 16 / (DT == GS_DTYPE_F32 ? 4 : 2), AHEAD = 4;
    double s = 0.0;
    const long long wide = ((uintptr_t)grad & 15) == 0 ? (end - begin) / N : 0;
    const V *g = (const V *)((const char *)grad + begin * (16 / N));
    long long q = threadIdx.x;
    for (; q + (AHEAD - 1) * GS_BLOCK < wide; q += AHEAD * GS_BLOCK) {
        V x[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) x[a] = g[q + a * GS_BLOCK];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) s = add_squares<N>(s, x[a]);
    }
    for (; q < wide; q += GS_BLOCK) s = add_squares<N>(s, g[q]);
    for (long long i = begin + N * wide + threadIdx.x; i < end; i += GS_BLOCK) {
        const double x = (double)load_one<DT>(grad, i);
        s = fma(x, x, s);
    }
    return s;
}

// Rows begin..end of a tensor with a row mask, element by element, GROUP lanes a row
template <int GROUP, int DT>
__device__ __forceinline__ double row_squares(const NormMaskedTensor &t, long long begin, long long end) {
    const int sub = threadIdx.x % GROUP, len = t.row_len;
    double s = 0.0;
    for (long long row = begin + threadIdx.x / GROUP; row < end; row += GS_BLOCK / GROUP) {
        if (t.row_mask[row] != 0) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (sub + j * GROUP < len) {
                const double y = (double)load_one<DT>(t.grad, row * len + sub + j * GROUP);
                s = fma(y, y, s);
            }
    }
    return s;
}

// The same rows with aligned quads, rows of 20 to 64 elements: a wave packs the live ones of 64 rows and reads them four at a
// time, AHEAD of them in flight.
template <int DT>
__device__ __forceinline__ double packed_row_squares(const NormMaskedTensor &t, long long begin, long long end) {
    constexpr int GROUP = 16, AHEAD = 4, BYTES = DT == GS_DTYPE_F32 ? 4 : 2;
    const int len = t.row_len, lane = gs_lane(), sub = lane % GROUP;
    double s = 0.0;
    for (long long row0 = begin + threadIdx.x / GS_WAVE * GS_WAVE; row0 < end; row0 += GS_BLOCK) {
        const bool live = row0 + lane < end && t.row_mask[row0 + lane < end ? row0 + lane : row0] == 0;
        const u64 lives = __ballot(live), below = (1ull << lane) - 1ull;
        const int n_live = __popcll(lives);
        const int order = __builtin_amdgcn_ds_permute(4 * (live ? __popcll(lives & below) : 63 - __popcll(~lives & below)), lane);
        for (int at = 0; at < n_live; at += 4 * AHEAD) {
            typename Four<DT>::type x[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int i = at + 4 * a + lane / GROUP;
                const long long row = row0 + __shfl(order, i < n_live ? i : 0, GS_WAVE);
                x[a] = {};
                if (i < n_live && 4 * sub < len) x[a] = *(const decltype(+x[a]) *)((const char *)t.grad + (row * len + 4 * sub) * BYTES);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) s = add_squares<4>(s, x[a]);
        }
    }
    return s;
}

// Float rows of up to four elements: a lane takes four rows in L quads.
template <int L>
__device__ __forceinline__ double narrow_squares(const NormMaskedTensor &t, long long begin, long long end) {
    double s = 0.0;
    const float *grad = (const float *)t.grad;
    // (begin is a multiple of four rows)
    for (long long row0 = begin + 4 * threadIdx.x; row0 < end; row0 += 4 * GS_BLOCK) {
        if (row0 + 4 > end) {
            for (long long r = row0; r < end; ++r)
                for (int j = 0; j < L && t.row_mask[r] == 0; ++j) s = fma((double)grad[r * L + j], (double)grad[r * L + j], s);
            break;
        }
        const uint32_t mask = *(const uint32_t *)(t.row_mask + row0);
        f32x4 x[L];
#pragma unroll
        for (int c = 0; c < L; ++c) x[c] = *(const f32x4 *)(grad + row0 * L + 4 * c);
#pragma unroll
        for (int e = 0; e < 4 * L; ++e)
            if ((mask >> (8 * (e / L)) & 255u) == 0u) s = fma((double)x[e / 4][e % 4], (double)x[e / 4][e % 4], s);
    }
    return s;
}

template <int DT>
__device__ __forceinline__ double masked_squares(const NormMaskedTensor &t, unsigned part, unsigned chunk) {
    const long long rows = t.numel / t.row_len, per = norm_rows(chunk, t.row_len);
    const long long begin = part * per, end = min(rows, begin + per);
    const bool aligned = ((uintptr_t)t.grad & (DT == GS_DTYPE_F32 ? 15 : 7)) == 0;
    if (t.row_len > 16) return aligned && t.row_len % 4 == 0 ? packed_row_squares<DT>(t, begin, end) : row_squares<16, DT>(t, begin, end);
    if (t.row_len > 4) return row_squares<4, DT>(t, begin, end);
    if constexpr (DT == GS_DTYPE_F32)
        if (aligned && ((uintptr_t)t.row_mask & 3) == 0) {
            if (t.row_len == 3) return narrow_squares<3>(t, begin, end);
            if (t.row_len == 1) return narrow_squares<1>(t, begin, end);
            if (t.row_len == 2) return narrow_squares<2>(t, begin, end);
            return narrow_squares<4>(t, begin, end);
        }
    return row_squares<1, DT>(t, begin, end);
}

// A workgroup's sum goes behind those of the launches before (`base` of them); spans[i] = {first, number} of tensor i's.
__device__ __forceinline__ void leave_partial(double s, unsigned base, unsigned part, unsigned parts, int id, double *partials, uint2 *spans) {
    s = block_sum<GS_BLOCK>(s);
    if (threadIdx.x == 0) {
        partials[base + blockIdx.x] = s;
        if (part == 0 && spans) spans[id] = make_uint2(base + blockIdx.x, parts);
    }
}

__global__ __launch_bounds__(GS_BLOCK) void norm_partial_kernel(NormBatch b, unsigned base, double *__restrict__ partials, uint2 *__restrict__ spans) {
    const int ti = find_tensor<MAX_NORM_TENSORS>(b.first_block, b.n_tensors, blockIdx.x);
    const unsigned part = blockIdx.x - b.first_block[ti];
    const void *grad = b.t[ti].grad;
    const long long numel = (long long)(b.t[ti].numel_type >> 2), begin = (long long)part * b.chunk;
    const long long end = min(numel, begin + (long long)b.chunk);
    const int type = (int)(b.t[ti].numel_type & 3);
    double s;
    if (type == GS_DTYPE_F32) s = flat_squares<GS_DTYPE_F32>(grad, begin, end);
    else if (type == GS_DTYPE_BF16) s = flat_squares<GS_DTYPE_BF16>(grad, begin, end);
    else s = flat_squares<GS_DTYPE_F16>(grad, begin, end);
    leave_partial(s, base, part, b.first_block[ti + 1] - b.first_block[ti], b.id[ti], partials, spans);
}

__global__ __launch_bounds__(GS_BLOCK) void norm_masked_kernel(NormMaskedBatch b, unsigned base, double *__restrict__ partials, uint2 *__restrict__ spans) {
    const int ti = find_tensor<MAX_NORM_MASKED>(b.first_block, b.n_tensors, blockIdx.x);
    const unsigned part = blockIdx.x - b.first_block[ti];
    const NormMaskedTensor &t = b.t[ti];
    double s;
    if (t.dtype == GS_DTYPE_F32) s = masked_squares<GS_DTYPE_F32>(t, part, b.chunk);
    else if (t.dtype == GS_DTYPE_BF16) s = masked_squares<GS_DTYPE_BF16>(t, part, b.chunk);
    else s = masked_squares<GS_DTYPE_F16>(t, part, b.chunk);
    leave_partial(s, base, part, b.first_block[ti + 1] - b.first_block[ti], b.id[ti], partials, spans);
}

__device__ __forceinline__ float clip_of(double sq_sum, double max_norm) {
    if (max_norm <= 0.0) return 1.f;
    const double c = max_norm / (sqrt(sq_sum) + 1e-6);
    return c > 1.0 ? 1.f : (float)c;        // (a norm that is NaN stays visible: the comparison fails)
}

// Block 0 adds up all partial sums; the waves of the others take a tensor each.
constexpr int FINISH_THREADS = 1024;
__global__ __launch_bounds__(FINISH_THREADS) void norm_finish_kernel(const double *__restrict__ partials, const uint2 *__restrict__ spans,
                                                                     unsigned n_partials, int n_tensors, double max_norm, double *sq_sum,
                                                                     float *norm, float *clip, float *each) {
    if (blockIdx.x > 0) {
        const int i = (int)(blockIdx.x - 1) * (FINISH_THREADS / GS_WAVE) + threadIdx.x / GS_WAVE;
        if (i >= n_tensors) return;
        const uint2 span = spans[i];
        double s = 0.0;
        for (unsigned j = gs_lane(); j < span.y; j += GS_WAVE) s += partials[span.x + j];
        s = wave_sum(s);
        if (gs_lane() == 0) each[i] = (float)sqrt(s);
        return;
    }
    double s = 0.0;
    for (unsigned j = threadIdx.x; j < n_partials; j += FINISH_THREADS) s += partials[j];
    s = block_sum<FINISH_THREADS>(s);
    if (threadIdx.x != 0) return;
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

// whether a written range meets any other
bool ranges_meet(Range *r, size_t n) {
    std::sort(r, r + n, [](const Range &a, const Range &b) { return a.begin < b.begin; });
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
bool aligned_to(u64 p, u64 bytes) { return p % bytes == 0; }
u64 entry(const uint64_t *column, int i) { return column ? column[i] : 0; }

// Small totals get small shares, so that they still reach every compute unit: 2048 workgroups are eight for each.
constexpr int UNROLL = 4;
constexpr long long SMALL_CHUNKS = 2048;

template <int U>
void launch_step(int dtype, bool master, bool state8, const AdamwBatch &b, hipStream_t s) {
    const dim3 grid(b.first_chunk[b.n_tensors]), block(GS_BLOCK);
#define GS_ADAMW_LAUNCH(DT, MASTER)                                                                                        \
    do {                                                                                                                   \
        if (state8) hipLaunchKernelGGL((adamw_kernel<U, DT, MASTER, true>), grid, block, 0, s, b);                         \
        else hipLaunchKernelGGL((adamw_kernel<U, DT, MASTER, false>), grid, block, 0, s, b);                               \
    } while (0)
    if (dtype == GS_DTYPE_F32) GS_ADAMW_LAUNCH(GS_DTYPE_F32, false);
    else if (dtype == GS_DTYPE_BF16 && master) GS_ADAMW_LAUNCH(GS_DTYPE_BF16, true);
    else if (dtype == GS_DTYPE_BF16) GS_ADAMW_LAUNCH(GS_DTYPE_BF16, false);
    else if (master) GS_ADAMW_LAUNCH(GS_DTYPE_F16, true);
    else GS_ADAMW_LAUNCH(GS_DTYPE_F16, false);
#undef GS_ADAMW_LAUNCH
}

template <int U>
void launch_moments(int dtype, const MomentsBatch &b, hipStream_t s) {
    const dim3 grid(b.first_chunk[b.n_tensors]), block(GS_BLOCK);
    if (dtype == GS_DTYPE_F32) hipLaunchKernelGGL((read_moments_kernel<U, GS_DTYPE_F32>), grid, block, 0, s, b);
    else hipLaunchKernelGGL((read_moments_kernel<U, GS_DTYPE_BF16>), grid, block, 0, s, b);
}

int launch_status(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    gs_set_error("%s: kernel launch failed: %s", what, hipGetErrorString(e));
    return -3;
}

// A batch is launched when its table is full; its tensors keep the caller's order.
struct StepBatch {
    AdamwBatch b;
    PrepareArgs prep;
    const double *hyper[MAX_SETS];      // of the sets in b.scalars, with their steps
    long long step[MAX_SETS];
    int n_sets;
    void clear() { b.n_tensors = n_sets = 0; b.first_chunk[0] = 0; }
};

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
    const bool on_device = host_step_device || host_lr_device, state8 = host_exponents != nullptr;
    GS_REQUIRE(!on_device || (workspace && aligned_to((u64)(uintptr_t)workspace, 4)),
               "gs_adamw_step: a step count or learning rate on the device needs the workspace");
    long long units_of_16 = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const long long n = host_numel[i];
        const int row = host_row_len[i], dt = host_dtype[i];
        const double *h = host_hyper + 5 * (size_t)i;
        GS_REQUIRE(n >= 0 && n < (1LL << 46) && row >= 0 && row <= UNIT && (row == 0 || n % row == 0),
                   "gs_adamw_step: numel in [0, 2^46), too large else, rows of 1..64 elements");
        GS_REQUIRE(dt == GS_DTYPE_F32 || dt == GS_DTYPE_BF16 || dt == GS_DTYPE_F16, "gs_adamw_step: unknown dtype");
        GS_REQUIRE(form_chunks(ELEMENTS, n, row, 1) < 0x7fffffffLL, "gs_adamw_step: tensor too large");
        GS_REQUIRE(n == 0 || (host_param[i] && host_grad[i] && host_exp_avg[i] && host_exp_avg_sq[i] && (!state8 || host_exponents[i])),
                   "gs_adamw_step: null tensor");
        GS_REQUIRE(!entry(host_row_mask, i) || (row > 0 && dt == GS_DTYPE_F32 && host_last_step[i]), "gs_adamw_step: a row mask needs float rows and last steps");
        GS_REQUIRE(!entry(host_master, i) || dt != GS_DTYPE_F32, "gs_adamw_step: a master copy belongs to a 16-bit parameter");
        GS_REQUIRE((host_step[i] >= 1 && host_step[i] < 0x7fffffffLL) || entry(host_step_device, i), "gs_adamw_step: step >= 1");
        GS_REQUIRE(h[1] >= 0.0 && h[1] < 1.0 && h[2] >= 0.0 && h[2] < 1.0 && h[3] >= 0.0, "gs_adamw_step: betas in [0, 1), eps >= 0");
        GS_REQUIRE(aligned_to(host_param[i] | host_grad[i], element_bytes(dt)) && aligned_to(state8 ? 0 : host_exp_avg[i] | host_exp_avg_sq[i], 4) &&
                       aligned_to(entry(host_master, i) | (entry(host_row_mask, i) ? host_last_step[i] : 0), 4),
                   "gs_adamw_step: an address is no multiple of its type's size");
        units_of_16 += form_chunks(FOURS, n, row, 1);
    }
    {
        Range *r = (Range *)malloc((size_t)n_tensors * 7 * sizeof(Range));
        GS_REQUIRE(r != nullptr, "gs_adamw_step: out of host memory");
        size_t k = 0;
        for (int i = 0; i < n_tensors; ++i) {
            const int row = host_row_len[i];
            const u64 n = (u64)host_numel[i], pe = n * element_bytes(host_dtype[i]), se = n * (state8 ? 1 : 4), blocks = row > 0 ? n / row : (n + UNIT - 1) / UNIT;
            r[k++] = {host_param[i], host_param[i] + pe, 1};
            r[k++] = {host_grad[i], host_grad[i] + pe, 0};
            r[k++] = {host_exp_avg[i], host_exp_avg[i] + se, 1};
            r[k++] = {host_exp_avg_sq[i], host_exp_avg_sq[i] + se, 1};
            if (state8) r[k++] = {host_exponents[i], host_exponents[i] + 2 * blocks, 1};
            if (entry(host_master, i)) r[k++] = {host_master[i], host_master[i] + 4 * n, 1};
            if (entry(host_row_mask, i)) r[k++] = {host_last_step[i], host_last_step[i] + 4 * blocks, 1};
        }
        const bool meet = ranges_meet(r, k);
        free(r);
        GS_REQUIRE(!meet, "gs_adamw_step: buffers overlap");
    }
    hipStream_t s = (hipStream_t)stream;
    AdamwScalars *device_scalars = (AdamwScalars *)workspace;
    const int unroll = units_of_16 <= SMALL_CHUNKS ? 1 : UNROLL;
    StepBatch q;
    q.b.grad_scale = grad_scale;
    // one type after the other: (parameter type, master copy)
    for (int kind = 0; kind < 6; ++kind) {
        const int dtype = kind / 2;
        const bool master = kind % 2 != 0;
        q.clear();
        for (int i = 0; i <= n_tensors; ++i) {
            const bool end = i == n_tensors;
            if (!end && (host_numel[i] == 0 || host_dtype[i] != dtype || (entry(host_master, i) != 0) != master)) continue;
            AdamwTensor t = {};
            long long chunks = 0;
            int set = 0;
            if (!end) {
                const u64 mask = entry(host_row_mask, i);
                const int row = mask || state8 ? host_row_len[i] : 0;      // (moments in 32 bits without a mask: units of 64 whatever the shape)
                const bool fours = aligned_to(host_param[i] | host_grad[i], 4 * element_bytes(dtype)) &&
                                   aligned_to(host_exp_avg[i] | host_exp_avg_sq[i], state8 ? 4 : 16) &&
                                   aligned_to(master ? host_master[i] : 0, 16) && aligned_to(state8 ? host_exponents[i] : 0, 2);
                const bool narrow = fours && dtype == GS_DTYPE_F32 && aligned_to(state8 ? host_exponents[i] : 0, 8) && aligned_to(mask, 4) &&
                                    aligned_to(mask ? host_last_step[i] : 0, 16);
                t.form = row >= 1 && row <= 4 && narrow ? NARROW : fours && (row == 0 || (row > 16 && row % 4 == 0)) ? (mask ? FOURS_MASKED : FOURS) : ELEMENTS;
                t.row_len = (uint8_t)row;
                t.masked = mask != 0;
                chunks = form_chunks(t.form, host_numel[i], row, unroll);
                while (!on_device && set < q.n_sets &&
                       (q.step[set] != host_step[i] || memcmp(q.hyper[set], host_hyper + 5 * (size_t)i, 5 * sizeof(double)) != 0)) ++set;
            }
            if (q.b.n_tensors > 0 && (end || q.b.n_tensors == MAX_TENSORS || set == MAX_SETS ||
                                      (long long)q.b.first_chunk[q.b.n_tensors] + chunks >= 0x7fffffffLL)) {
                q.b.device_scalars = on_device ? device_scalars : nullptr;
                if (on_device) {
                    q.prep.n = q.b.n_tensors;
                    q.prep.seed = seed;
                    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(GS_WAVE), 0, s, q.prep, device_scalars);
                    device_scalars += q.b.n_tensors;      // (every batch has its own part: n_tensors in all)
                }
                if (unroll == 1) launch_step<1>(dtype, master, state8, q.b, s);
                else launch_step<UNROLL>(dtype, master, state8, q.b, s);
                if (const int status = launch_status("gs_adamw_step")) return status;
                q.clear();
                set = 0;
            }
            if (end) break;
            const double *h = host_hyper + 5 * (size_t)i;
            const uint32_t id = (uint32_t)host_tensor_id[i];
            const int at = q.b.n_tensors++;
            if (on_device) {
                q.prep.t[at] = {(const long long *)entry(host_step_device, i), (const float *)entry(host_lr_device, i), h[0], h[1], h[2], h[3], h[4], host_step[i], id};
            } else {
                if (set == q.n_sets) {
                    q.hyper[set] = h;
                    q.step[set] = host_step[i];
                    q.b.scalars[q.n_sets++] = adamw_scalars(h[0], h[1], h[2], h[3], h[4], host_step[i], seed, id);
                }
                t.key = tensor_key(seed, id, (uint32_t)host_step[i]);
            }
            t.set = (uint8_t)set;
            t.param = (void *)host_param[i];
            t.grad = (const void *)host_grad[i];
            t.exp_avg = (void *)host_exp_avg[i];
            t.exp_avg_sq = (void *)host_exp_avg_sq[i];
            t.exponents = (uint8_t *)entry(host_exponents, i);
            t.master_or_mask = (void *)(master ? host_master[i] : entry(host_row_mask, i));
            t.last_step = (int32_t *)entry(host_last_step, i);
            t.numel = host_numel[i];
            q.b.t[at] = t;
            q.b.first_chunk[at + 1] = q.b.first_chunk[at] + (unsigned)chunks;
        }
    }
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
    long long units_of_16 = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const long long n = host_numel[i];
        const int row = host_row_len[i];
        GS_REQUIRE(n >= 0 && n < (1LL << 46) && row >= 0 && row <= UNIT && (row == 0 || n % row == 0),
                   "gs_read_moments: numel in [0, 2^46), rows of 1..64 elements");
        GS_REQUIRE(form_chunks(ELEMENTS, n, row, 1) < 0x7fffffffLL, "gs_read_moments: tensor too large");
        GS_REQUIRE(n == 0 || (host_exp_avg[i] && host_exp_avg_sq[i] && host_exponents[i] && host_m_out[i] && host_v_out[i]),
                   "gs_read_moments: null tensor");
        GS_REQUIRE(aligned_to(host_m_out[i] | host_v_out[i], element_bytes(out_dtype)), "gs_read_moments: misaligned output");
        units_of_16 += form_chunks(FOURS, n, row, 1);
    }
    const int unroll = units_of_16 <= SMALL_CHUNKS ? 1 : UNROLL;
    MomentsBatch b;
    b.n_tensors = 0;
    b.first_chunk[0] = 0;
    for (int i = 0; i <= n_tensors; ++i) {
        const bool end = i == n_tensors;
        if (!end && host_numel[i] == 0) continue;
        MomentsTensor t = {};
        long long chunks = 0;
        if (!end) {
            const int row = host_row_len[i];
            const bool fours = aligned_to(host_exp_avg[i] | host_exp_avg_sq[i], 4) && aligned_to(host_m_out[i] | host_v_out[i], 4 * element_bytes(out_dtype)) &&
                               aligned_to(host_exponents[i], 2);
            t = {(const uint8_t *)host_exp_avg[i], (const uint8_t *)host_exp_avg_sq[i], (const uint8_t *)host_exponents[i],
                 (void *)host_m_out[i], (void *)host_v_out[i], host_numel[i], row, 0};
            t.form = row >= 1 && row <= 4 && fours && aligned_to(host_exponents[i], 8) ? NARROW : fours && (row == 0 || (row > 16 && row % 4 == 0)) ? FOURS : ELEMENTS;
            chunks = form_chunks(t.form, host_numel[i], row, unroll);
        }
        if (b.n_tensors > 0 && (end || b.n_tensors == MAX_TENSORS || (long long)b.first_chunk[b.n_tensors] + chunks >= 0x7fffffffLL)) {
            if (unroll == 1) launch_moments<1>(out_dtype, b, (hipStream_t)stream);
            else launch_moments<UNROLL>(out_dtype, b, (hipStream_t)stream);
            if (const int status = launch_status("gs_read_moments")) return status;
            b.n_tensors = 0;
        }
        if (end) break;
        b.t[b.n_tensors] = t;
        b.first_chunk[b.n_tensors + 1] = b.first_chunk[b.n_tensors] + (unsigned)chunks;
        ++b.n_tensors;
    }
    return 0;
}

extern "C" long long gs_grad_norm_workspace_bytes(int n_tensors) {
    return n_tensors < 0 ? 0 : ((long long)NORM_PARTIALS + 2LL * n_tensors) * 8;
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
        GS_REQUIRE(n >= 0 && n < (1LL << 46), "gs_grad_norm: numel in [0, 2^46)");
        GS_REQUIRE(dt == GS_DTYPE_F32 || dt == GS_DTYPE_BF16 || dt == GS_DTYPE_F16, "gs_grad_norm: unknown dtype");
        GS_REQUIRE(n == 0 || (host_grad[i] && aligned_to(host_grad[i], element_bytes(dt))), "gs_grad_norm: null or misaligned tensor");
        GS_REQUIRE(!entry(host_row_mask, i) || (host_row_len[i] > 0 && host_row_len[i] <= UNIT && n % host_row_len[i] == 0), "gs_grad_norm: a row mask needs rows");
        total += n;
    }
    // chunks of a multiple of 1024 elements, so that there are at most NORM_PARTIALS of them and one more for each tensor
    long long chunk = (total + NORM_PARTIALS - 1) / NORM_PARTIALS;
    chunk = chunk < 4096 ? 4096 : (chunk + 1023) / 1024 * 1024;
    GS_REQUIRE(chunk < 0x7fffffffLL, "gs_grad_norm: too many elements");
    hipStream_t s = (hipStream_t)stream;
    double *partials = (double *)workspace;
    uint2 *spans = each ? (uint2 *)(partials + NORM_PARTIALS + n_tensors) : nullptr;
    unsigned n_partials = 0;
    // (a tensor without elements has one partial sum too: zero)
    NormBatch b;
    b.chunk = (unsigned)chunk;
    b.n_tensors = 0;
    b.first_block[0] = 0;
    for (int i = 0; i <= n_tensors; ++i) {
        const bool end = i == n_tensors;
        if (!end && entry(host_row_mask, i)) continue;
        if (b.n_tensors > 0 && (end || b.n_tensors == MAX_NORM_TENSORS)) {
            hipLaunchKernelGGL(norm_partial_kernel, dim3(b.first_block[b.n_tensors]), dim3(GS_BLOCK), 0, s, b, n_partials, partials, spans);
            GS_CHECK_LAUNCH();
            n_partials += b.first_block[b.n_tensors];
            b.n_tensors = 0;
        }
        if (end) break;
        const long long parts = host_numel[i] == 0 ? 1 : (host_numel[i] + chunk - 1) / chunk;
        b.t[b.n_tensors] = {(const void *)host_grad[i], (u64)host_numel[i] << 2 | (u64)host_dtype[i]};
        b.id[b.n_tensors] = i;
        b.first_block[b.n_tensors + 1] = b.first_block[b.n_tensors] + (unsigned)parts;
        ++b.n_tensors;
    }
    NormMaskedBatch m;
    m.chunk = (unsigned)chunk;
    m.n_tensors = 0;
    m.first_block[0] = 0;
    for (int i = 0; host_row_mask && i <= n_tensors; ++i) {
        const bool end = i == n_tensors;
        if (!end && !host_row_mask[i]) continue;
        if (m.n_tensors > 0 && (end || m.n_tensors == MAX_NORM_MASKED)) {
            hipLaunchKernelGGL(norm_masked_kernel, dim3(m.first_block[m.n_tensors]), dim3(GS_BLOCK), 0, s, m, n_partials, partials, spans);
            GS_CHECK_LAUNCH();
            n_partials += m.first_block[m.n_tensors];
            m.n_tensors = 0;
        }
        if (end) break;
        const long long rows = host_numel[i] / host_row_len[i], per = norm_rows(chunk, host_row_len[i]), parts = rows == 0 ? 1 : (rows + per - 1) / per;
        m.t[m.n_tensors] = {(const void *)host_grad[i], (const int8_t *)host_row_mask[i], host_numel[i], host_row_len[i], host_dtype[i]};
        m.id[m.n_tensors] = i;
        m.first_block[m.n_tensors + 1] = m.first_block[m.n_tensors] + (unsigned)parts;
        ++m.n_tensors;
    }
    const int each_blocks = each ? (n_tensors + FINISH_THREADS / GS_WAVE - 1) / (FINISH_THREADS / GS_WAVE) : 0;
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1 + each_blocks), dim3(FINISH_THREADS), 0, s, partials, spans, n_partials, n_tensors, max_norm,
                       sq_sum, norm, clip, each);
    GS_CHECK_LAUNCH();
    return 0;
}

extern "C" int gs_clip_coefficient(const double *sq_sum, double max_norm, float *norm, float *clip, void *stream) {
    GS_REQUIRE(sq_sum && norm && clip, "gs_clip_coefficient: null pointer");
    hipLaunchKernelGGL(clip_coefficient_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, sq_sum, max_norm, norm, clip);
    GS_CHECK_LAUNCH();
    return 0;
}
