// gs_adamw.hip -- AdamW over many tensors with moments in 32 or 8 bits, the norm of gradients, the reading of 8-bit moments.
//
// All of it is streaming: per element a step reads and writes parameter, gradient and moments once (28 bytes for float
// tensors with 32-bit moments, 16.06 with 8-bit ones) and computes 20 to 60 instructions, so HBM bounds the large cases and
// launches the small ones.  Hence: one launch for many tensors (their addresses travel as kernel arguments: no table to
// upload, nothing to keep, capturable), a workgroup finds its tensor from its block index.
//
// A tensor is cut into units: a row (1..64 elements) or 64 consecutive elements.  GROUP lanes (up to 16) work on a unit, so
// the largest value of a block -- the 8-bit moments' exponent -- is a reduction inside a DPP row: no shared memory, no
// barrier.
#include "gs_common.h"

#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

namespace {

typedef unsigned long long u64;
constexpr int UNIT = 64;            // elements of a block where blocks are not rows
constexpr int MAX_TENSORS = 48;     // a batch's table is 3.9 KB of kernel arguments
constexpr int MAX_SETS = 4;         // different (learning rate, step, ...) in a batch
constexpr int MAX_NORM_TENSORS = 192, MAX_NORM_MASKED = 64;
// Most workgroups that the norm's first pass aims at, beyond one for each tensor: a round of eight to a compute unit.
constexpr int NORM_PARTIALS = 2000;
// Gradients of more bytes than this pass the caches by: what is read next (a clipped step's first gradients) is gone by
// then.  Below, the step finds them there.  (944 MB: 205 -> 185 us by, 109 MB and a step: 273 us through, 285 by.)
constexpr long long NORM_STREAM_BYTES = 128LL << 20;

// What a step needs besides the tensors; key and step belong to one tensor
struct AdamwScalars {
    float rate, root, keep, one_minus_beta1, beta2, one_minus_beta2, eps, beta1;    // rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
    int step;
    uint32_t key;
};

// Quads of four consecutive elements a lane, so that an access is 16 bytes of each float buffer.  Two side by side (PAIR)
// where the parameter has 16 bits, its moments 8 and there is no master copy: 16 bytes of the parameter again, and half the
// instructions an element for a block's largest value, exponents and scales, which bound that case.
constexpr bool pairs(int dtype, bool master, bool state8) { return state8 && dtype != GS_DTYPE_F32 && !master; }
// Rows under a mask that a wave packs, all of them in flight.  us of a step of 1.2M rows, all live / 30 % at random / the first
// 30 %: 32 bits: 16 rows 335 / 175 / 114, 32: 362 / 182 / 117, 64: 376 / 173 / 128; 8 bits: 196 / 118 / 76, 203 / 122 / 73,
// 215 / 127 / 74, and 132, 120, 121 of the second where a tenth of the rows comes back late.
// Shorter rows: as many quads in flight, up to a row a lane.
__host__ __device__ constexpr int masked_rows(int lanes, bool state8) { return lanes <= 4 || (lanes == 8 && state8) ? GS_WAVE : GS_WAVE / lanes * (state8 ? 8 : 4); }

// How a tensor is cut among lanes
enum Form : int {
    QUADS,          // units of 64, or rows of 36, 40 .. 64 (of 40, 48 .. with pairs of quads): 16 lanes a unit, or 8 with pairs
    ROWS,           // other rows from five elements on: 2, 4, 8 or 16 lanes a row
    QUADS_MASKED,   // the rows of QUADS under a mask: a wave packs the live ones
    ROWS_MASKED,    // the rows of ROWS under a mask, the same way
    NARROW          // rows of 1 to 4 elements: whole quads of rows a lane
};
// Passes of a lane over its workgroup's units, of a quad each, or of a pair where QUADS has pairs (ROWS has none)
constexpr int passes(int quads, bool pair) { return pair ? (quads + 1) / 2 : quads; }
// Lanes for a row of ROWS.  40M floats with 8-bit moments in rows of 5 / 8 / 17 / 24 / 45: 128 / 107 / 144 / 112 / 128 us (element by
// element 404 / 278 / 461 / 178 / 235; 16 lanes for all would idle most of them), rows of 56 as QUADS 113; all live under a mask
// 202 / 133 / 162 / 123 / 138 (646 / 426 / 715 / 176 / 325), rows of 56 118.
__host__ __device__ constexpr int lanes_of(int row_len) { return row_len == 0 || row_len > 32 ? 16 : (row_len > 16 ? 8 : (row_len > 8 ? 4 : 2)); }

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

// One hash serves four consecutive elements, element j with the hash rotated by 8 j; of an element's 32 bits the lower half
// rounds the first moment, the upper half the second.  Here: a half in the middle of 20 bits, 16 h + 8.
__device__ __forceinline__ uint32_t bits_for_m(uint32_t hash, int j) { return (__builtin_rotateleft32(hash, 8 * j + 4) & 0xFFFF0u) | 8u; }
__device__ __forceinline__ uint32_t bits_for_v(uint32_t hash, int j) { return (__builtin_rotateleft32(hash, 8 * j + 20) & 0xFFFF0u) | 8u; }

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

// A type at any address: the wide accesses need no alignment here, so views at odd offsets take the same code.
template <typename T> struct Anywhere { typedef T type __attribute__((aligned(1), may_alias)); };
template <typename T>
__device__ __forceinline__ T load_at(const void *p) { return *(const typename Anywhere<T>::type *)p; }
template <typename T>
__device__ __forceinline__ void store_at(void *p, T x) { *(typename Anywhere<T>::type *)p = x; }

template <int DT> struct Four;
template <> struct Four<GS_DTYPE_F32> { typedef f32x4 type; };
template <> struct Four<GS_DTYPE_BF16> { typedef bf16x4 type; };
template <> struct Four<GS_DTYPE_F16> { typedef f16x4 type; };

// sixteen bytes
template <int DT> struct Wide;
template <> struct Wide<GS_DTYPE_F32> { typedef f32x4 type; };
template <> struct Wide<GS_DTYPE_BF16> { typedef bf16x8 type; };
template <> struct Wide<GS_DTYPE_F16> { typedef f16x8 type; };

// ------------------------------------------------------------------ 8-bit moments
__device__ __forceinline__ float from_bits(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t to_bits(float x) { return __builtin_bit_cast(uint32_t, x); }

// A first moment's code is an 8-bit float of 4 exponent and 3 mantissa bits (with gradual underflow), which the hardware
// converts; its block's factor is 2^(X - 135).  A second moment's code c is the upper bits of a float: its bits are
// (c << 20) + v_base with v_base = (X - 31) << 23, no factor needed.
__device__ __forceinline__ float m_scale(uint32_t x) {
    const uint32_t xm = x & 255u;
    return xm == 255u ? __builtin_nanf("") : from_bits(((xm < 9u ? 9u : xm) - 8u) << 23);
}
__device__ __forceinline__ uint32_t v_base(uint32_t x) {
    const uint32_t xv = x >> 8 & 255u;
    return ((xv < 32u ? 32u : xv) - 31u) << 23;
}
__device__ __forceinline__ bool v_is_nan(uint32_t x) { return (x >> 8 & 255u) == 255u; }
__device__ __forceinline__ float v_of(uint32_t c, uint32_t base) { return c == 0u ? 0.f : from_bits((c << 20) + base); }
__device__ __forceinline__ float unit_of(uint32_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

template <int J>
__device__ __forceinline__ float unit_byte(uint32_t codes) { return __builtin_amdgcn_cvt_f32_fp8((int)codes, J); }
__device__ __forceinline__ float unit_at(uint32_t codes, int j) {
    return j == 0 ? unit_byte<0>(codes) : j == 1 ? unit_byte<1>(codes) : j == 2 ? unit_byte<2>(codes) : unit_byte<3>(codes);
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x4 units_of(uint32_t codes) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    return f32x4{a[0], a[1], b[0], b[1]};
}

// Exponent byte of a block from the bits of its largest magnitude (positive floats order like their bits, NaN above all):
// `carry` moves values whose mantissa is over the largest code's to the next power, so that rounding up stays in range.  A finite
// value makes 254 at most, what is infinite or NaN makes 255.
constexpr uint32_t INF_BITS = 0x7F800000u;
__device__ __forceinline__ uint32_t block_exponent(uint32_t largest, uint32_t carry, uint32_t low) {
    return max(min(largest + carry, max(largest, INF_BITS - 1u)) >> 23, low);
}
constexpr uint32_t CARRY_M = 0x1FFFFFu, CARRY_V = 0x0FFFFFu, LOW_M = 9u, LOW_V = 32u;

// Code of a first moment, in the top byte of a word.  |m| 2^(15 - X) is a float whose bits, cut after the third mantissa
// bit, are the code: float's own gradual underflow falls where the code's begins.  The 20 bits below meet 20 random ones:
// the carry into the code has the chance that keeps the mean.  Under X = 254 the largest code stands for 1.75 2^127, and finite
// values beyond become that.  (A minimum an element: a branch for the rare blocks that need it parts the quads of a lane, and 1M
// points took 230 us with it, 226 without.)
constexpr uint32_t TOP_M = INF_BITS - 1u - CARRY_M;
__device__ __forceinline__ uint32_t m_word(float m, uint32_t xm, uint32_t bits) {
    const uint32_t u = (to_bits(ldexpf(fminf(fabsf(m), from_bits(TOP_M)), 15 - (int)xm)) + bits) << 4;
    return (u & 0x7FFFFFFFu) | (to_bits(m) & 0x80000000u);
}
// Code of a second moment: v's bits less the block's base, rounded the same way; a value over zero stays over zero (it is a
// divisor's square), and 255 is the last.  The difference is negative below the smallest code, and does not pass 2^28 + 2^20 above.
__device__ __forceinline__ uint32_t v_code(float v, uint32_t base, uint32_t bits) {
    const int c = (int)(to_bits(v) - base + bits) >> 20, low = (int)min(to_bits(v), 1u);
    int code;       // between low and 255, in one instruction
    asm("v_med3_i32 %0, %1, %2, %3" : "=v"(code) : "v"(c), "v"(low), "s"(255));
    return (uint32_t)code;
}
__device__ __forceinline__ uint32_t pack_top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0703u) | __builtin_amdgcn_perm(d, c, 0x07030c0cu);
}

// Largest of GROUP consecutive lanes, in all of them (GROUP = 2, 4: quad permutations, 8: and a mirrored half row, 16: rotations
// of a DPP row)
template <int GROUP>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
    if (GROUP == 2 || GROUP == 4 || GROUP == 8) {
        x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
        if (GROUP > 2) x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
        if (GROUP == 8) x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));
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

template <bool MASTER>
__device__ __forceinline__ float moved(float p, float change, const AdamwScalars &k) {
    p = p * k.keep - k.rate * change;
    // (a 16-bit parameter is its master copy rounded: without the stop the conversion may join the last operation)
    if (MASTER) asm volatile("" : "+v"(p));
    return p;
}

// Moments in 32 bits: the correctly rounded square root and division, hidden behind 28 bytes an element
template <bool MASTER>
__device__ __forceinline__ float update_one(float p, float g, float &m, float &v, const AdamwScalars &k) {
    m = fmaf(k.one_minus_beta1, g - m, m);
    v = fmaf(k.one_minus_beta2 * g, g, k.beta2 * v);
    return moved<MASTER>(p, m / (sqrtf(v) * k.root + k.eps), k);
}

// Moments in 8 bits are bound by their arithmetic: what is the same for a block goes into two factors, and the square root
// and the reciprocal are the hardware's (one unit in the last place each; the codes do not depend on them).  The moments
// themselves are computed one rounding an operation, as the formulas are written: a code is decided by the last bits of a
// moment, and this way they are those of any other float implementation.
struct OldBlock {
    float m_factor, v_factor;       // 2^(X - 135) and 1, times what late rows lost; NaN for 255
    uint32_t base;
    __device__ __forceinline__ OldBlock(uint32_t x, float decay_m, float decay_v)
        : m_factor(decay_m * m_scale(x)), v_factor(v_is_nan(x) ? __builtin_nanf("") : decay_v), base(v_base(x)) {}
};
// LATE: the row may have a decay.  (Without, beta2 joins the factor that is 1 or NaN: an operation less.)
template <bool MASTER, bool LATE>
__device__ __forceinline__ float update_coded(float p, float g, float m_unit, uint32_t v_old, const OldBlock &o, float &m, float &v, const AdamwScalars &k) {
    {
#pragma clang fp contract(off)
        m = o.m_factor * m_unit;
        m = m + k.one_minus_beta1 * (g - m);
        const float old = v_of(v_old, o.base);
        v = (LATE ? k.beta2 * (o.v_factor * old) : (k.beta2 * o.v_factor) * old) + k.one_minus_beta2 * g * g;
    }
    return moved<MASTER>(p, m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * k.root + k.eps), k);
}

// What a row that was last stepped at `last` has to be multiplied with before this step
__device__ __forceinline__ void row_decay(const AdamwScalars &k, int last, float &decay_m, float &decay_v) {
    const int gap = k.step - 1 - last;
    if (gap > 0) {
        decay_m = powf(k.beta1, (float)gap);
        decay_v = powf(k.beta2, (float)gap);
    }
}

// Codes and exponent bytes of a block from the lanes that share it: Q quads of consecutive elements a lane, the first of
// which begins at element 4 quad + shift; SHIFTED: shift may be other than 0, so that a quad's elements meet two hashes.
template <int GROUP, bool SHIFTED, int Q>
__device__ __forceinline__ uint32_t encode(const f32x4 (&m)[Q], const f32x4 (&v)[Q], uint32_t quad, uint32_t shift, uint32_t key, uint32_t (&mc)[Q], uint32_t (&vc)[Q]) {
    uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) {
        top_m = max(top_m, to_bits(m[e / 4][e % 4]) & 0x7FFFFFFFu);
        top_v = max(top_v, to_bits(v[e / 4][e % 4]));
    }
    // (v is not negative; a NaN may carry a sign)
    const uint32_t xm = block_exponent(group_max<GROUP>(top_m), CARRY_M, LOW_M), xv = block_exponent(group_max<GROUP>(top_v & 0x7FFFFFFFu), CARRY_V, LOW_V);
    const uint32_t base = (xv - 31u) << 23;
#pragma unroll
    for (int c = 0; c < Q; ++c) {
        const uint32_t hash = mix32((quad + c) ^ key), next = SHIFTED ? mix32((quad + c + 1u) ^ key) : 0u;
        uint32_t w[4];
        vc[c] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (element j's place in its aligned quad is (shift + j) % 4: the rotation by 8 times that, the last two bits of the
            // shift being all that it takes)
            const uint32_t h = SHIFTED ? __builtin_rotateleft32(shift + j < 4u ? hash : next, 8u * (shift & 3u)) : hash;
            w[j] = m_word(m[c][j], xm, bits_for_m(h, j));
            vc[c] |= v_code(v[c][j], base, bits_for_v(h, j)) << (8 * j);
        }
        mc[c] = xm == 255u ? 0u : pack_top_bytes(w[0], w[1], w[2], w[3]);
        vc[c] = xv == 255u ? 0u : vc[c];
    }
    return xm | xv << 8;
}

// A tensor's buffers from one place on (the same for a whole workgroup or wave: scalar registers), indexed by 32 bits
template <int DT, bool MASTER, bool STATE8>
struct Buffers {
    const char *source;     // what the step starts from: the master copy or the parameter
    char *param;
    const char *grad;
    char *m, *v;
    uint8_t *exponents;
    uint32_t quad, shift;   // the first element's index / 4 and the rest, for the rounding bits
    __device__ __forceinline__ Buffers(const AdamwTensor &t, long long element, long long unit) {
        constexpr int BYTES = DT == GS_DTYPE_F32 ? 4 : 2, STATE = STATE8 ? 1 : 4;
        source = (const char *)(MASTER ? t.master_or_mask : t.param) + element * (MASTER ? 4 : BYTES);
        param = (char *)t.param + element * BYTES;
        grad = (const char *)t.grad + element * BYTES;
        m = (char *)t.exp_avg + element * STATE;
        v = (char *)t.exp_avg_sq + element * STATE;
        exponents = t.exponents + 2 * unit;
        quad = (uint32_t)(element >> 2);
        shift = (uint32_t)element & 3u;
    }
};

// Parameter, gradient and moments are read once and written once a step, and the next reader of most of them is the next step:
// they pass the caches by.
template <typename T>
__device__ __forceinline__ T stream_load(const void *p) { return __builtin_nontemporal_load((const typename Anywhere<T>::type *)p); }
template <typename T>
__device__ __forceinline__ void stream_store(void *p, T x) { __builtin_nontemporal_store(x, (typename Anywhere<T>::type *)p); }

// One or two quads of consecutive elements a lane: what a lane reads before the step and writes after it.  (Two float quads
// a lane are no gain: an access of the wave then covers half of each cache line, and every line is asked for twice.)
// LANES: of a row of any length from 4 elements on, 0 for units of QUADS.  Where a row's length is no multiple of four its last
// lane takes the last four elements, some of which its neighbour has, too: both read them before either writes the same result.
template <int DT, bool MASTER, bool STATE8, int LANES = 0, bool STREAM = true>
struct Share {
    typedef Buffers<DT, MASTER, STATE8> B;
    typedef typename Four<DT>::type Value;
    typedef typename Four<MASTER ? GS_DTYPE_F32 : DT>::type Source;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    static constexpr bool PAIR = LANES == 0 && pairs(DT, MASTER, STATE8);
    static constexpr int Q = PAIR ? 2 : 1, GROUP = LANES > 0 ? LANES : 16 / Q;
    Source p[Q];
    Value g[Q];
    f32x4 m[Q], v[Q];
    uint32_t mc[Q], vc[Q];
    uint32_t e;             // the first element, counted from the buffers' beginning

    // Lane `sub` of a block that begins at `first` and has `len` elements; a lane past its end takes the block's last ones.
    __device__ __forceinline__ void place(uint32_t first, uint32_t len, uint32_t sub) { e = first + min(4u * Q * sub, len - 4u * Q); }
    static __device__ __forceinline__ bool inside(uint32_t len, uint32_t sub) { return 4u * Q * sub < len; }

    template <typename T>
    static __device__ __forceinline__ T get(const char *p) { return STREAM ? stream_load<T>(p) : load_at<T>(p); }
    template <typename T>
    static __device__ __forceinline__ void put(char *p, T x) {
        if (STREAM) stream_store(p, x);
        else store_at(p, x);
    }
    __device__ __forceinline__ void load(const B &b) {
        if constexpr (PAIR) {
            const u32x4 x = get<u32x4>(b.source + e * 2u), y = get<u32x4>(b.grad + e * 2u);
            const u32x2 a = get<u32x2>(b.m + e), d = get<u32x2>(b.v + e);
#pragma unroll
            for (int c = 0; c < Q; ++c) {
                p[c] = __builtin_bit_cast(Source, (u32x2){x[2 * c], x[2 * c + 1]});
                g[c] = __builtin_bit_cast(Value, (u32x2){y[2 * c], y[2 * c + 1]});
                mc[c] = a[c];
                vc[c] = d[c];
            }
        } else {
            p[0] = get<Source>(b.source + e * (uint32_t)(sizeof(Source) / 4));
            g[0] = get<Value>(b.grad + e * (uint32_t)(sizeof(Value) / 4));
            if constexpr (STATE8) {
                mc[0] = get<uint32_t>(b.m + e);
                vc[0] = get<uint32_t>(b.v + e);
            } else {
                m[0] = get<f32x4>(b.m + e * 4u);
                v[0] = get<f32x4>(b.v + e * 4u);
            }
        }
    }
    __device__ __forceinline__ void store(const B &b, const f32x4 (&out)[Q]) const {
        if constexpr (PAIR) {
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_convertvector(out[0], Value)), y = __builtin_bit_cast(u32x2, __builtin_convertvector(out[1], Value));
            put(b.param + e * 2u, (u32x4){x[0], x[1], y[0], y[1]});
            put(b.m + e, (u32x2){mc[0], mc[1]});
            put(b.v + e, (u32x2){vc[0], vc[1]});
        } else {
            if (MASTER) put((char *)b.source + e * 4u, out[0]);
            put(b.param + e * (uint32_t)(sizeof(Value) / 4), __builtin_convertvector(out[0], Value));
            if constexpr (STATE8) {
                put(b.m + e, mc[0]);
                put(b.v + e, vc[0]);
            } else {
                put(b.m + e * 4u, m[0]);
                put(b.v + e * 4u, v[0]);
            }
        }
    }
    // The step; returns the exponent bytes of the block that GROUP lanes share
    template <bool LATE>
    __device__ __forceinline__ uint32_t step(f32x4 (&out)[Q], uint32_t x, float decay_m, float decay_v, const B &b, float scale, const AdamwScalars &k) {
#pragma unroll
        for (int c = 0; c < Q; ++c) out[c] = __builtin_convertvector(p[c], f32x4);
        if constexpr (STATE8) {
            const OldBlock o(x, decay_m, decay_v);
#pragma unroll
            for (int c = 0; c < Q; ++c) {
                const f32x4 units = units_of(mc[c]), grad = __builtin_convertvector(g[c], f32x4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float mj, vj;
                    out[c][j] = update_coded<MASTER, LATE>(out[c][j], scaled(grad[j], scale), units[j], (vc[c] >> (8 * j)) & 255u, o, mj, vj, k);
                    m[c][j] = mj;
                    v[c][j] = vj;
                }
            }
            const uint32_t at = b.shift + e;
            return encode<GROUP, (LANES > 0)>(m, v, b.quad + (LANES > 0 ? at : e) / 4u, at % 4u, k.key, mc, vc);
        } else {
#pragma unroll
            for (int c = 0; c < Q; ++c) {
                const f32x4 grad = __builtin_convertvector(g[c], f32x4);
                if (LATE) {
                    m[c] *= decay_m;
                    v[c] *= decay_v;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float mj = m[c][j], vj = v[c][j];
                    out[c][j] = update_one<MASTER>(out[c][j], scaled(grad[j], scale), mj, vj, k);
                    m[c][j] = mj;
                    v[c][j] = vj;
                }
            }
            return 0u;
        }
    }
};

// The element-wise form, for what the others leave: the last unit of a flat tensor (GROUP 16) and narrow rows behind the last
// whole quads (GROUP 1).  GROUP lanes take a unit, elements GROUP apart.
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
    const uint32_t x = STATE8 && live ? t.exponents[2 * unit] | (uint32_t)t.exponents[2 * unit + 1] << 8 : 0u;
    const OldBlock o(x, decay_m, decay_v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[j] = m[j] = v[j] = 0.f;
        if (j < count) {
            const long long i = base + sub + j * GROUP;
            p[j] = MASTER ? ((const float *)t.master_or_mask)[i] : load_one<DT>(t.param, i);
            const float g = scaled(load_one<DT>(t.grad, i), scale);
            if (STATE8) {
                p[j] = update_coded<MASTER, true>(p[j], g, unit_of(((const uint8_t *)t.exp_avg)[i]), ((const uint8_t *)t.exp_avg_sq)[i], o, m[j], v[j], k);
            } else {
                m[j] = ((const float *)t.exp_avg)[i] * decay_m;
                v[j] = ((const float *)t.exp_avg_sq)[i] * decay_v;
                p[j] = update_one<MASTER>(p[j], g, m[j], v[j], k);
            }
        }
    }
    uint32_t xm = 0, xv = 0;
    if (STATE8) {
        uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            top_m = max(top_m, to_bits(m[j]) & 0x7FFFFFFFu);
            top_v = max(top_v, to_bits(v[j]) & 0x7FFFFFFFu);
        }
        xm = block_exponent(group_max<GROUP>(top_m), CARRY_M, LOW_M);
        xv = block_exponent(group_max<GROUP>(top_v), CARRY_V, LOW_V);
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
                const uint32_t hash = mix32((uint32_t)(i >> 2) ^ k.key);
                const int place = (int)(i & 3);
                ((uint8_t *)t.exp_avg)[i] = xm == 255u ? 0 : (uint8_t)(m_word(m[j], xm, bits_for_m(hash, place)) >> 24);
                ((uint8_t *)t.exp_avg_sq)[i] = xv == 255u ? 0 : (uint8_t)v_code(v[j], (xv - 31u) << 23, bits_for_v(hash, place));
            } else {
                ((float *)t.exp_avg)[i] = m[j];
                ((float *)t.exp_avg_sq)[i] = v[j];
            }
        }
    }
}

// A workgroup's share in units is a block's groups of lanes times UNROLL; a lane asks for all its units' data before it uses
// any.  Lanes past a row's end and units past the tensor's read their neighbours' data again (the same largest value) and store
// nothing.
template <int UNROLL, int DT, bool MASTER, bool STATE8, int LANES>
__device__ __forceinline__ void step_quads(const AdamwTensor &t, const AdamwScalars &k, float scale, unsigned chunk) {
    typedef Share<DT, MASTER, STATE8, LANES> S;
    constexpr int GROUP = S::GROUP, PER_PASS = GS_BLOCK / GROUP, SHARE = PER_PASS * UNROLL;
    const uint32_t unit_len = t.row_len > 0 ? t.row_len : UNIT;
    const long long chunk_unit = (long long)chunk * SHARE, whole = t.numel / unit_len;         // units of full length
    const uint32_t units = (uint32_t)min((long long)SHARE, max(0LL, whole - chunk_unit));
    const uint32_t sub = threadIdx.x % GROUP;
    if (units > 0) {
        const Buffers<DT, MASTER, STATE8> b(t, chunk_unit * unit_len, chunk_unit);
        S q[UNROLL];
        uint32_t x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint32_t unit = min(threadIdx.x / GROUP + u * PER_PASS, units - 1u);
            q[u].place(unit * unit_len, unit_len, sub);
            q[u].load(b);
            x[u] = STATE8 ? load_at<uint16_t>(b.exponents + 2u * unit) : 0u;
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint32_t unit = threadIdx.x / GROUP + u * PER_PASS;
            f32x4 p[S::Q];
            const uint32_t new_x = q[u].template step<false>(p, x[u], 1.f, 1.f, b, scale, k);
            if (unit < units && S::inside(unit_len, sub)) {
                q[u].store(b, p);
                if (STATE8 && sub == 0) store_at(b.exponents + 2u * unit, (uint16_t)new_x);
            }
        }
    }
    // the last unit of a flat tensor, where it is shorter
    if (LANES == 0 && whole * unit_len < t.numel && whole >= chunk_unit && whole < chunk_unit + SHARE && threadIdx.x < GS_WAVE)
        step_unit<16, DT, MASTER, STATE8>(t, k, scale, whole + threadIdx.x / 16, (int)unit_len);
}

// Rows under a mask: a wave reads the mask and the stamps of its rows, packs the live ones and steps them PER_PASS at a time, so
// that no lane waits beside a row without a point and none of such a row's data is asked for.
template <bool STATE8, int LANES>
__device__ __forceinline__ void step_quads_masked(const AdamwTensor &t, const AdamwScalars &k, float scale, unsigned chunk) {
    typedef Share<GS_DTYPE_F32, false, STATE8, LANES> S;
    constexpr int GROUP = S::GROUP, PER_PASS = GS_WAVE / GROUP, WAVE_ROWS = masked_rows(GROUP, STATE8), UNROLL = WAVE_ROWS / PER_PASS;
    const uint32_t row_len = t.row_len, lane = gs_lane(), sub = lane % GROUP;
    const long long row0 = ((long long)chunk * (GS_BLOCK / GS_WAVE) + __builtin_amdgcn_readfirstlane(threadIdx.x / GS_WAVE)) * WAVE_ROWS;
    const long long rows = t.numel / row_len;
    if (row0 >= rows) return;
    const bool there = lane < WAVE_ROWS && row0 + lane < rows;
    const bool live = there && ((const int8_t *)t.master_or_mask)[there ? row0 + lane : row0] == 0;
    const u64 lives = __ballot(live), below = (1ull << lane) - 1ull;
    if (lives == 0) return;
    float decay_m = 1.f, decay_v = 1.f;
    int x = 0;
    if (live) {
        row_decay(k, t.last_step[row0 + lane], decay_m, decay_v);
        t.last_step[row0 + lane] = k.step;
        if (STATE8) x = load_at<uint16_t>(t.exponents + 2 * (row0 + lane));
    }
    // lane i learns which lane has the i-th live row
    const int n_live = __popcll(lives);
    const int order = __builtin_amdgcn_ds_permute(4 * (live ? __popcll(lives & below) : 63 - __popcll(~lives & below)), (int)lane);
    const bool any_late = __ballot(decay_m != 1.f || decay_v != 1.f) != 0;
    const Buffers<GS_DTYPE_F32, false, STATE8> b(t, row0 * row_len, row0);
    S q[UNROLL];
    int from[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (PER_PASS * u >= n_live) break;      // (the same for the wave)
        from[u] = __shfl(order, min(PER_PASS * u + (int)(lane / GROUP), n_live - 1), GS_WAVE);
        q[u].place(from[u] * row_len, row_len, sub);
        q[u].load(b);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (PER_PASS * u >= n_live) break;
        const uint32_t old_x = STATE8 ? (uint32_t)__shfl(x, from[u], GS_WAVE) : 0u;
        const float dm = any_late ? __shfl(decay_m, from[u], GS_WAVE) : 1.f, dv = any_late ? __shfl(decay_v, from[u], GS_WAVE) : 1.f;
        f32x4 p[S::Q];
        const uint32_t new_x = q[u].template step<true>(p, old_x, dm, dv, b, scale, k);
        if (PER_PASS * u + (int)(lane / GROUP) < n_live && S::inside(row_len, sub)) {
            q[u].store(b, p);
            if (STATE8 && sub == 0) store_at(b.exponents + 2 * from[u], (uint16_t)new_x);
        }
    }
}

// Rows of L = 1..4 elements, as many rows a lane as make whole quads (rows of three: four rows, three quads): every access
// is four elements although a row is not.  With codes of one quad only a lane has too little in flight: it takes rows at two places
// (40M floats, rows of 1 / 2 / 4: 157 / 143 / 136 us at one, 145 / 134 / 127 at two, 152 / 140 / 132 at four; all live under a mask
// 268 / 237 / 235, 210 / 179 / 164, 217 / 181 / 155).
// 40M bfloat16 in rows of 1 / 2 / 3 / 4: 115 / 95 / 93 / 71 us, a row a lane and element by element 304 / 188 / 152 / 148.
// Masked rows are not written, someone else may do so meanwhile: where some of a lane's rows are masked it stores the others row by
// row.  40M floats under a mask, rows of 1 / 2 / 3, 32 bits, all live 262 / 233 / 243 us, half of them at random 342 / 261 / 290
// (266 / 237 / 248 with whole quads, masked rows as they were read), 30 % 326 / 267 / 276; 8 bits 212 / 181 / 162,
// 279 / 199 / 197, 262 / 197 / 182; row by row throughout, all live: 342 / 246 / 292 and 269 / 189 / 197.
__host__ __device__ constexpr int narrow_rows(int row_len) { return row_len == 4 ? 1 : (row_len == 2 ? 2 : 4); }
__host__ __device__ constexpr int narrow_passes(int row_len, bool state8) { return state8 && row_len != 3 ? 2 : 1; }

template <int L, int DT, bool MASTER, bool STATE8, bool MASKED>
__device__ __forceinline__ void step_narrow(const AdamwTensor &t, const AdamwScalars &k, float scale, unsigned chunk) {
    constexpr int R = narrow_rows(L), Q = R * L / 4, PASSES = narrow_passes(L, STATE8), SHARE = R * PASSES * GS_BLOCK;
    const long long rows = t.numel / L, first = (long long)chunk * SHARE;
    const int left = (int)min((long long)SHARE, rows - first);
    const Buffers<DT, MASTER, STATE8> b(t, first * L, first);
    const int8_t *mask_of = (const int8_t *)t.master_or_mask + (MASKED ? first : 0);
    int32_t *stamps = t.last_step + (MASKED ? first : 0);
    int8_t mask[PASSES][R];
    int last[PASSES][R];
    bool go[PASSES];
    // (single quads; cached: several accesses of the lane touch a line; 202 us, else 232)
    Share<DT, MASTER, STATE8, 2, false> q[PASSES][Q];
    uint16_t x[PASSES][R];
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
        const int row = R * (u * GS_BLOCK + (int)threadIdx.x);
        go[u] = row + R <= left;
        if (MASKED && go[u]) {
            __builtin_memcpy(mask[u], mask_of + row, R);
            __builtin_memcpy(last[u], stamps + row, 4 * R);
        }
    }
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
        const int row = R * (u * GS_BLOCK + (int)threadIdx.x);
        if (MASKED) {
            bool any = false;
#pragma unroll
            for (int r = 0; r < R; ++r) any = any || mask[u][r] == 0;
            go[u] = go[u] && any;
        }
        if (!go[u]) continue;
#pragma unroll
        for (int c = 0; c < Q; ++c) {
            q[u][c].e = (uint32_t)(row * L + 4 * c);
            q[u][c].load(b);
        }
        if (STATE8) __builtin_memcpy(x[u], b.exponents + 2 * row, 2 * R);
    }
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
        if (!go[u]) continue;
        const int row = R * (u * GS_BLOCK + (int)threadIdx.x);
        f32x4 p[Q][1];
        uint32_t mc[Q] = {}, vc[Q] = {};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool live = !MASKED || mask[u][r] == 0;
            float decay_m = 1.f, decay_v = 1.f;
            if (MASKED && live) {
                row_decay(k, last[u][r], decay_m, decay_v);
                last[u][r] = k.step;
            }
            if constexpr (STATE8) {
                const OldBlock o(x[u][r], decay_m, decay_v);
                float m[L], v[L];
                uint32_t top_m = 0u, top_v = 0u;
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    const int c = (r * L + i) / 4, j = (r * L + i) % 4;
                    const auto &s = q[u][c];
                    const float old = (float)s.p[0][j];
                    const float out = update_coded<MASTER, MASKED>(old, scaled((float)s.g[0][j], scale), unit_at(s.mc[0], j), (s.vc[0] >> (8 * j)) & 255u, o, m[i], v[i], k);
                    p[c][0][j] = live ? out : old;
                    top_m = max(top_m, to_bits(m[i]) & 0x7FFFFFFFu);
                    top_v = max(top_v, to_bits(v[i]) & 0x7FFFFFFFu);
                }
                const uint32_t xm = block_exponent(top_m, CARRY_M, LOW_M), xv = block_exponent(top_v, CARRY_V, LOW_V);
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    const int c = (r * L + i) / 4, j = (r * L + i) % 4;
                    const uint32_t hash = mix32((b.quad + q[u][c].e / 4u) ^ k.key);
                    const uint32_t a = xm == 255u ? 0u : m_word(m[i], xm, bits_for_m(hash, j)) >> 24;
                    const uint32_t d = xv == 255u ? 0u : v_code(v[i], (xv - 31u) << 23, bits_for_v(hash, j));
                    mc[c] |= live ? a << (8 * j) : q[u][c].mc[0] & (255u << (8 * j));
                    vc[c] |= live ? d << (8 * j) : q[u][c].vc[0] & (255u << (8 * j));
                }
                if (live) x[u][r] = (uint16_t)(xm | xv << 8);
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    const int c = (r * L + i) / 4, j = (r * L + i) % 4;
                    auto &s = q[u][c];
                    float m = s.m[0][j] * decay_m, v = s.v[0][j] * decay_v;
                    const float out = update_one<false>(s.p[0][j], scaled(s.g[0][j], scale), m, v, k);
                    p[c][0][j] = live ? out : s.p[0][j];
                    s.m[0][j] = live ? m : s.m[0][j];
                    s.v[0][j] = live ? v : s.v[0][j];
                }
            }
        }
        if (MASKED && R > 1) {
            bool all = true;
#pragma unroll
            for (int r = 0; r < R; ++r) all = all && mask[u][r] == 0;
            if (!all) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (mask[u][r] != 0) continue;
                    const uint32_t e = (uint32_t)((row + r) * L);
                    float out[3][L];
                    uint8_t codes[2][L];
#pragma unroll
                    for (int i = 0; i < L; ++i) {
                        const int c = (r * L + i) / 4, j = (r * L + i) % 4;
                        out[0][i] = p[c][0][j];
                        if constexpr (STATE8) {
                            codes[0][i] = (uint8_t)(mc[c] >> (8 * j));
                            codes[1][i] = (uint8_t)(vc[c] >> (8 * j));
                        } else {
                            out[1][i] = q[u][c].m[0][j];
                            out[2][i] = q[u][c].v[0][j];
                        }
                    }
                    __builtin_memcpy(b.param + 4 * e, out[0], 4 * L);
                    if constexpr (STATE8) {
                        __builtin_memcpy(b.m + e, codes[0], L);
                        __builtin_memcpy(b.v + e, codes[1], L);
                        store_at(b.exponents + 2 * (row + r), x[u][r]);
                    } else {
                        __builtin_memcpy(b.m + 4 * e, out[1], 4 * L);
                        __builtin_memcpy(b.v + 4 * e, out[2], 4 * L);
                    }
                    stamps[row + r] = k.step;
                }
                continue;
            }
        }
        if (MASKED) __builtin_memcpy(stamps + row, last[u], 4 * R);
        if (STATE8) __builtin_memcpy(b.exponents + 2 * row, x[u], 2 * R);
#pragma unroll
        for (int c = 0; c < Q; ++c) {
            if (STATE8) {
                q[u][c].mc[0] = mc[c];
                q[u][c].vc[0] = vc[c];
            }
            q[u][c].store(b, p[c]);
        }
    }
    // rows behind the last whole quads
    if (threadIdx.x == 0)
        for (int r = left / R * R; r < left; ++r) step_unit<1, DT, MASTER, STATE8>(t, k, scale, first + r, L);
}

// Chunks that a form makes of a tensor (a workgroup each)
__host__ __device__ inline long long form_chunks(int form, long long numel, int row_len, int quads, bool pair, bool state8) {
    const long long units = row_len > 0 ? numel / row_len : (numel + UNIT - 1) / UNIT;
    const int lanes = form == QUADS || form == QUADS_MASKED ? 16 : lanes_of(row_len);
    const int per = form == QUADS                                 ? GS_BLOCK / lanes * passes(quads, pair) * (pair ? 2 : 1)
                    : form == ROWS                                ? GS_BLOCK / lanes * passes(quads, pair)
                    : form == QUADS_MASKED || form == ROWS_MASKED ? GS_BLOCK / GS_WAVE * masked_rows(lanes, state8)
                                                                  : narrow_rows(row_len) * narrow_passes(row_len, state8) * GS_BLOCK;
    return (units + per - 1) / per;
}

// All tensors of one parameter type and one form of moments, whatever their shapes: the branches on `form` are uniform in a
// workgroup.  Masked tensors have a kernel of their own, whose registers would cost the others occupancy.  Where pairs of quads
// are bound by arithmetic, narrow rows of three would take 83 registers: at least six waves to a SIMD, for which they spill 12 bytes a
// lane (40M bfloat16, rows of 3 / 4 / 7 / 16 / 56: 92 / 79 / 103 / 83 / 71 us; five waves 81 / 84 / 110 / 91 / 74, seven
// 142 / 75 / 97 / 80 / 70).  The other 8-bit forms: five; left alone the float one takes 97 registers and has four (1M points 226 us,
// four waves 224; 40M floats in rows of 5 / 17: 130 / 146, four waves 135 / 153).
template <int QUADS_A_LANE, int DT, bool MASTER, bool STATE8, bool MASKED>
__global__ __launch_bounds__(GS_BLOCK, pairs(DT, MASTER, STATE8) ? 6 : (STATE8 && !MASKED ? 5 : 1)) void adamw_kernel(AdamwBatch b) {
    const int ti = find_tensor<MAX_TENSORS>(b.first_chunk, b.n_tensors, blockIdx.x);
    const AdamwTensor &t = b.t[ti];
    AdamwScalars k = b.device_scalars ? b.device_scalars[ti] : b.scalars[t.set];
    if (!b.device_scalars) k.key = t.key;
    const float scale = b.grad_scale ? *b.grad_scale : 1.f;
    const unsigned chunk = blockIdx.x - b.first_chunk[ti];
    constexpr int PASSES = passes(QUADS_A_LANE, pairs(DT, MASTER, STATE8));
    if constexpr (!MASKED) {
        if (t.form == QUADS) return step_quads<PASSES, DT, MASTER, STATE8, 0>(t, k, scale, chunk);
    }
    if constexpr (MASKED) {
        if (t.form == QUADS_MASKED) return step_quads_masked<STATE8, 0>(t, k, scale, chunk);
        if (t.form == ROWS_MASKED) {
            if (t.row_len > 32) return step_quads_masked<STATE8, 16>(t, k, scale, chunk);
            if (t.row_len > 16) return step_quads_masked<STATE8, 8>(t, k, scale, chunk);
            if (t.row_len > 8) return step_quads_masked<STATE8, 4>(t, k, scale, chunk);
            return step_quads_masked<STATE8, 2>(t, k, scale, chunk);
        }
    } else if constexpr (STATE8) {
        if (t.form == ROWS) {
            if (t.row_len > 32) return step_quads<PASSES, DT, MASTER, true, 16>(t, k, scale, chunk);
            if (t.row_len > 16) return step_quads<PASSES, DT, MASTER, true, 8>(t, k, scale, chunk);
            if (t.row_len > 8) return step_quads<PASSES, DT, MASTER, true, 4>(t, k, scale, chunk);
            return step_quads<PASSES, DT, MASTER, true, 2>(t, k, scale, chunk);
        }
    }
    if constexpr (MASKED || STATE8) {
        if (t.row_len == 3) return step_narrow<3, DT, MASTER, STATE8, MASKED>(t, k, scale, chunk);
        if (t.row_len == 1) return step_narrow<1, DT, MASTER, STATE8, MASKED>(t, k, scale, chunk);
        if (t.row_len == 2) return step_narrow<2, DT, MASTER, STATE8, MASKED>(t, k, scale, chunk);
        return step_narrow<4, DT, MASTER, STATE8, MASKED>(t, k, scale, chunk);
    }
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
    int row_len;
};
struct MomentsBatch {
    int n_tensors;
    unsigned first_chunk[MAX_TENSORS + 1];
    MomentsTensor t[MAX_TENSORS];
};
static_assert(sizeof(MomentsBatch) <= 4000, "kernel arguments");

__device__ __forceinline__ float v_value(uint32_t c, uint32_t x) { return v_is_nan(x) ? __builtin_nanf("") : v_of(c, v_base(x)); }

template <int GROUP, int DT>
__device__ __forceinline__ void read_unit(const MomentsTensor &t, long long unit, int unit_len) {
    const long long base = unit * unit_len, left = t.numel - base;
    const int len = left <= 0 ? 0 : (left < unit_len ? (int)left : unit_len);
    if (len == 0) return;
    const uint32_t x = t.exponents[2 * unit] | (uint32_t)t.exponents[2 * unit + 1] << 8;
    for (int e = threadIdx.x % GROUP; e < len; e += GROUP) {
        store_one<DT>(t.m_out, base + e, unit_of(t.m[base + e]) * m_scale(x));
        store_one<DT>(t.v_out, base + e, v_value(t.v[base + e], x));
    }
}

// (whole cache lines, not read again soon: 240 -> 227 us for a step of 1M points and this, the codes from the caches)
template <int DT, int Q, typename Codes>
__device__ __forceinline__ void read_codes(Codes mc, Codes vc, uint32_t x, char *m_out, char *v_out) {
    typedef float Floats __attribute__((ext_vector_type(4 * Q)));
    typedef typename std::conditional<DT == GS_DTYPE_F32, float, __bf16>::type Element;
    typedef Element Value __attribute__((ext_vector_type(4 * Q)));
    Floats m, v;
#pragma unroll
    for (int c = 0; c < Q; ++c) {
        const f32x4 units = units_of(mc[c]) * m_scale(x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[4 * c + j] = units[j];
            v[4 * c + j] = v_value((vc[c] >> (8 * j)) & 255u, x);
        }
    }
    stream_store(m_out, __builtin_convertvector(m, Value));
    stream_store(v_out, __builtin_convertvector(v, Value));
}

// Units of 64 or rows from five elements on, GROUP lanes each, as in the step; PAIR: two quads a lane
template <int UNROLL, int DT, int GROUP, bool PAIR>
__device__ __forceinline__ void read_quads(const MomentsTensor &t, unsigned chunk) {
    constexpr int PER_PASS = GS_BLOCK / GROUP, SHARE = PER_PASS * UNROLL, BYTES = DT == GS_DTYPE_F32 ? 4 : 2, Q = PAIR ? 2 : 1;
    typedef uint32_t Codes __attribute__((ext_vector_type(Q)));
    const uint32_t unit_len = t.row_len > 0 ? t.row_len : UNIT;
    const long long chunk_unit = (long long)chunk * SHARE, whole = t.numel / unit_len;
    const uint32_t units = (uint32_t)min((long long)SHARE, max(0LL, whole - chunk_unit)), first = 4u * Q * (threadIdx.x % GROUP);
    if (units > 0) {
        const uint8_t *m = t.m + chunk_unit * unit_len, *v = t.v + chunk_unit * unit_len, *exponents = t.exponents + 2 * chunk_unit;
        char *m_out = (char *)t.m_out + chunk_unit * unit_len * BYTES, *v_out = (char *)t.v_out + chunk_unit * unit_len * BYTES;
        Codes mc[UNROLL], vc[UNROLL];
        uint32_t x[UNROLL], e[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const uint32_t unit = min(threadIdx.x / GROUP + u * PER_PASS, units - 1u);
            e[u] = unit * unit_len + min(first, unit_len - 4u * Q);
            mc[u] = load_at<Codes>(m + e[u]);
            vc[u] = load_at<Codes>(v + e[u]);
            x[u] = load_at<uint16_t>(exponents + 2u * unit);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (threadIdx.x / GROUP + u * PER_PASS < units && first < unit_len) read_codes<DT, Q>(mc[u], vc[u], x[u], m_out + e[u] * BYTES, v_out + e[u] * BYTES);
    }
    if (GROUP * Q == 16 && whole * unit_len < t.numel && whole >= chunk_unit && whole < chunk_unit + SHARE && threadIdx.x < GROUP)
        read_unit<GROUP, DT>(t, whole, (int)unit_len);
}

// Rows of L = 1..4 elements: nothing is shared by a row but its exponents, so a lane reads quads wherever rows begin (rows of
// three, 56M elements to bfloat16 / float: 55 / 88 us; with whole rows a lane, 48 bytes from lane to lane, 109 / 242)
template <int UNROLL, int L, int DT>
__device__ __forceinline__ void read_narrow(const MomentsTensor &t, unsigned chunk) {
    constexpr uint32_t SHARE = 4 * GS_BLOCK * UNROLL, BYTES = DT == GS_DTYPE_F32 ? 4 : 2;
    constexpr int R = L == 1 ? 4 : (L == 4 ? 1 : 2);        // rows that a quad meets
    typedef typename Four<DT>::type Value;
    const long long first = (long long)chunk * SHARE, row0 = first / L;
    const uint32_t left = (uint32_t)min((long long)SHARE, t.numel - first), ahead = (uint32_t)(first - row0 * L);
    const uint8_t *m = t.m + first, *v = t.v + first, *exponents = t.exponents + 2 * row0;
    char *m_out = (char *)t.m_out + first * BYTES, *v_out = (char *)t.v_out + first * BYTES;
    uint32_t mc[UNROLL], vc[UNROLL];
    uint16_t x[UNROLL][R];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t e = 4u * (u * GS_BLOCK + threadIdx.x);
        if (e + 4u > left) continue;
        mc[u] = load_at<uint32_t>(m + e);
        vc[u] = load_at<uint32_t>(v + e);
        __builtin_memcpy(x[u], exponents + 2u * ((ahead + e) / L), 2 * R);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint32_t e = 4u * (u * GS_BLOCK + threadIdx.x), phase = L == 3 ? (ahead + e) % L : 0u;      // (place in the first row)
        if (e + 4u > left) continue;
        const f32x4 units = units_of(mc[u]);
        f32x4 mo, vo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t xr = L == 3 ? x[u][phase + j < 3u ? 0 : R - 1] : x[u][j / L];
            mo[j] = units[j] * m_scale(xr);
            vo[j] = v_value((vc[u] >> (8 * j)) & 255u, xr);
        }
        stream_store(m_out + e * BYTES, __builtin_convertvector(mo, Value));
        stream_store(v_out + e * BYTES, __builtin_convertvector(vo, Value));
    }
    if (const uint32_t e = left / 4u * 4u + threadIdx.x; e < left && threadIdx.x < 4) {     // behind the last whole quad
        const uint32_t row = (ahead + e) / L, xr = load_at<uint16_t>(exponents + 2u * row);
        store_one<DT>(m_out, e, unit_of(m[e]) * m_scale(xr));
        store_one<DT>(v_out, e, v_value(v[e], xr));
    }
}

// Two quads a lane to 16-bit values, so that they are 16 bytes: units of 64 and rows of 40, 48, 56 and 64 (56M elements in rows
// of 56: 50 us, 6.7 TB/s, a quad a lane 53)
__host__ __device__ constexpr bool read_pairs(int row_len) { return row_len == 0 || (row_len > 32 && row_len % 8 == 0); }

template <int UNROLL, int DT>
__global__ __launch_bounds__(GS_BLOCK) void read_moments_kernel(MomentsBatch b) {
    const int ti = find_tensor<MAX_TENSORS>(b.first_chunk, b.n_tensors, blockIdx.x);
    const MomentsTensor &t = b.t[ti];
    const unsigned chunk = blockIdx.x - b.first_chunk[ti];
    const int lanes = lanes_of(t.row_len);
    if (t.row_len == 0 || t.row_len > 4) {
        if constexpr (DT != GS_DTYPE_F32)
            if (read_pairs(t.row_len)) return read_quads<passes(UNROLL, true), DT, 8, true>(t, chunk);
        if (lanes == 16) return read_quads<UNROLL, DT, 16, false>(t, chunk);
        if (lanes == 8) return read_quads<UNROLL, DT, 8, false>(t, chunk);
        if (lanes == 4) return read_quads<UNROLL, DT, 4, false>(t, chunk);
        return read_quads<UNROLL, DT, 2, false>(t, chunk);
    }
    if (t.row_len == 3) return read_narrow<UNROLL, 3, DT>(t, chunk);
    if (t.row_len == 1) return read_narrow<UNROLL, 1, DT>(t, chunk);
    if (t.row_len == 2) return read_narrow<UNROLL, 2, DT>(t, chunk);
    return read_narrow<UNROLL, 4, DT>(t, chunk);
}

// ------------------------------------------------------------------ norm of gradients
// First pass: each workgroup adds the squares of one chunk in double precision (a float's square is exact there) and
// leaves a partial sum; the second adds the partial sums.  The order is fixed, so equal inputs give equal bits; the sum of n squares is
// off by n 2^-53 of itself at worst.
struct NormTensor {
    const void *grad;
    u64 numel_type;             // numel * 4 + type
};
struct NormBatch {              // tensors without a row mask
    int n_tensors;
    unsigned chunk;             // elements, a multiple of NORM_STEP
    int first_id;               // of the first tensor in the caller's list; the others follow it
    unsigned first_block[MAX_NORM_TENSORS + 1];
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

constexpr int NORM_STEP = 4096;     // what a workgroup has in flight of float gradients

// Rows of a masked tensor that a workgroup of the first pass takes: at least a chunk's elements, so that there are no more
// parts than without a mask; whole workgroups' worth of rows
__host__ __device__ __forceinline__ long long norm_rows(long long chunk, int row_len) {
    return ((chunk + row_len - 1) / row_len + GS_BLOCK - 1) / GS_BLOCK * GS_BLOCK;
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

// Elements begin..end: 16 bytes a lane, AHEAD requests in flight, past the end none.
template <int DT, bool STREAM>
__device__ __forceinline__ double flat_squares(const void *grad, long long begin, long long end) {
    typedef typename Wide<DT>::type V;
    constexpr int N = 16 / (DT == GS_DTYPE_F32 ? 4 : 2), AHEAD = 4;
    double s = 0.0;
    const unsigned wide = (unsigned)((end - begin) / N);
    const char *g = (const char *)grad + begin * (16 / N);
    for (unsigned q = threadIdx.x; q < wide; q += AHEAD * GS_BLOCK) {
        V x[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            x[a] = {};
            if (q + a * GS_BLOCK < wide) x[a] = STREAM ? stream_load<V>(g + 16ll * (q + a * GS_BLOCK)) : load_at<V>(g + 16ll * (q + a * GS_BLOCK));
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) s = add_squares<N>(s, x[a]);
    }
    for (long long i = begin + (long long)N * wide + threadIdx.x; i < end; i += GS_BLOCK) {
        const double x = (double)load_one<DT>(grad, i);
        s = fma(x, x, s);
    }
    return s;
}

// Rows begin..end of a tensor with a row mask, of up to four elements: a row a lane
template <int DT>
__device__ __forceinline__ double row_squares(const NormMaskedTensor &t, long long begin, long long end) {
    double s = 0.0;
    for (long long row = begin + threadIdx.x; row < end; row += GS_BLOCK) {
        if (t.row_mask[row] != 0) continue;
        for (int j = 0; j < t.row_len; ++j) {
            const double y = (double)load_one<DT>(t.grad, row * t.row_len + j);
            s = fma(y, y, s);
        }
    }
    return s;
}

// The same for longer rows, GROUP lanes each: a wave packs the live ones of 64 rows and has AHEAD quads a lane in flight.  The last
// lane of a row whose length is no multiple of four leaves out what its neighbour has.
template <int DT, int GROUP>
__device__ __forceinline__ double packed_row_squares(const NormMaskedTensor &t, long long begin, long long end) {
    constexpr int AHEAD = 4, PER_PASS = GS_WAVE / GROUP, BYTES = DT == GS_DTYPE_F32 ? 4 : 2;
    const int len = t.row_len, lane = gs_lane(), sub = lane % GROUP, from = min(4 * sub, len - 4), skip = 4 * sub - from;
    double s = 0.0;
    for (long long row0 = begin + threadIdx.x / GS_WAVE * GS_WAVE; row0 < end; row0 += GS_BLOCK) {
        const bool live = row0 + lane < end && t.row_mask[row0 + lane < end ? row0 + lane : row0] == 0;
        const u64 lives = __ballot(live), below = (1ull << lane) - 1ull;
        const int n_live = __popcll(lives);
        const int order = __builtin_amdgcn_ds_permute(4 * (live ? __popcll(lives & below) : 63 - __popcll(~lives & below)), lane);
        for (int at = 0; at < n_live; at += PER_PASS * AHEAD) {
            typename Four<DT>::type x[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int i = at + PER_PASS * a + lane / GROUP;
                const long long row = row0 + __shfl(order, i < n_live ? i : 0, GS_WAVE);
                x[a] = {};
                if (i < n_live && skip < 4) x[a] = load_at<typename Four<DT>::type>((const char *)t.grad + (row * len + from) * BYTES);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double y = j >= skip ? (double)(float)x[a][j] : 0.0;
                    s = fma(y, y, s);
                }
            }
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
        const uint32_t mask = load_at<uint32_t>(t.row_mask + row0);
        f32x4 x[L];
#pragma unroll
        for (int c = 0; c < L; ++c) x[c] = load_at<f32x4>(grad + row0 * L + 4 * c);
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
    if (t.row_len > 32) return packed_row_squares<DT, 16>(t, begin, end);
    if (t.row_len > 16) return packed_row_squares<DT, 8>(t, begin, end);
    if (t.row_len > 8) return packed_row_squares<DT, 4>(t, begin, end);
    if (t.row_len > 4) return packed_row_squares<DT, 2>(t, begin, end);
    if constexpr (DT == GS_DTYPE_F32) {
        if (t.row_len == 3) return narrow_squares<3>(t, begin, end);
        if (t.row_len == 1) return narrow_squares<1>(t, begin, end);
        if (t.row_len == 2) return narrow_squares<2>(t, begin, end);
        return narrow_squares<4>(t, begin, end);
    }
    return row_squares<DT>(t, begin, end);
}

// A workgroup's sum goes behind those of the launches before (`base` of them); spans[i] = {first, number} of tensor i's.
__device__ __forceinline__ void leave_partial(double s, unsigned base, unsigned part, unsigned parts, int id, double *partials, uint2 *spans) {
    s = block_sum<GS_BLOCK>(s);
    if (threadIdx.x == 0) {
        partials[base + blockIdx.x] = s;
        if (part == 0 && spans) spans[id] = make_uint2(base + blockIdx.x, parts);
    }
}

template <bool STREAM>
__global__ __launch_bounds__(GS_BLOCK) void norm_partial_kernel(NormBatch b, unsigned base, double *__restrict__ partials, uint2 *__restrict__ spans) {
    const int ti = find_tensor<MAX_NORM_TENSORS>(b.first_block, b.n_tensors, blockIdx.x);
    const unsigned part = blockIdx.x - b.first_block[ti];
    const void *grad = b.t[ti].grad;
    const long long numel = (long long)(b.t[ti].numel_type >> 2), begin = (long long)part * b.chunk;
    const long long end = min(numel, begin + (long long)b.chunk);
    const int type = (int)(b.t[ti].numel_type & 3);
    double s;
    if (type == GS_DTYPE_F32) s = flat_squares<GS_DTYPE_F32, STREAM>(grad, begin, end);
    else if (type == GS_DTYPE_BF16) s = flat_squares<GS_DTYPE_BF16, STREAM>(grad, begin, end);
    else s = flat_squares<GS_DTYPE_F16, STREAM>(grad, begin, end);
    leave_partial(s, base, part, b.first_block[ti + 1] - b.first_block[ti], b.first_id + ti, partials, spans);
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

// Quads that a lane of step_quads takes.  8 bits: four, to have enough in flight; small totals one (a pair), so that they
// still reach every compute unit.  32 bits: one, and at most four workgroups to a compute unit (OCCUPANCY_LDS bytes each of
// shared memory that nothing uses): more requests to seven streams at once only lose the memory's open rows (1M points: four
// quads 282 us, one 282, one with the limit 263, seven streams of 1652 MB in all).
constexpr int UNROLL = 4, UNROLL_READ = 4;
constexpr int OCCUPANCY_LDS = 40960;
constexpr long long SMALL_CHUNKS = 2048;    // of 16 units
// Workgroups of the largest launch: gridDim.x * blockDim.x has to stay below 2^32
constexpr long long MAX_CHUNKS = (1LL << 32) / GS_BLOCK - 1;

int form_of(int row, bool masked, bool pair) {
    if (row >= 1 && row <= 4) return NARROW;
    if (row == 0 || (row > 32 && row % (pair ? 8 : 4) == 0)) return masked ? QUADS_MASKED : QUADS;
    return masked ? ROWS_MASKED : ROWS;
}
long long read_chunks(long long numel, int row, int dtype, int unroll) {
    const long long units = row > 0 ? numel / row : (numel + UNIT - 1) / UNIT;
    if (row >= 1 && row <= 4) return (numel + 4 * GS_BLOCK * unroll - 1) / (4 * GS_BLOCK * unroll);
    const int per = dtype != GS_DTYPE_F32 && read_pairs(row) ? GS_BLOCK / 8 * passes(unroll, true) : GS_BLOCK / lanes_of(row) * unroll;
    return (units + per - 1) / per;
}

template <int U, bool STATE8>
void launch_step(int dtype, bool master, bool masked, const AdamwBatch &b, hipStream_t s) {
    const dim3 grid(b.first_chunk[b.n_tensors]), block(GS_BLOCK);
    const int lds = STATE8 || masked ? 0 : OCCUPANCY_LDS;
    if (masked) hipLaunchKernelGGL((adamw_kernel<1, GS_DTYPE_F32, false, STATE8, true>), grid, block, 0, s, b);
    else if (dtype == GS_DTYPE_F32) hipLaunchKernelGGL((adamw_kernel<U, GS_DTYPE_F32, false, STATE8, false>), grid, block, lds, s, b);
    else if (dtype == GS_DTYPE_BF16 && master) hipLaunchKernelGGL((adamw_kernel<U, GS_DTYPE_BF16, true, STATE8, false>), grid, block, lds, s, b);
    else if (dtype == GS_DTYPE_BF16) hipLaunchKernelGGL((adamw_kernel<U, GS_DTYPE_BF16, false, STATE8, false>), grid, block, lds, s, b);
    else if (master) hipLaunchKernelGGL((adamw_kernel<U, GS_DTYPE_F16, true, STATE8, false>), grid, block, lds, s, b);
    else hipLaunchKernelGGL((adamw_kernel<U, GS_DTYPE_F16, false, STATE8, false>), grid, block, lds, s, b);
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
        GS_REQUIRE(n == 0 || (host_param[i] && host_grad[i] && host_exp_avg[i] && host_exp_avg_sq[i] && (!state8 || host_exponents[i])),
                   "gs_adamw_step: null tensor");
        GS_REQUIRE(!entry(host_row_mask, i) || (row > 0 && dt == GS_DTYPE_F32 && host_last_step[i]), "gs_adamw_step: a row mask needs float rows and last steps");
        GS_REQUIRE(!entry(host_master, i) || dt != GS_DTYPE_F32, "gs_adamw_step: a master copy belongs to a 16-bit parameter");
        GS_REQUIRE((host_step[i] >= 1 && host_step[i] < 0x7fffffffLL) || entry(host_step_device, i), "gs_adamw_step: step >= 1");
        GS_REQUIRE(h[1] >= 0.0 && h[1] < 1.0 && h[2] >= 0.0 && h[2] < 1.0 && h[3] >= 0.0, "gs_adamw_step: betas in [0, 1), eps >= 0");
        GS_REQUIRE(aligned_to(host_param[i] | host_grad[i], element_bytes(dt)) && aligned_to(state8 ? 0 : host_exp_avg[i] | host_exp_avg_sq[i], 4) &&
                       aligned_to(entry(host_master, i) | (entry(host_row_mask, i) ? host_last_step[i] : 0), 4),
                   "gs_adamw_step: an address is no multiple of its type's size");
        units_of_16 += form_chunks(QUADS, n, row, 1, false, false);
    }
    const int unroll = !state8 || units_of_16 <= SMALL_CHUNKS ? 1 : UNROLL;
    for (int i = 0; i < n_tensors; ++i) {
        const bool masked = entry(host_row_mask, i) != 0, pair = pairs(host_dtype[i], entry(host_master, i) != 0, state8);
        const int row = masked || state8 ? host_row_len[i] : 0;      // (moments in 32 bits without a mask: units of 64 whatever the shape)
        GS_REQUIRE(form_chunks(form_of(row, masked, pair), host_numel[i], row, unroll, pair, state8) <= MAX_CHUNKS, "gs_adamw_step: tensor too large");
    }
    {
        Range *r = (Range *)malloc(((size_t)n_tensors * 10 + 1) * sizeof(Range));
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
            if (entry(host_row_mask, i)) {
                r[k++] = {host_last_step[i], host_last_step[i] + 4 * blocks, 1};
                r[k++] = {host_row_mask[i], host_row_mask[i] + blocks, 0};
            }
            if (entry(host_step_device, i)) r[k++] = {host_step_device[i], host_step_device[i] + 8, 0};
            if (entry(host_lr_device, i)) r[k++] = {host_lr_device[i], host_lr_device[i] + 4, 0};
        }
        if (grad_scale) r[k++] = {(u64)(uintptr_t)grad_scale, (u64)(uintptr_t)grad_scale + 4, 0};
        const bool meet = ranges_meet(r, k);
        free(r);
        GS_REQUIRE(!meet, "gs_adamw_step: buffers overlap");
    }
    hipStream_t s = (hipStream_t)stream;
    AdamwScalars *device_scalars = (AdamwScalars *)workspace;
    StepBatch q;
    q.b.grad_scale = grad_scale;
    // one type after the other: float, float under a mask, 16 bits with and without a master copy
    for (int kind = 0; kind < 6; ++kind) {
        const int dtype = kind / 2;
        const bool masked = kind == 1, master = kind > 1 && kind % 2 != 0;
        q.clear();
        for (int i = 0; i <= n_tensors; ++i) {
            const bool end = i == n_tensors;
            if (!end && (host_numel[i] == 0 || host_dtype[i] != dtype || (entry(host_master, i) != 0) != master ||
                         (entry(host_row_mask, i) != 0) != masked)) continue;
            AdamwTensor t = {};
            long long chunks = 0;
            int set = 0;
            if (!end) {
                const int row = masked || state8 ? host_row_len[i] : 0;
                const bool pair = pairs(dtype, master, state8);
                t.form = form_of(row, masked, pair);
                t.row_len = (uint8_t)row;
                t.masked = masked;
                chunks = form_chunks(t.form, host_numel[i], row, unroll, pair, state8);
                while (!on_device && set < q.n_sets &&
                       (q.step[set] != host_step[i] || memcmp(q.hyper[set], host_hyper + 5 * (size_t)i, 5 * sizeof(double)) != 0)) ++set;
            }
            if (q.b.n_tensors > 0 && (end || q.b.n_tensors == MAX_TENSORS || set == MAX_SETS ||
                                      (long long)q.b.first_chunk[q.b.n_tensors] + chunks > MAX_CHUNKS)) {
                q.b.device_scalars = on_device ? device_scalars : nullptr;
                if (on_device) {
                    q.prep.n = q.b.n_tensors;
                    q.prep.seed = seed;
                    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(GS_WAVE), 0, s, q.prep, device_scalars);
                    device_scalars += q.b.n_tensors;      // (every batch has its own part: n_tensors in all)
                }
                if (!state8) launch_step<1, false>(dtype, master, masked, q.b, s);
                else if (unroll == 1) launch_step<1, true>(dtype, master, masked, q.b, s);
                else launch_step<UNROLL, true>(dtype, master, masked, q.b, s);
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
        GS_REQUIRE(n == 0 || (host_exp_avg[i] && host_exp_avg_sq[i] && host_exponents[i] && host_m_out[i] && host_v_out[i]),
                   "gs_read_moments: null tensor");
        GS_REQUIRE(aligned_to(host_m_out[i] | host_v_out[i], element_bytes(out_dtype)), "gs_read_moments: misaligned output");
        units_of_16 += form_chunks(QUADS, n, row, 1, false, false);
    }
    const int unroll = units_of_16 <= SMALL_CHUNKS ? 1 : UNROLL_READ;
    for (int i = 0; i < n_tensors; ++i)
        GS_REQUIRE(read_chunks(host_numel[i], host_row_len[i], out_dtype, unroll) <= MAX_CHUNKS, "gs_read_moments: tensor too large");
    {
        Range *r = (Range *)malloc((size_t)n_tensors * 5 * sizeof(Range));
        GS_REQUIRE(r != nullptr, "gs_read_moments: out of host memory");
        size_t k = 0;
        for (int i = 0; i < n_tensors; ++i) {
            const u64 n = (u64)host_numel[i], oe = n * element_bytes(out_dtype), row = (u64)host_row_len[i], blocks = row > 0 ? n / row : (n + UNIT - 1) / UNIT;
            r[k++] = {host_exp_avg[i], host_exp_avg[i] + n, 0};
            r[k++] = {host_exp_avg_sq[i], host_exp_avg_sq[i] + n, 0};
            r[k++] = {host_exponents[i], host_exponents[i] + 2 * blocks, 0};
            r[k++] = {host_m_out[i], host_m_out[i] + oe, 1};
            r[k++] = {host_v_out[i], host_v_out[i] + oe, 1};
        }
        const bool meet = ranges_meet(r, k);
        free(r);
        GS_REQUIRE(!meet, "gs_read_moments: an output overlaps another buffer");
    }
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
            t = {(const uint8_t *)host_exp_avg[i], (const uint8_t *)host_exp_avg_sq[i], (const uint8_t *)host_exponents[i],
                 (void *)host_m_out[i], (void *)host_v_out[i], host_numel[i], row};
            chunks = read_chunks(host_numel[i], row, out_dtype, unroll);
        }
        if (b.n_tensors > 0 && (end || b.n_tensors == MAX_TENSORS || (long long)b.first_chunk[b.n_tensors] + chunks > MAX_CHUNKS)) {
            if (unroll == 1) launch_moments<1>(out_dtype, b, (hipStream_t)stream);
            else launch_moments<UNROLL_READ>(out_dtype, b, (hipStream_t)stream);
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
    long long total = 0, bytes = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const long long n = host_numel[i];
        const int dt = host_dtype[i];
        GS_REQUIRE(n >= 0 && n < (1LL << 46), "gs_grad_norm: numel in [0, 2^46)");
        GS_REQUIRE(dt == GS_DTYPE_F32 || dt == GS_DTYPE_BF16 || dt == GS_DTYPE_F16, "gs_grad_norm: unknown dtype");
        GS_REQUIRE(n == 0 || (host_grad[i] && aligned_to(host_grad[i], element_bytes(dt))), "gs_grad_norm: null or misaligned tensor");
        GS_REQUIRE(!entry(host_row_mask, i) || (host_row_len[i] > 0 && host_row_len[i] <= UNIT && n % host_row_len[i] == 0), "gs_grad_norm: a row mask needs rows");
        total += n;
        bytes += n * element_bytes(dt);
    }
    // chunks of a multiple of NORM_STEP elements, so that there are at most NORM_PARTIALS of them and one more for each tensor
    long long chunk = (total + NORM_PARTIALS - 1) / NORM_PARTIALS;
    chunk = chunk < NORM_STEP ? NORM_STEP : (chunk + NORM_STEP - 1) / NORM_STEP * NORM_STEP;
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
        const bool end = i == n_tensors, other = !end && entry(host_row_mask, i);
        if (b.n_tensors > 0 && (end || other || b.n_tensors == MAX_NORM_TENSORS)) {
            const dim3 grid(b.first_block[b.n_tensors]), block(GS_BLOCK);
            if (bytes > NORM_STREAM_BYTES) hipLaunchKernelGGL(norm_partial_kernel<true>, grid, block, 0, s, b, n_partials, partials, spans);
            else hipLaunchKernelGGL(norm_partial_kernel<false>, grid, block, 0, s, b, n_partials, partials, spans);
            GS_CHECK_LAUNCH();
            n_partials += b.first_block[b.n_tensors];
            b.n_tensors = 0;
        }
        if (end) break;
        if (other) continue;
        if (b.n_tensors == 0) b.first_id = i;
        const long long parts = host_numel[i] == 0 ? 1 : (host_numel[i] + chunk - 1) / chunk;
        b.t[b.n_tensors] = {(const void *)host_grad[i], (u64)host_numel[i] << 2 | (u64)host_dtype[i]};
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
