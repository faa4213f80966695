// What the two attention kernels share (attend.hip: few rows; attend_prompt.hip: many): arguments, operands, cross-lane steps.
#pragma once
#include "kv.hpp"

namespace oxhip {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttendArgs {
    KvView kv;
    KvBatchView b;
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    const float* slopes;
    const int32_t *prefix, *first;
    float* partial;
    uint32_t* counters;
    float scale, cap;  // scale: the mantissa of the call's, times log2 e
    int32_t power;     // the call's scale's
    uint32_t g, window, cols, vec, quantum, many, least, prompt;  // cols: entries of a tile that may be in use; vec: q by 16 bytes, out by 16 bytes
};

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NO_MAX = -1.7e38f;      // below any score, and far enough from it that 2^(NO_MAX - score) is 0
constexpr uint32_t MOST_SPLITS = 512;  // parts of a tile: the workgroups that the chip holds, at most
constexpr float HEAD_ROOM = 11.0f, MOST_ROOM = 15.0f;  // log2 of a weight when the maximum is set, and before it is set anew
// Maxima past this are far: a step of f32 there is 1/8 and more, and an exponent made in one rounding of a score, or of the maximum and the value scale's
// logarithm, may be off by one, past what f16 holds. Far rows take score less maximum first, which is exact for those that count; what the
// maximum's own rounding leaves (the logarithm at most) is cut off below 2^16.
constexpr float FAR = 0x1p20f, F16_ROOM = 15.9f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > FAR && m > NO_MAX; }
// What a block's largest score may be before a step leaves the common path: the maximum is to be set anew, or `each` step has what that path does not do.
__device__ __forceinline__ float bar_of(float m, bool each) { return each || is_far(m) ? -__builtin_inff() : m + (MOST_ROOM - HEAD_ROOM); }

// Scales under KV_SCALE_MIN count as 0. A block of such keys scores 0. A block of such values has a logarithm that no other has, its weights are taken for
// the sum alone.
__device__ __forceinline__ float key_scale(float held) { return held < KV_SCALE_MIN ? 0.0f : held; }
constexpr float NO_VALUES = -61.0f;
__device__ __forceinline__ float value_log(float held) { return held < KV_SCALE_MIN ? NO_VALUES : __builtin_amdgcn_logf(held); }
__device__ __forceinline__ bool no_values(float log) { return __float_as_uint(log) == __builtin_bit_cast(uint32_t, NO_VALUES); }

// What makes a score, times log2 e, of the product of a row's operands and a block's codes: the call's scale (its mantissa times log2 e, which the key scales
// are multiplied with) and two powers of two, the call's and the one that the row's operands were divided by. Either may lie outside f32, so they are added first. A masked
// score times its factor is to stay -infinity: without rules it is above 0 (products are below 2^29, so that no weight shows a factor of 2^-100).
template <bool RULES>
__device__ __forceinline__ float score_factor(float scaled_key, int power) {
    const float f = ldexpf(scaled_key, power);
    return RULES ? f : fmaxf(f, 0x1p-100f);
}
// The power of two by which a row whose largest value is `top` is divided, so that it lies below 2^14; a row of zeros has a factor that is not infinite.
__device__ __forceinline__ int row_power(float top) { return top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 14 : -1000; }

// Eight codes as f16 values, exactly.
__device__ __forceinline__ half8 code_values(uint32_t a, uint32_t b) {
    const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    union { half2v h[4]; half8 v; } o;
    o.h[0] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(a, 0x64646464u, 0x00050004u)) + off;
    o.h[1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(a, 0x64646464u, 0x00070006u)) + off;
    o.h[2] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u)) + off;
    o.h[3] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)) + off;
    return o.v;
}
__device__ __forceinline__ f32x4 mma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// Over the four lanes that hold an entry's scores, 16 apart: the largest, and the sum.
template <class F>
__device__ __forceinline__ float entry_fold(float v, F f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float entry_max(float v) {
    return entry_fold(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float entry_sum(float v) {
    return entry_fold(v, [](float a, float b) { return a + b; });
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int32_t lanes_of(int32_t v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
// Over the 16 entries (the lanes of a row of 16), as a scalar.
template <class F>
__device__ __forceinline__ int32_t tile_fold(int32_t v, F f) {
    v = f(v, lanes_of<0x128>(v));  // row_ror:8, 4, 2, 1
    v = f(v, lanes_of<0x124>(v));
    v = f(v, lanes_of<0x122>(v));
    v = f(v, lanes_of<0x121>(v));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int32_t tile_min(int32_t v) {
    return tile_fold(v, [](int32_t a, int32_t b) { return min(a, b); });
}
__device__ __forceinline__ int32_t tile_max(int32_t v) {
    return tile_fold(v, [](int32_t a, int32_t b) { return max(a, b); });
}
// The sum of a wave's lanes up to one's own.
__device__ __forceinline__ uint32_t lanes_upto(uint32_t v) {
    v += (uint32_t)lanes_of<0x111>((int32_t)v);  // row_shr:1, 2, 4, 8
    v += (uint32_t)lanes_of<0x112>((int32_t)v);
    v += (uint32_t)lanes_of<0x114>((int32_t)v);
    v += (uint32_t)lanes_of<0x118>((int32_t)v);
    v += (uint32_t)lanes_of<0x142, 0xA>((int32_t)v);  // row_bcast:15, then :31
    v += (uint32_t)lanes_of<0x143, 0xC>((int32_t)v);
    return v;
}
// tanh: by its series below 1/4 (the next term is 2^-27 of the value), where 1 - 2 / (e^2x + 1) cancels, and by that above.
__device__ __forceinline__ float tanh_of(float x) {
    const float a = fabsf(x), z = x * x;
    const float series = x + x * z * (-0.333333333f + z * (0.133333333f + z * (-0.0539682540f + z * (0.0218694885f - z * 0.00886323553f))));
    const float e = __builtin_amdgcn_exp2f(2.0f * LOG2E * a);
    return a < 0.25f ? series : copysignf(fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f), x);
}

// A value that all lanes hold alike, as a scalar.
__device__ __forceinline__ uint32_t scalar(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// Eight consecutive values of a row of queries; `vec`: by 16 bytes.
template <bool F32>
__device__ __forceinline__ void load_query(const void* q, size_t at, bool vec, float* v) {
    if constexpr (F32) {
        const float* p = static_cast<const float*>(q) + at;
        if (vec) {
            const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
            v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = p[j];
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(q) + at;
        if (vec) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = bf16_bits_to_f32(p[j]);
        }
    }
}

// Entries (rows x heads of a group) of a sequence from which on attend_prompt_kernel takes it.
constexpr uint32_t PROMPT_ENTRIES = 128;
hipError_t launch_attend_prompt(const AttendArgs& a, bool bf16, bool rules, hipStream_t s);

}  // namespace oxhip
