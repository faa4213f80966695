// Filling the 8-bit key / value cache and reading it back: the rotation of queries and keys, the quantization per block of 32 tokens and
// head, and the blocks' layout (kv_plan.hpp).
#include "kv.hpp"

namespace oxhip {

template <bool BF16>
__device__ __forceinline__ float load_value(const void* p, size_t i) {
    if constexpr (BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}
// Eight consecutive values; `vec`: they begin at a 16-byte boundary.
template <bool BF16>
__device__ __forceinline__ void load_eight(const void* p, size_t i, bool vec, float* v) {
    if (vec) {
        if constexpr (BF16) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i), b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = load_value<BF16>(p, i + j);
    }
}

// Channels c .. c + 7 of a head rotated by the angles of position `pos`, in f64 (exact products, one rounding): (a, b) -> (a cos - b sin,
// b cos + a sin) for the pairs (i, i + half), or (2 i, 2 i + 1) where they are interleaved; channels past the pairs stay as they are.
// A position that the table does not hold gives NaN.
template <bool BF16>
__device__ __forceinline__ void rotate_eight(const RopeView& r, const void* p, size_t head, uint32_t c, int32_t pos, bool vec, double* x) {
    float v[8];
    load_eight<BF16>(p, head + c, vec, v);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = v[j];
    if (c >= 2 * r.half) return;
    if ((uint32_t)pos >= r.n_pos) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = c + j < 2 * r.half ? (double)__builtin_nanf("") : x[j];
        return;
    }
    const float2* t = reinterpret_cast<const float2*>(r.table) + (size_t)(uint32_t)pos * r.half;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t cj = c + j;
        if (cj >= 2 * r.half) continue;
        const bool second = r.interleaved ? (cj & 1) : cj >= r.half;
        const uint32_t pair = r.interleaved ? cj / 2 : cj - (second ? r.half : 0u);
        const double other = r.interleaved ? (double)v[j ^ 1] : (double)load_value<BF16>(p, head + (second ? cj - r.half : cj + r.half));
        const float2 a = t[pair];
        const double turned = other * (double)a.y;
        x[j] = (double)v[j] * (double)a.x + (second ? turned : -turned);
    }
}

template <bool BF16>
__device__ __forceinline__ void store_value(void* p, size_t i, double x) {
    if constexpr (BF16) {
        static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits((float)x);  // (by way of f32: half a step of bf16 and 2^-24 of the value at most)
    } else {
        static_cast<float*>(p)[i] = (float)x;
    }
}

struct AppendArgs {
    KvView kv;
    KvBatchView b;
    RopeView rope;
    const void *k, *v, *q;
    void* q_out;
    size_t k_stride, v_stride, q_stride, q_out_stride;
    uint32_t vec;  // k, v and q by 16 bytes
};

// One block of 32 positions (those of them that the call's rows take) of one head per workgroup: blockIdx.y below n_kv its keys, below
// 2 n_kv its values, behind them a query head of the same rows.
// A block's scale s is the largest magnitude of its values over 127 as long as all of them come in one call. Tokens that come later and
// do not fit make it s 2^k, the least such scale that holds them, and the codes that are there are rounded to it: their errors halve
// with every growth, so that none is ever further than s from its value, however the tokens come. (A scale at its floor holds next to
// nothing and grows to what is needed.)
// The bound is memory: rows read once, a byte a value written. A block that is new, or most of it, goes out as whole 16-byte lines through an
// image in LDS (a value operand's tokens lie 1 byte apart, its channels 16); single tokens are stored as they lie.
template <bool BF16>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    __shared__ double top_s[4];
    __shared__ __align__(16) uint8_t image[KV_BLOCK * KV_MAX_D];
    const uint32_t d = a.kv.d, tid = threadIdx.x;
    int32_t s = (int32_t)blockIdx.x, place = 0;
    if (a.b.row_start) {
        s = kv_find(a.b, blockIdx.x, 1, KV_BLOCK, 2);
        place = (int32_t)(blockIdx.x - (uint32_t)kv_first_place((uint32_t)max(a.b.row_start[s], 0), s, KV_BLOCK, 2));
    }
    const KvSeq q = kv_seq(a.b, s, a.kv.shift);
    const int32_t before = q.len - q.n;  // (negative: rows before the sequence's first token are left out)
    const int32_t from = max(before, 0);
    const int32_t block = from / (int32_t)KV_BLOCK + place, p0 = block * (int32_t)KV_BLOCK;
    const int32_t lo = max(p0, from), hi = min(p0 + (int32_t)KV_BLOCK, q.len);  // positions of this block that are new
    if (place < 0 || hi <= lo || q.n <= 0) return;
    const uint32_t per = d / 8, units = (uint32_t)(hi - lo) * per;  // eight channels of a token each
    const size_t first = (size_t)(q.row0 + (lo - before));

    constexpr int MOST = KV_BLOCK * KV_MAX_D / 8 / 256;
    double x[MOST][8];
    if (blockIdx.y >= 2 * a.kv.n_kv) {
        const size_t head = (size_t)(blockIdx.y - 2 * a.kv.n_kv) * d;
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            const uint32_t u = tid + i * 256, t = u / per, c = u % per * 8;
            if (u < units) rotate_eight<BF16>(a.rope, a.q, (first + t) * a.q_stride + head, c, lo + (int32_t)t, a.vec & 4, x[i]);
        }
        __syncthreads();  // q_out may be q: a pair's other half is read by another thread, before anything is stored
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            const uint32_t u = tid + i * 256, t = u / per, c = u % per * 8;
            if (u >= units) continue;
#pragma unroll
            for (int j = 0; j < 8; j++) store_value<BF16>(a.q_out, (first + t) * a.q_out_stride + head + c + j, x[i][j]);
        }
        return;
    }

    const bool values = blockIdx.y >= a.kv.n_kv;
    const uint32_t head = blockIdx.y - (values ? a.kv.n_kv : 0u);
    const int32_t page = kv_page(a.b, a.kv, s, (uint32_t)block);
    if (page < 0) return;  // (a table that names no page of the cache: nothing is written)
    const size_t index = kv_block_index(a.kv, page, head, (uint32_t)block);
    uint8_t* codes = (values ? a.kv.v : a.kv.k) + index * KV_BLOCK * d;
    float* scale_at = (values ? a.kv.v_scale : a.kv.k_scale) + index;
    const bool old = lo > p0;  // the block holds tokens of earlier calls
    const float held = old ? *scale_at : KV_SCALE_MIN;

    double top = 0.0;
    RopeView none{};
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const uint32_t u = tid + i * 256;
        if (u < units) {
            const uint32_t t = u / per, c = u % per * 8;
            if (values) rotate_eight<BF16>(none, a.v, (first + t) * a.v_stride + (size_t)head * d, c, 0, a.vec & 2, x[i]);
            else rotate_eight<BF16>(a.rope, a.k, (first + t) * a.k_stride + (size_t)head * d, c, lo + (int32_t)t, a.vec & 1, x[i]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[i][j] = x[i][j] == x[i][j] ? fmin(fmax(x[i][j], -127.0 * KV_SCALE_MAX), 127.0 * KV_SCALE_MAX) : 0.0;  // (8 bits hold no NaN)
                top = fmax(top, fabs(x[i][j]));
            }
        }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) top = fmax(top, __shfl_xor(top, m));
    if ((tid & 63) == 0) top_s[tid >> 6] = top;
    __syncthreads();
    top = fmax(fmax(top_s[0], top_s[1]), fmax(top_s[2], top_s[3]));
    const float need = fmaxf((float)(top / 127.0), KV_SCALE_MIN);
    const float was = held > KV_SCALE_MIN && held < 2.0f * KV_SCALE_MAX ? held : KV_SCALE_MIN;
    float scale = need;
    if (was > KV_SCALE_MIN) {
        const int more = __builtin_amdgcn_frexp_expf(need) - __builtin_amdgcn_frexp_expf(was) + (__builtin_amdgcn_frexp_mantf(need) > __builtin_amdgcn_frexp_mantf(was) ? 1 : 0);
        scale = ldexpf(was, max(more, 0));
    }
    const bool rescale = old && scale != was;
    const bool whole = rescale || hi - lo > 8;  // the block goes out through its image
    if (whole && old) {
        const float ratio = was / scale;
        for (uint32_t i = tid; i < KV_BLOCK * d / 16; i += 256) {
            const uint4 u = *reinterpret_cast<const uint4*>(codes + 16 * i);
            uint32_t w[4] = {u.x, u.y, u.z, u.w};
            if (rescale) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t r = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float c = rintf(((float)((w[k] >> (8 * j)) & 0xFF) - 128.0f) * ratio);
                        r |= (uint32_t)((int)c + 128) << (8 * j);
                    }
                    w[k] = r;
                }
            }
            *reinterpret_cast<uint4*>(image + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
    }
    const double inv = 1.0 / (double)scale, half = 0.5 * (double)scale;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const uint32_t u = tid + i * 256;
        if (u >= units) continue;
        const uint32_t t = (uint32_t)(lo - p0) + u / per, c = u % per * 8;
        uint32_t code[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            // the integer next to x / scale, halves to the even one: x - r scale is exact, so a product with the reciprocal that came to
            // lie on the other side of a border shows
            double r = rint(x[i][j] * inv);
            const double off = fma(-r, (double)scale, x[i][j]), far = fabs(off);
            if (far > half || (far == half && ((int)r & 1))) r += off > 0.0 ? 1.0 : -1.0;
            code[j] = (uint32_t)((int)fmin(fmax(r, -127.0), 127.0) + 128);
        }
        if (values) {
            uint8_t* to = (whole ? image : codes) + kv_value_offset(t, c);  // (eight consecutive channels lie 16 bytes apart)
#pragma unroll
            for (int j = 0; j < 8; j++) to[16 * j] = (uint8_t)code[j];
        } else {
            uint8_t* to = (whole ? image : codes) + kv_key_offset(t, c);
            *reinterpret_cast<uint2*>(to) = make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24, code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
        }
    }
    if (tid == 0 && (!old || rescale)) *scale_at = scale;
    if (!whole) return;
    __syncthreads();
    if (old) {
        for (uint32_t i = tid; i < KV_BLOCK * d / 16; i += 256) *reinterpret_cast<uint4*>(codes + 16 * i) = *reinterpret_cast<const uint4*>(image + 16 * i);
        return;
    }
    // a block without older tokens: what lies behind the last new one is nobody's yet, and becomes zeros
    for (uint32_t i = tid; i < KV_BLOCK * d / 16; i += 256) {
        uint4 u = *reinterpret_cast<const uint4*>(image + 16 * i);
        if (hi - p0 < (int32_t)KV_BLOCK) {
            const uint32_t g = i * 16 % 1024 / 256, n = i % 16;
            uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (uint32_t k = 0; k < 16; k++) {
                const uint32_t t = values ? k % 8 / 4 * 16 + 4 * g + k % 4 : k / 8 * 16 + n;
                if (t >= (uint32_t)(hi - p0)) w[k / 4] = (w[k / 4] & ~(0xFFu << (8 * (k % 4)))) | 128u << (8 * (k % 4));
            }
            u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(codes + 16 * i) = u;
    }
}

struct ReadArgs {
    KvView kv;
    KvBatchView b;
    void *k_out, *v_out;
    int32_t count;
    uint32_t blocks;  // of a sequence's places, whole or in part
};

// The values that the last `count` tokens of every sequence stand for, [sequence][token][head][d]: a block's part of them per workgroup
// (blockIdx.y: the head's keys, then the head's values), through an image of the block in LDS. Places before a sequence's first token are
// zeros, those of a page that the table does not name NaN. The bound is memory: a byte read, an f32 (or bf16) written.
template <bool BF16>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    __shared__ __align__(16) uint8_t image[KV_BLOCK * KV_MAX_D];
    const uint32_t d = a.kv.d, tid = threadIdx.x;
    const bool values = blockIdx.y >= a.kv.n_kv;
    void* out = values ? a.v_out : a.k_out;
    if (!out) return;
    const int32_t s = (int32_t)(blockIdx.x / a.blocks);
    const KvSeq q = kv_seq(a.b, s, a.kv.shift);
    const int32_t start = q.len - a.count;  // of the places; negative where the sequence is shorter
    const int32_t block = (start >= 0 ? start / (int32_t)KV_BLOCK : -((-start + (int32_t)KV_BLOCK - 1) / (int32_t)KV_BLOCK)) + (int32_t)(blockIdx.x % a.blocks);
    const int32_t p0 = block * (int32_t)KV_BLOCK, lo = max(p0, start), hi = min(p0 + (int32_t)KV_BLOCK, q.len);
    if (hi <= lo) return;
    const uint32_t head = blockIdx.y - (values ? a.kv.n_kv : 0u);
    float scale = 0.0f;
    if (block >= 0) {
        const int32_t page = kv_page(a.b, a.kv, s, (uint32_t)block);
        scale = __builtin_nanf("");
        if (page >= 0) {
            const size_t index = kv_block_index(a.kv, page, head, (uint32_t)block);
            const uint8_t* codes = (values ? a.kv.v : a.kv.k) + index * KV_BLOCK * d;
            scale = (values ? a.kv.v_scale : a.kv.k_scale)[index];
            for (uint32_t i = tid; i < KV_BLOCK * d / 16; i += 256) *reinterpret_cast<uint4*>(image + 16 * i) = *reinterpret_cast<const uint4*>(codes + 16 * i);
        }
        __syncthreads();
    }
    const bool none = block < 0 || scale != scale;  // (the image holds nothing)
    for (uint32_t u = tid; u < (uint32_t)(hi - lo) * d; u += 256) {
        const uint32_t t = (uint32_t)(lo - p0) + u / d, c = u % d;
        const float code = none ? 0.0f : (float)image[values ? kv_value_offset(t, c) : kv_key_offset(t, c)] - 128.0f;
        const size_t to = (((size_t)s * a.count + (size_t)(p0 + (int32_t)t - start)) * a.kv.n_kv + head) * d + c;
        const float x = none ? scale : code * scale;
        if constexpr (BF16) static_cast<uint16_t*>(out)[to] = f32_to_bf16_bits(x);
        else static_cast<float*>(out)[to] = x;
    }
}

hipError_t launch_kv_append(const KvView& kv, const KvBatchView& b, const RopeView& rope, const void* k, size_t k_stride, const void* v, size_t v_stride, const void* q,
                            size_t q_stride, void* q_out, size_t q_out_stride, uint32_t n_q, bool bf16, hipStream_t s) {
    AppendArgs a{kv, b, rope, k, v, q, q_out, k_stride, v_stride, q_stride, q_out_stride, 0};
    const size_t size = bf16 ? 2 : 4;
    auto vec = [&](const void* p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
    a.vec = (vec(k, k_stride) ? 1u : 0u) | (vec(v, v_stride) ? 2u : 0u) | (vec(q, q_stride) ? 4u : 0u);
    const dim3 grid((unsigned)(b.row_start ? kv_places(b.rows, b.n_seqs, KV_BLOCK, 2) : b.n_seqs), 2 * kv.n_kv + n_q);
    if (bf16) kv_append_kernel<true><<<grid, 256, 0, s>>>(a);
    else kv_append_kernel<false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvView& kv, const KvBatchView& b, size_t count, void* k_out, void* v_out, bool bf16, hipStream_t s) {
    const ReadArgs a{kv, b, k_out, v_out, (int32_t)count, (uint32_t)((count + 2 * KV_BLOCK - 2) / KV_BLOCK)};
    const dim3 grid(a.blocks * b.n_seqs, 2 * kv.n_kv);
    if (bf16) kv_read_kernel<true><<<grid, 256, 0, s>>>(a);
    else kv_read_kernel<false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
