// Filling the 8-bit key / value cache and reading it back: the rotation of queries and keys, the quantization per block of 32 tokens and
// head, and the blocks' layout (kv_plan.hpp).
#include <type_traits>

#include "kv.hpp"

namespace oxhip {

template <bool BF16>
__device__ __forceinline__ float load_value(const void* p, size_t i) {
    if constexpr (BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}
// N (4 or 8) consecutive values; `vec`: they begin at a 16-byte boundary (four bf16 ones: at an 8-byte one).
template <bool BF16, int N>
__device__ __forceinline__ void load_run(const void* p, size_t i, bool vec, float* v) {
    if (vec) {
        uint32_t w[BF16 ? N / 2 : N];
        if constexpr (BF16 && N == 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
            w[0] = u.x; w[1] = u.y;
        } else {
#pragma unroll
            for (int k = 0; k < (BF16 ? N / 2 : N); k += 4) {
                const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * (BF16 ? 2 : 4) + 4 * k);
                w[k] = u.x; w[k + 1] = u.y; w[k + 2] = u.z; w[k + 3] = u.w;
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = __uint_as_float(!BF16 ? w[BF16 ? 0 : j] : j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = load_value<BF16>(p, i + j);
    }
}

// N (4 or 8) channels c .. of a head rotated by the angles of position `pos`, in f64 (exact products, one rounding): (a, b) -> (a cos - b sin,
// b cos + a sin) for the pairs (i, i + half), or (2 i, 2 i + 1) where they are interleaved; channels past the pairs stay as they are.
// A position that the table does not hold gives NaN. `even`: half is a multiple of 8, so that a run of channels is all of one kind and its
// partners and angles are runs too.
template <bool BF16, int N>
__device__ __forceinline__ void rotate(const RopeView& r, const void* p, size_t head, uint32_t c, int32_t pos, bool vec, bool even, double* x) {
    float v[N];
    load_run<BF16, N>(p, head + c, vec, v);
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = v[j];
    if (c >= 2 * r.half) return;
    if ((uint32_t)pos >= r.n_pos) {
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = c + j < 2 * r.half ? (double)__builtin_nanf("") : x[j];
        return;
    }
    const float2* t = reinterpret_cast<const float2*>(r.table) + (size_t)(uint32_t)pos * r.half;
    if (even && !r.interleaved) {
        const bool second = c >= r.half;
        const uint32_t other = second ? c - r.half : c + r.half;
        float o[N];
        load_run<BF16, N>(p, head + other, vec, o);
        const float2* angle = t + (second ? other : c);
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float2 a = angle[j];
            const double turned = (double)o[j] * (double)a.y;
            x[j] = (double)v[j] * (double)a.x + (second ? turned : -turned);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
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

// 16 (or 8) bytes of a large result, past the L2: lines that stay there dirty are written back at the kernel's end, which nothing hides (two
// prompts of 4096 rows: appended in 54.5 -> 52.8 us, read back in 29 -> 14; 64 sequences' last 32 tokens read back in 13.5 -> 7.0).
__device__ __forceinline__ void stream_out(void* p, uint4 v) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, static_cast<u32x4*>(p));
}
__device__ __forceinline__ void stream_out(void* p, uint2 v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    __builtin_nontemporal_store(u32x2{v.x, v.y}, static_cast<u32x2*>(p));
}

// Runs of eight channels are a prompt's, of four a step's.
template <bool BF16, int N>
__device__ __forceinline__ void store_run(void* p, size_t i, bool vec, const double* x) {
    uint32_t w[N];  // (f64 to bf16 by way of f32: half a step of bf16 and 2^-24 of the value at most)
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = BF16 ? f32_to_bf16_bits((float)x[j]) : __float_as_uint((float)x[j]);
    if (vec && BF16) {
        uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + i);
        if constexpr (N == 4) *reinterpret_cast<uint2*>(o) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
        else stream_out(o, make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4 % N] | w[5 % N] << 16, w[6 % N] | w[7 % N] << 16));
    } else if (vec) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            uint32_t* o = static_cast<uint32_t*>(p) + i + j;
            const uint4 u = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
            if constexpr (N == 4) *reinterpret_cast<uint4*>(o) = u;
            else stream_out(o, u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) {
            if constexpr (BF16) static_cast<uint16_t*>(p)[i + j] = (uint16_t)w[j];
            else static_cast<uint32_t*>(p)[i + j] = w[j];
        }
    }
}

// What 8 bits hold: no NaN, and nothing past the largest scale.
__device__ __forceinline__ double storable(double x) {
    return x == x ? fmin(fmax(x, -127.0 * KV_SCALE_MAX), 127.0 * KV_SCALE_MAX) : 0.0;
}
// The scale of a block whose new tokens' largest magnitude is `top`; `was`: what it has been for the tokens that are there, KV_SCALE_MIN if there are none.
__device__ __forceinline__ float grown_scale(float was, double top) {
    const float need = fmaxf((float)(top / 127.0), KV_SCALE_MIN);
    if (!(was > KV_SCALE_MIN)) return need;
    const int more = __builtin_amdgcn_frexp_expf(need) - __builtin_amdgcn_frexp_expf(was) + (__builtin_amdgcn_frexp_mantf(need) > __builtin_amdgcn_frexp_mantf(was) ? 1 : 0);
    return ldexpf(was, max(more, 0));
}
__device__ __forceinline__ float sound_scale(float held) { return held > KV_SCALE_MIN && held < 2.0f * KV_SCALE_MAX ? held : KV_SCALE_MIN; }
// The code of x: the integer next to x / scale, halves to the even one (x - r scale is exact, so a product with the reciprocal that came to lie on the
// other side of a border shows).
__device__ __forceinline__ uint32_t code_of(double x, double scale, double inv) {
    double r = rint(x * inv);
    const double off = fma(-r, scale, x), far = fabs(off), half = 0.5 * scale;
    if (far > half || (far == half && ((int)r & 1))) r += off > 0.0 ? 1.0 : -1.0;
    return (uint32_t)((int)fmin(fmax(r, -127.0), 127.0) + 128);
}
// Four codes held by `was` / `scale` of their steps.
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) r |= (uint32_t)((int)rintf(((float)((w >> (8 * j)) & 0xFF) - 128.0f) * ratio) + 128) << (8 * j);
    return r;
}

struct AppendArgs {
    KvView kv;
    KvBatchView b;
    RopeView rope;
    const void *k, *v, *q;
    void* q_out;
    size_t k_stride, v_stride, q_stride, q_out_stride;
    uint32_t vec, even;  // k, v, q and q_out by 16 bytes; whole runs of 8 channels rotate alike
    uint32_t tasks;      // heads of a sequence: keys, values, queries
    SharedView shared;   // or none (group_start nullptr)
};

// The first position that is sequence s's own, by one wave: of the tokens before it, which its group's first sequence holds, nothing is stored, and what the
// cache has in front of it in the same block is no token of this sequence's.
__device__ __forceinline__ int32_t first_own(const SharedView& shared, int32_t s) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0, n = shared.n_groups + 1;  // the last of the groups' borders at s or before it; up to 64 of them take one request
    while (n > 1) {
        const uint32_t step = (n + 63) / 64;
        const uint64_t m = __ballot(lane * step < n && shared.group_start[min(base + lane * step, shared.n_groups)] <= s);
        const uint32_t at = m ? 63u - (uint32_t)__builtin_clzll(m) : 0u;
        base += at * step;
        n = min(step, n - at * step);
    }
    if (base >= shared.n_groups) return 0;
    const int32_t leader = shared.group_start[base];
    return leader >= 0 && leader < s ? max(shared.common[base], 0) : 0;
}

// One block of 32 positions (those of them that the call's rows take) of one head per workgroup: blockIdx.y below n_kv its keys, below
// 2 n_kv its values, behind them a query head of the same rows.
// A block's scale s is the largest magnitude of its values over 127 as long as all of them come in one call. Tokens that come later and
// do not fit make it s 2^k, the least such scale that holds them, and the codes that are there are rounded to it: their errors halve
// with every growth, so that none is ever further than s from its value, however the tokens come. (A scale at its floor holds next to
// nothing and grows to what is needed.)
// The bound is memory: rows read once, a byte a value written. A block that is new, or most of it, goes out as whole 16-byte lines through an
// image in LDS (a value operand's tokens lie 1 byte apart, its channels 16); single tokens are stored as they lie.
// MOST: runs of eight channels a thread holds, d / 64. SHARED: the batch's sequences share first tokens.
template <bool BF16, int MOST, bool SHARED>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    __shared__ double top_s[4];
    __shared__ __align__(16) uint8_t image[KV_BLOCK * 64 * MOST];
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
    int32_t lo = max(p0, from);
    const int32_t hi = min(p0 + (int32_t)KV_BLOCK, q.len);  // positions of this block that are new
    if (place < 0 || hi <= lo || q.n <= 0) return;
    int32_t own = 0;
    const bool query = blockIdx.y >= 2 * a.kv.n_kv;
    if constexpr (SHARED) {
        if (!query) {
            own = first_own(a.shared, s);
            lo = max(lo, own);
            if (hi <= lo) return;
        }
    }
    const uint32_t per = d / 8, units = (uint32_t)(hi - lo) * per;  // eight channels of a token each
    const size_t first = (size_t)(q.row0 + (lo - before));

    double x[MOST][8];
    if (query) {
        const size_t head = (size_t)(blockIdx.y - 2 * a.kv.n_kv) * d;
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            const uint32_t u = tid + i * 256, t = u / per, c = u % per * 8;
            if (u < units) rotate<BF16, 8>(a.rope, a.q, (first + t) * a.q_stride + head, c, lo + (int32_t)t, a.vec & 4, a.even, x[i]);
        }
        __syncthreads();  // q_out may be q: a pair's other half is read by another thread, before anything is stored
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            const uint32_t u = tid + i * 256, t = u / per, c = u % per * 8;
            if (u < units) store_run<BF16, 8>(a.q_out, (first + t) * a.q_out_stride + head + c, a.vec & 8, x[i]);
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
    const bool old = lo > max(p0, own);  // the block holds tokens of earlier calls
    const float held = old ? *scale_at : KV_SCALE_MIN;

    double top = 0.0;
    RopeView none{};
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const uint32_t u = tid + i * 256;
        if (u < units) {
            const uint32_t t = u / per, c = u % per * 8;
            if (values) rotate<BF16, 8>(none, a.v, (first + t) * a.v_stride + (size_t)head * d, c, 0, a.vec & 2, true, x[i]);
            else rotate<BF16, 8>(a.rope, a.k, (first + t) * a.k_stride + (size_t)head * d, c, lo + (int32_t)t, a.vec & 1, a.even, x[i]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[i][j] = storable(x[i][j]);
                top = fmax(top, fabs(x[i][j]));
            }
        }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) top = fmax(top, __shfl_xor(top, m));
    if ((tid & 63) == 0) top_s[tid >> 6] = top;
    __syncthreads();
    top = fmax(fmax(top_s[0], top_s[1]), fmax(top_s[2], top_s[3]));
    const float was = sound_scale(held), scale = grown_scale(was, top);
    const bool rescale = old && scale != was;
    const bool whole = rescale || hi - lo > 8;  // the block goes out through its image
    if (whole && old) {
        const float ratio = was / scale;
        for (uint32_t i = tid; i < KV_BLOCK * d / 16; i += 256) {
            const uint4 u = *reinterpret_cast<const uint4*>(codes + 16 * i);
            uint32_t w[4] = {u.x, u.y, u.z, u.w};
            if (rescale) {
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] = rescaled(w[k], ratio);
            }
            *reinterpret_cast<uint4*>(image + 16 * i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
    }
    const double inv = 1.0 / (double)scale;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const uint32_t u = tid + i * 256;
        if (u >= units) continue;
        const uint32_t t = (uint32_t)(lo - p0) + u / per, c = u % per * 8;
        uint32_t code[8];
#pragma unroll
        for (int j = 0; j < 8; j++) code[j] = code_of(x[i][j], scale, inv);
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
    // a block without older tokens: what lies behind the last new one is nobody's yet, and becomes zeros (so do the places in front of the sequence's first own token)
    for (uint32_t i = tid; i < KV_BLOCK * d / 16; i += 256) {
        uint4 u = *reinterpret_cast<const uint4*>(image + 16 * i);
        if (hi - lo < (int32_t)KV_BLOCK) {
            const uint32_t g = i * 16 % 1024 / 256, n = i % 16;
            uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (uint32_t k = 0; k < 16; k++) {
                const uint32_t t = values ? k % 8 / 4 * 16 + 4 * g + k % 4 : k / 8 * 16 + n;
                if (t >= (uint32_t)(hi - p0) || (SHARED && t < (uint32_t)(lo - p0))) w[k / 4] = (w[k / 4] & ~(0xFFu << (8 * (k % 4)))) | 128u << (8 * (k % 4));
            }
            u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(codes + 16 * i) = u;
    }
}

// The same for one new token a sequence (row_start NULL): a wave takes one head's keys, values or query, four channels a lane, and needs no other
// wave. A step of 64 sequences, 32 query heads over 8 of 128 channels: 11.9 us with the kernel above, a workgroup to a head, 5.7 here.
template <bool BF16, bool SHARED>
__global__ __launch_bounds__(256) void kv_append_step_kernel(AppendArgs a) {
    const uint32_t d = a.kv.d, lane = threadIdx.x & 63, c = 4 * lane;
    const uint32_t task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), s = task / a.tasks, what = task % a.tasks;  // (a sequence's heads: keys, values, queries)
    if (s >= a.b.n_seqs) return;
    const bool live = c < d;
    const bool key = what < a.kv.n_kv, query = what >= 2 * a.kv.n_kv;
    const uint32_t head = query ? what - 2 * a.kv.n_kv : key ? what : what - a.kv.n_kv;
    // what the arrays of the batch say is on its way while the values come
    const int32_t len = a.b.kv_len[s];
    const KvSeq q = kv_part((int32_t)s, (int32_t)s, (int32_t)s + 1, len, a.b.rows, a.b.max_pages, a.kv.shift);
    const int32_t pos = q.len - 1;
    double x[4] = {0.0, 0.0, 0.0, 0.0};
    if (live) {
        RopeView none{};
        if (query) rotate<BF16, 4>(a.rope, a.q, (size_t)s * a.q_stride + (size_t)head * d, c, pos, a.vec & 4, a.even, x);
        else if (key) rotate<BF16, 4>(a.rope, a.k, (size_t)s * a.k_stride + (size_t)head * d, c, pos, a.vec & 1, a.even, x);
        else rotate<BF16, 4>(none, a.v, (size_t)s * a.v_stride + (size_t)head * d, c, 0, a.vec & 2, true, x);
    }
    if (pos < 0) return;
    if (query) {
        // (q_out may be q: a pair's other half was read by another lane of this wave, before)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (live) store_run<BF16, 4>(a.q_out, (size_t)s * a.q_out_stride + (size_t)head * d + c, a.vec & 8, x);
        return;
    }
    int32_t own = 0;
    if constexpr (SHARED) {
        own = first_own(a.shared, (int32_t)s);
        if (pos < own) return;
    }
    const uint32_t block = (uint32_t)pos / KV_BLOCK, t = (uint32_t)pos % KV_BLOCK;
    const bool old = t && (!SHARED || pos > own);  // the block holds tokens of earlier calls
    const int32_t page = kv_page(a.b, a.kv, (int32_t)s, block);
    if (page < 0) return;
    const size_t index = kv_block_index(a.kv, page, head, block);
    uint8_t* codes = (key ? a.kv.k : a.kv.v) + index * KV_BLOCK * d;
    float* scale_at = (key ? a.kv.k_scale : a.kv.v_scale) + index;
    const float was = old ? sound_scale(*scale_at) : KV_SCALE_MIN;
    double top = 0.0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[j] = storable(x[j]);
        top = fmax(top, fabs(x[j]));
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) top = fmax(top, __shfl_xor(top, m));
    const float scale = grown_scale(was, top);
    if (old && scale != was) {  // the codes that are there, first
        for (uint32_t i = lane; i < KV_BLOCK * d / 16; i += 64) {
            uint4 u = *reinterpret_cast<const uint4*>(codes + 16 * i);
            const float ratio = was / scale;
            u.x = rescaled(u.x, ratio);
            u.y = rescaled(u.y, ratio);
            u.z = rescaled(u.z, ratio);
            u.w = rescaled(u.w, ratio);
            *reinterpret_cast<uint4*>(codes + 16 * i) = u;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the token's own bytes go there behind them)
    }
    if (lane == 0 && (!old || scale != was)) *scale_at = scale;
    if (!live) return;
    const double inv = 1.0 / (double)scale;
    uint32_t code[4];
#pragma unroll
    for (int j = 0; j < 4; j++) code[j] = code_of(x[j], scale, inv);
    if (key) {
        *reinterpret_cast<uint32_t*>(codes + kv_key_offset(t, c)) = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
    } else {
        uint8_t* to = codes + kv_value_offset(t, c);
#pragma unroll
        for (int j = 0; j < 4; j++) to[16 * j] = (uint8_t)code[j];
    }
}

struct ReadArgs {
    KvView kv;
    KvBatchView b;
    void *k_out, *v_out;
    int32_t count;
    uint32_t blocks;  // of a sequence's places, whole or in part
    uint32_t vec;     // k_out and v_out by 16 bytes
};

// The values that the last `count` tokens of every sequence stand for, [sequence][token][head][d]: a block's part of them per workgroup
// (blockIdx.y: the head's keys, then the head's values). The block goes through LDS, so that whole rows are written: keys lie there by octets of
// channels (264 bytes each, an odd number of 8-byte banks), values by KiB as in the cache (1056 bytes), which lets the lanes of a token's
// channels read from banks of their own. Places before a sequence's first token are zeros, those of a page that the table does not name
// NaN. The bound is memory: a byte read, an f32 (or bf16) written.
template <bool BF16>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a) {
    __shared__ __align__(16) uint8_t image[KV_MAX_D / 8 * 264];
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
    const int32_t page = block >= 0 ? kv_page(a.b, a.kv, s, (uint32_t)block) : -1;
    float scale = block >= 0 ? __builtin_nanf("") : 0.0f;
    if (page >= 0) {
        const size_t index = kv_block_index(a.kv, page, head, (uint32_t)block);
        const uint8_t* codes = (values ? a.kv.v : a.kv.k) + index * KV_BLOCK * d;
        scale = (values ? a.kv.v_scale : a.kv.k_scale)[index];
        for (uint32_t i = tid; i < 2 * d; i += 256) {
            const uint4 u = *reinterpret_cast<const uint4*>(codes + 16 * i);
            if (values) {
                *reinterpret_cast<uint4*>(image + i / 64 * 1056 + i % 64 * 16) = u;
            } else {
                uint8_t* to = image + i / 16 * 264 + i % 16 * 8;
                *reinterpret_cast<uint2*>(to) = make_uint2(u.x, u.y);
                *reinterpret_cast<uint2*>(to + 128) = make_uint2(u.z, u.w);
            }
        }
    }
    __syncthreads();
    const uint32_t per = d / 4, many = (uint32_t)(hi - lo) * per;  // four channels a thread
    const size_t row = (size_t)a.kv.n_kv * d, base = ((size_t)s * a.count + (size_t)(lo - start)) * row + (size_t)head * d;
    for (uint32_t u = tid; u < many; u += 256) {
        const uint32_t r = divide(u, per), c = (u - r * per) * 4, t = (uint32_t)(lo - p0) + r;
        uint32_t code[4];
        if (values) {
            const uint8_t* from = image + c / 32 * 1056 + t % 16 / 4 * 256 + c % 16 * 16 + c % 32 / 16 * 8 + t / 16 * 4 + t % 4;
#pragma unroll
            for (int j = 0; j < 4; j++) code[j] = from[16 * j];
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(image + c / 8 * 264 + t * 8 + c % 8);
#pragma unroll
            for (int j = 0; j < 4; j++) code[j] = (w >> (8 * j)) & 0xFF;
        }
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x = page >= 0 ? ((float)code[j] - 128.0f) * scale : scale;
            w[j] = BF16 ? f32_to_bf16_bits(x) : __float_as_uint(x);
        }
        const size_t to = base + r * row + c;
        if constexpr (BF16) {
            uint16_t* o = static_cast<uint16_t*>(out) + to;
            if (a.vec) stream_out(o, make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16));
            else o[0] = (uint16_t)w[0], o[1] = (uint16_t)w[1], o[2] = (uint16_t)w[2], o[3] = (uint16_t)w[3];
        } else {
            uint32_t* o = static_cast<uint32_t*>(out) + to;
            if (a.vec) stream_out(o, make_uint4(w[0], w[1], w[2], w[3]));
            else o[0] = w[0], o[1] = w[1], o[2] = w[2], o[3] = w[3];
        }
    }
}

hipError_t launch_kv_append(const KvView& kv, const KvBatchView& b, const SharedView& shared, const RopeView& rope, const void* k, size_t k_stride, const void* v, size_t v_stride, const void* q,
                            size_t q_stride, void* q_out, size_t q_out_stride, uint32_t n_q, bool bf16, hipStream_t s) {
    AppendArgs a{kv, b, rope, k, v, q, q_out, k_stride, v_stride, q_stride, q_out_stride, 0, 0, 2 * kv.n_kv + n_q, shared};
    const size_t size = bf16 ? 2 : 4;
    auto vec = [&](const void* p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
    a.vec = (vec(k, k_stride) ? 1u : 0u) | (vec(v, v_stride) ? 2u : 0u) | (vec(q, q_stride) ? 4u : 0u) | (vec(q_out, q_out_stride) ? 8u : 0u);
    a.even = rope.half % 8 == 0;
    if (!b.row_start) {
        const unsigned grid = (unsigned)kv_append_workgroups(false, b.rows, b.n_seqs, a.tasks);
        auto step = [&](auto kern) { kern<<<grid, 256, 0, s>>>(a); };
        if (shared.group_start) bf16 ? step(kv_append_step_kernel<true, true>) : step(kv_append_step_kernel<false, true>);
        else bf16 ? step(kv_append_step_kernel<true, false>) : step(kv_append_step_kernel<false, false>);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)kv_append_workgroups(true, b.rows, b.n_seqs, a.tasks), a.tasks);
    auto go = [&](auto kern) { kern<<<grid, 256, 0, s>>>(a); };
    auto of = [&](auto sharing) {
        constexpr bool SHARED = decltype(sharing)::value;
        if (kv.d <= 64) bf16 ? go(kv_append_kernel<true, 1, SHARED>) : go(kv_append_kernel<false, 1, SHARED>);
        else if (kv.d <= 128) bf16 ? go(kv_append_kernel<true, 2, SHARED>) : go(kv_append_kernel<false, 2, SHARED>);
        else bf16 ? go(kv_append_kernel<true, 4, SHARED>) : go(kv_append_kernel<false, 4, SHARED>);
    };
    if (shared.group_start) of(std::true_type{});
    else of(std::false_type{});
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvView& kv, const KvBatchView& b, size_t count, void* k_out, void* v_out, bool bf16, hipStream_t s) {
    const ReadArgs a{kv, b, k_out, v_out, (int32_t)count, (uint32_t)kv_read_blocks(count), (reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 == 0};
    const dim3 grid(a.blocks * b.n_seqs, 2 * kv.n_kv);
    if (bf16) kv_read_kernel<true><<<grid, 256, 0, s>>>(a);
    else kv_read_kernel<false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
