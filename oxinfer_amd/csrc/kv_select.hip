// Which parts of a long cache a row's attention is to read: the mean key of every span of the cache in 8 bits, and for each row and key head the
// spans that score best.
//
// A span is a power of two of tokens of one page and key head. Its mean key m over the tokens that the cache holds of it is kept as signed bytes c with one f32
// scale, s = max |m| / 127, c = rint(m / s). A query is made bytes in the same way for the score (its scale being max |q| times the f32 nearest to 1 / 127),
//   score(span) = max over the heads of the group of (sum of products of bytes) * s_span * s_query:
// the sum is exact (int8 matrix instructions, 32-bit sums), the product of the three is formed in f64, so that which spans are chosen does not depend on the
// order of any sum. A span costs d + 4 bytes to score, 1 / (2 span) of what its keys and values take.
#include "kv.hpp"

namespace oxhip {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// f64 as an integer in the same order (0 and -0 alike), above 0; NaN is 0.
__device__ __forceinline__ uint64_t ordered(double x) {
    if (x != x) return 0;
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double unordered(uint64_t u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }

// ---- the mean keys ------------------------------------------------------------------------------------------------------------------------

// A workgroup makes one span of one key head; a wave takes 32 channels at a time: a lane has 8 of them of two tokens of a block.
__global__ __launch_bounds__(256) void kv_summarize_kernel(SummaryArgs a) {
    __shared__ double mean_s[KV_MAX_D], top_s[4];
    const uint32_t d = a.kv.d, tid = threadIdx.x, lane = tid & 63, n = lane & 15, grp = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t head = blockIdx.x % a.kv.n_kv, place = blockIdx.x / a.kv.n_kv, tokens = KV_BLOCK << a.span_shift;
    int32_t s = (int32_t)place, at = 0;
    if (a.b.row_start) {
        s = kv_find(a.b, place, 1, tokens, 2);
        at = (int32_t)(place - (uint32_t)kv_first_place((uint32_t)max(a.b.row_start[s], 0), s, tokens, 2));
    }
    const KvSeq q = kv_seq(a.b, s, a.kv.shift);
    const int64_t span = (int64_t)(max(q.len - q.n, 0) / (int32_t)tokens) + at, p0 = span * tokens;
    if (at < 0 || q.n <= 0 || p0 >= q.len) return;
    const uint32_t held = (uint32_t)min((int64_t)tokens, q.len - p0), blocks = (held + KV_BLOCK - 1) / KV_BLOCK, block0 = (uint32_t)(p0 / KV_BLOCK);
    const int32_t page = kv_page(a.b, a.kv, s, block0);
    if (page < 0) return;  // (a table that names no page of the cache: nothing is written)
    const size_t index = kv_block_index(a.kv, page, head, block0);
    for (uint32_t ks = wave; ks < d / 32; ks += 4) {
        double sum[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
        for (uint32_t blk = 0; blk < blocks; blk++) {
            const uint32_t in = min(KV_BLOCK, held - blk * KV_BLOCK);
            const uint4 u = *reinterpret_cast<const uint4*>(a.kv.k + (index + blk) * (KV_BLOCK * d) + ks * 1024 + lane * 16);
            const float scale = a.kv.k_scale[index + blk];
            // two channels' codes a register: sums over the block's tokens stay below 2^16
            const uint32_t a0 = n < in ? u.x : 0u, a1 = n < in ? u.y : 0u, b0 = 16 + n < in ? u.z : 0u, b1 = 16 + n < in ? u.w : 0u;
            uint32_t w[4] = {(a0 & 0xFF00FFu) + (b0 & 0xFF00FFu), (a0 >> 8 & 0xFF00FFu) + (b0 >> 8 & 0xFF00FFu), (a1 & 0xFF00FFu) + (b1 & 0xFF00FFu), (a1 >> 8 & 0xFF00FFu) + (b1 >> 8 & 0xFF00FFu)};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                w[j] += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[j], 0x128, 0xF, 0xF, true);  // row_ror:8, 4, 2, 1
                w[j] += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[j], 0x124, 0xF, 0xF, true);
                w[j] += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[j], 0x122, 0xF, 0xF, true);
                w[j] += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[j], 0x121, 0xF, 0xF, true);
            }
            const double by = scale < KV_SCALE_MIN ? 0.0 : (double)scale;  // (as the attention takes it)
            const int32_t off = 128 * (int32_t)in;
#pragma unroll
            for (int j = 0; j < 8; j++) sum[j] += by * (double)((int32_t)(w[j / 4 * 2 + (j & 1)] >> (j & 2 ? 16 : 0) & 0xFFFFu) - off);
        }
        if (n == 0)
#pragma unroll
            for (int j = 0; j < 8; j++) mean_s[ks * 32 + grp * 8 + j] = sum[j] / (double)held;
    }
    __syncthreads();
    double top = tid < d ? fabs(mean_s[tid]) : 0.0;
#pragma unroll
    for (int x = 32; x; x >>= 1) top = fmax(top, __shfl_xor(top, x));
    if (lane == 0) top_s[wave] = top;
    __syncthreads();
    const float scale = (float)(fmax(fmax(top_s[0], top_s[1]), fmax(top_s[2], top_s[3])) / 127.0);
    const size_t to = index >> a.span_shift;
    if (tid < d) a.code[to * d + tid] = scale > 0.0f ? (int8_t)(int)fmin(fmax(rint(mean_s[tid] / (double)scale), -127.0), 127.0) : (int8_t)0;
    if (tid == 0) a.scale[to] = scale;
}

// ---- and back -----------------------------------------------------------------------------------------------------------------------------

// Four channels a thread.
__global__ __launch_bounds__(256) void kv_summary_read_kernel(SummaryArgs a, uint32_t count, float* out) {
    const uint32_t d = a.kv.d, per = d / 4, tokens = KV_BLOCK << a.span_shift;
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x, row = id / per;  // [n_seqs][count][n_kv]
    const uint32_t head = (uint32_t)(row % a.kv.n_kv);
    const uint64_t place = row / a.kv.n_kv, s = place / count;
    if (s >= a.b.n_seqs) return;
    const KvSeq q = kv_seq(a.b, (int32_t)s, a.kv.shift);
    const int64_t span = q.len > 0 ? (int64_t)((q.len - 1) / (int32_t)tokens) + 1 + (int64_t)(place % count) - count : -1;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (span >= 0) {
        const uint32_t block = (uint32_t)span << a.span_shift;
        const int32_t page = kv_page(a.b, a.kv, (int32_t)s, block);
        const float nan = __builtin_nanf("");
        v = make_float4(nan, nan, nan, nan);
        if (page >= 0) {
            const size_t at = kv_block_index(a.kv, page, head, block) >> a.span_shift;
            const char4 c = *reinterpret_cast<const char4*>(a.code + at * d + id % per * 4);
            const float f = a.scale[at];
            v = make_float4((float)c.x * f, (float)c.y * f, (float)c.z * f, (float)c.w * f);
        }
    }
    *reinterpret_cast<float4*>(out + id * 4) = v;
}

// ---- the choice ---------------------------------------------------------------------------------------------------------------------------

constexpr uint32_t SELECT_THREADS = 512, SELECT_BINS = 1024;

// A workgroup chooses one row's spans for one key head. Scores of 16 spans x 16 heads come from d / 64 matrix instructions, spans as columns, so that a
// lane has four heads of one span; all spans' scores lie in LDS, as integers in their order. The score of the last span to be taken is then found by
// counting: how many scores fall into each of 1024 equal parts of the range from the lowest to the highest, the part that the count falls into becoming the
// range, until it holds one score alone (two or three rounds).
template <bool BF16>
__global__ __launch_bounds__(SELECT_THREADS) void kv_select_kernel(SelectArgs a) {
    extern __shared__ uint64_t score_s[];  // one of each span
    constexpr uint32_t WAVES = SELECT_THREADS / 64;
    __shared__ __align__(16) int8_t q_s[16][KV_MAX_D + 16];
    __shared__ float q_scale[16];
    __shared__ uint32_t bins[SELECT_BINS], sums[WAVES];
    __shared__ unsigned long long range[2];
    __shared__ uint32_t found[2];
    const uint32_t d = a.kv.d, tid = threadIdx.x, lane = tid & 63, n = lane & 15, grp = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t head = blockIdx.x % a.kv.n_kv, row = blockIdx.x / a.kv.n_kv, tokens = KV_BLOCK << a.span_shift;
    const int32_t s = a.b.row_start ? kv_find(a.b, row, 1, 1, 0) : (int32_t)row;
    const KvSeq q = kv_seq(a.b, s, a.kv.shift);
    const int64_t within = (int64_t)row - q.row0;
    if (within < 0 || within >= q.n) return;  // (a row behind the last sequence)
    const int32_t pos = q.len - q.n + (int32_t)within;
    int32_t* out = a.out + ((size_t)row * a.kv.n_kv + head) * a.count;
    const uint32_t spans = pos < 0 ? 0u : (uint32_t)pos / tokens + 1;
    if (spans <= a.count) {
        for (uint32_t x = tid; x < a.count; x += SELECT_THREADS) out[x] = x < spans ? (int32_t)x : -1;
        return;
    }
    for (uint32_t g0 = 0; g0 < a.g; g0 += 16) {  // 16 heads at a time
        const uint32_t heads = min(16u, a.g - g0);
        if (g0) __syncthreads();
        for (uint32_t e = wave; e < 16; e += WAVES) {
            float v[KV_MAX_D / 64];
            float top = 0.0f;
#pragma unroll
            for (uint32_t j = 0; j < KV_MAX_D / 64; j++) {
                const uint32_t c = j * 64 + lane;
                v[j] = 0.0f;
                if (e < heads && c < d) {
                    const size_t at = (size_t)row * a.q_stride + (size_t)(head * a.g + g0 + e) * d + c;
                    v[j] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(a.q)[at]) : static_cast<const float*>(a.q)[at];
                    v[j] = v[j] != v[j] ? 0.0f : fminf(fmaxf(v[j], -3.40282347e38f), 3.40282347e38f);  // (NaN counts as 0, infinity as the largest value)
                }
                top = fmaxf(top, fabsf(v[j]));
            }
#pragma unroll
            for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
            const float scale = top * (1.0f / 127.0f);
#pragma unroll
            for (uint32_t j = 0; j < KV_MAX_D / 64; j++)
                q_s[e][j * 64 + lane] = scale > 0.0f ? (int8_t)(int)fmin(fmax(rint((double)v[j] / (double)scale), -127.0), 127.0) : (int8_t)0;
            if (lane == 0) q_scale[e] = scale;
        }
        __syncthreads();
        for (uint32_t x0 = wave * 16; x0 < spans; x0 += WAVES * 16) {
            const uint32_t x = x0 + n, block = min(x, spans - 1) << a.span_shift;
            const int32_t page = kv_page(a.b, a.kv, s, block);
            const size_t at = page < 0 ? 0 : kv_block_index(a.kv, page, head, block) >> a.span_shift;
            const float scale = a.scale[at];
            i32x4 dot = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t j = 0; j < KV_MAX_D / 64; j++) {
                if (j * 64 >= d) break;
                const uint32_t c = j * 64 + grp * 16;
                i32x4 key = {0, 0, 0, 0};
                if (c < d) key = *reinterpret_cast<const i32x4*>(a.code + at * d + c);
                dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(&q_s[n][c]), key, dot, 0, 0, 0);
            }
            double best = -__builtin_inf();
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                const double y = (double)dot[r] * (double)scale * (double)q_scale[grp * 4 + r];
                if (grp * 4 + r < heads) best = best > y ? best : y;  // (a scale of NaN leaves the other heads' scores)
            }
            uint64_t u = ordered(best);
#pragma unroll
            for (int y = 16; y <= 32; y *= 2) {
                const uint64_t o = __shfl_xor((unsigned long long)u, y);
                u = o > u ? o : u;
            }
            if (page < 0) u = 0;
            if (grp == 0 && x < spans) score_s[x] = g0 && score_s[x] > u ? score_s[x] : u;
        }
    }
    __syncthreads();
    // those that are taken whatever they score are out of the count
    const uint32_t last = max(spans - a.last, a.first);  // (first + last <= count < spans)
    const uint32_t need = a.count - a.first - (spans - last);
    uint64_t lo = ~0ull, hi = 0;
    for (uint32_t x = a.first + tid; x < last; x += SELECT_THREADS) {
        lo = min(lo, score_s[x]);
        hi = max(hi, score_s[x]);
    }
    if (tid == 0) range[0] = ~0ull, range[1] = 0;
    __syncthreads();
#pragma unroll
    for (int y = 32; y; y >>= 1) {
        lo = min(lo, (uint64_t)__shfl_xor((unsigned long long)lo, y));
        hi = max(hi, (uint64_t)__shfl_xor((unsigned long long)hi, y));
    }
    if (lane == 0) {
        atomicMin(&range[0], (unsigned long long)lo);
        atomicMax(&range[1], (unsigned long long)hi);
    }
    __syncthreads();
    lo = range[0];
    hi = range[1];
    uint32_t above = 0;  // spans that score more than the range
    while (need && lo != hi) {
        // A part of the range: by value where both ends are finite values of a sum that is one too, else (and at last) by the integers themselves.
        const double top = unordered(hi), wide = top - unordered(lo), by = (double)(SELECT_BINS - 1) / wide;
        const bool values = lo && wide > 0.0 && wide < __builtin_inf() && by < __builtin_inf();
        const int shift = max(0, 54 - (int)__builtin_clzll(hi - lo));  // (by integers: 1024 parts)
        auto part = [&](uint64_t u) { return values ? min((uint32_t)((top - unordered(u)) * by), SELECT_BINS - 1) : min((uint32_t)((hi - u) >> shift), SELECT_BINS - 1); };
        for (uint32_t x = tid; x < SELECT_BINS; x += SELECT_THREADS) bins[x] = 0;
        __syncthreads();
        for (uint32_t x = a.first + tid; x < last; x += SELECT_THREADS)
            if (score_s[x] >= lo && score_s[x] <= hi) atomicAdd(&bins[part(score_s[x])], 1u);
        if (tid == 0) range[0] = ~0ull, range[1] = 0;
        __syncthreads();
        // the part that the count falls into: a thread has two
        const uint32_t b0 = bins[2 * tid], b1 = bins[2 * tid + 1];
        uint32_t upto = b0 + b1;
#pragma unroll
        for (int y = 1; y < 64; y *= 2) {
            const uint32_t o = __shfl_up(upto, y);
            upto += lane >= (uint32_t)y ? o : 0u;
        }
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        uint32_t before = above + upto - b0 - b1;
        for (uint32_t w = 0; w < wave; w++) before += sums[w];
        if (before < need && before + b0 >= need) found[0] = 2 * tid, found[1] = before;
        else if (before + b0 < need && before + b0 + b1 >= need) found[0] = 2 * tid + 1, found[1] = before + b0;
        __syncthreads();
        const uint32_t in = found[0];
        above = found[1];
        uint64_t l = ~0ull, h = 0;
        for (uint32_t x = a.first + tid; x < last; x += SELECT_THREADS)
            if (score_s[x] >= lo && score_s[x] <= hi && part(score_s[x]) == in) {
                l = min(l, score_s[x]);
                h = max(h, score_s[x]);
            }
        if (h) {
            atomicMin(&range[0], (unsigned long long)l);
            atomicMax(&range[1], (unsigned long long)h);
        } else if (l != ~0ull) {
            atomicMin(&range[0], 0ull);
        }
        __syncthreads();
        lo = range[0];
        hi = range[1];
        __syncthreads();
    }
    // The numbers, ascending: all that score more than `hi` (= lo), and the first of those that score as much.
    const uint32_t equal = need - above, per = (spans + SELECT_THREADS - 1) / SELECT_THREADS, x0 = min(tid * per, spans), x1 = min(x0 + per, spans);
    auto upto = [&](uint32_t v) {  // the sum of the threads before
        uint32_t u = v;
#pragma unroll
        for (int y = 1; y < 64; y *= 2) {
            const uint32_t o = __shfl_up(u, y);
            u += lane >= (uint32_t)y ? o : 0u;
        }
        __syncthreads();
        if (lane == 63) sums[wave] = u;
        __syncthreads();
        u -= v;
        for (uint32_t w = 0; w < wave; w++) u += sums[w];
        return u;
    };
    auto always = [&](uint32_t x) { return x < a.first || x >= last; };
    uint32_t ties = 0;
    for (uint32_t x = x0; x < x1; x++) ties += need && !always(x) && score_s[x] == hi ? 1u : 0u;
    const uint32_t ties_before = upto(ties);
    auto taken = [&](uint32_t x, uint32_t& tie) {
        if (always(x)) return true;
        if (!need) return false;
        if (score_s[x] > hi) return true;
        return score_s[x] == hi && tie++ < equal;
    };
    uint32_t tie = ties_before, many = 0;
    for (uint32_t x = x0; x < x1; x++) many += taken(x, tie) ? 1u : 0u;
    uint32_t to = upto(many);
    tie = ties_before;
    for (uint32_t x = x0; x < x1; x++)
        if (taken(x, tie)) out[to++] = (int32_t)x;
}

hipError_t launch_kv_summarize(const SummaryArgs& a, hipStream_t s) {
    const uint64_t places = a.b.row_start ? kv_places(a.b.rows, a.b.n_seqs, KV_BLOCK << a.span_shift, 2) : a.b.n_seqs;
    if (!kv_launch_fits(places * a.kv.n_kv, 256)) return hipErrorInvalidValue;
    kv_summarize_kernel<<<(unsigned)(places * a.kv.n_kv), 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_summary_read(const SummaryArgs& a, size_t count, float* out, hipStream_t s) {
    const uint64_t groups = ((uint64_t)a.b.n_seqs * count * a.kv.n_kv * (a.kv.d / 4) + 255) / 256;
    if (!kv_launch_fits(groups, 256)) return hipErrorInvalidValue;
    kv_summary_read_kernel<<<(unsigned)groups, 256, 0, s>>>(a, (uint32_t)count, out);
    return hipGetLastError();
}

hipError_t launch_kv_select(const SelectArgs& a, bool bf16, hipStream_t s) {
    const uint64_t groups = (uint64_t)a.b.rows * a.kv.n_kv, spans = ((uint64_t)a.b.max_pages << a.kv.shift) >> a.span_shift;
    if (!kv_launch_fits(groups, SELECT_THREADS) || spans > SELECT_SPANS) return hipErrorInvalidValue;
    const void* kern = bf16 ? reinterpret_cast<const void*>(kv_select_kernel<true>) : reinterpret_cast<const void*>(kv_select_kernel<false>);
    const size_t lds = spans * 8;
    if (lds > 32768) {
        const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(SELECT_SPANS * 8));
        if (e != hipSuccess) return e;
    }
    if (bf16) kv_select_kernel<true><<<(unsigned)groups, SELECT_THREADS, lds, s>>>(a);
    else kv_select_kernel<false><<<(unsigned)groups, SELECT_THREADS, lds, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
