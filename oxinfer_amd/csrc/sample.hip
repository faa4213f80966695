// The draw of a row's next token: of the weights w_i = exp((l_i - max l) / temperature), those that top-k, top-p and min-p leave, the first token, in the
// order of the ids, up to which they sum to more than u times their whole sum.
//
// Weights are made in f64 and kept as whole numbers of 2^-unit of the largest (44 bits for a vocabulary of 2^18): sums of them are exact whatever their order,
// so that neither the number of threads nor atomics decide a draw at a border.
#include "sample.hpp"

namespace oxhip {

constexpr uint32_t SAMPLE_THREADS = 1024, SAMPLE_BINS = 2048;
constexpr double SAMPLE_LOG2E = 1.4426950408889634074;

__device__ __forceinline__ uint32_t order_of(float x) {  // in the same order, 0 and -0 alike
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

template <class T>
__device__ __forceinline__ T wave_upto(T v) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int y = 1; y < 64; y *= 2) {
        const T o = __shfl_up(v, y);
        v += lane >= (uint32_t)y ? o : (T)0;
    }
    return v;
}

// One workgroup a row.
template <bool BF16>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_kernel(SampleArgs a) {
    constexpr uint32_t WAVES = SAMPLE_THREADS / 64;
    __shared__ uint32_t count_s[SAMPLE_BINS];
    __shared__ unsigned long long weight_s[SAMPLE_BINS], sums[WAVES], found_s[3];
    __shared__ uint32_t top_s[WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    const uint8_t* in = static_cast<const uint8_t*>(a.x) + (size_t)row * a.stride * (BF16 ? 2 : 4);
    auto logit = [&](uint32_t i) { return BF16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(in)[i]) : reinterpret_cast<const float*>(in)[i]; };
    auto each = [&](auto f) {
        for (uint32_t i = tid; i < a.vocab; i += SAMPLE_THREADS) f(i, logit(i));
    };
    const float heat = a.temperature ? a.temperature[row] : 1.0f;
    const float u = a.u[row];

    // the largest logit (NaN passed over)
    float top = -__builtin_inff();
    each([&](uint32_t, float x) { top = fmaxf(top, x); });
#pragma unroll
    for (int y = 32; y; y >>= 1) top = fmaxf(top, __shfl_xor(top, y));
    if (lane == 0) top_s[wave] = __float_as_uint(top);
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; w++) top = fmaxf(top, __uint_as_float(top_s[w]));
    if (top == -__builtin_inff()) {  // nothing to draw from
        if (tid == 0) {
            a.next[row] = -1;
            if (a.logp) a.logp[row] = -__builtin_inff();
        }
        return;
    }
    const bool greedy = !(heat > 0.0f), flat = top == __builtin_inff();
    const double by = SAMPLE_LOG2E / (double)heat;
    const uint64_t one = 1ull << a.unit;
    auto weight = [&](float x) -> uint64_t {
        if (x == top) return one;
        if (greedy || flat || !(x < top)) return 0;
        const double y = ((double)x - (double)top) * by;
        return y > -64.0 ? (uint64_t)rint(ldexp(exp2(y), (int)a.unit)) : 0;
    };
    // the first id up to which f sums to `target` and more (some does): by the waves' parts of the row, three times over
    auto first_to = [&](uint64_t target, auto f) {
        uint32_t from = 0, to = a.vocab;
        for (;;) {
            const uint32_t per = ((to - from + WAVES - 1) / WAVES + 63) / 64 * 64, b = min(from + wave * per, to), e = min(b + per, to);
            if (to - from <= 64) {  // (all waves do the same)
                const uint64_t v = from + lane < to ? f(from + lane, logit(from + lane)) : 0;
                const uint64_t m = __ballot(wave_upto((unsigned long long)v) >= target);
                return from + (m ? (uint32_t)__builtin_ctzll(m) : to - from - 1);
            }
            unsigned long long v = 0;
            for (uint32_t i = b + lane; i < e; i += 64) v += f(i, logit(i));
#pragma unroll
            for (int y = 32; y; y >>= 1) v += __shfl_xor(v, y);
            __syncthreads();
            if (lane == 0) sums[wave] = v;
            __syncthreads();
            uint32_t w = 0;
            uint64_t before = 0;
            while (w + 1 < WAVES && before + sums[w] < target) before += sums[w++];
            target -= before;
            from = min(from + w * per, to);
            to = min(from + per, to);
        }
    };
    // A limit: tokens above logit `cut` are kept, and of those at it the first `ties`.
    uint32_t cut = 0, ties = 0xFFFFFFFFu;  // (in order_of's order; 0: no limit)
    // Tightens it to the first tokens, in the order of their weights, that come to `want` (by number, or by weight); also what is kept then.
    auto narrow = [&](bool number, uint64_t want) {
        const double wide = 43.0 * (double)heat, scale = (double)(SAMPLE_BINS - 1) / wide;  // (weights of 2^-62 and more lie within 43 temperatures)
        uint32_t hi = order_of(top), shift = 0;
        uint64_t above_n = 0, above_w = 0;
        uint32_t part0 = 0, low = 0, high = 0;  // of the first level; then the range of logits left
        for (int level = 0;; level++) {
            auto part = [&](float x, uint32_t o) -> uint32_t {
                const uint32_t p = (uint32_t)fmin(((double)top - (double)x) * scale, (double)(SAMPLE_BINS - 1));
                if (level == 0) return p;
                if (p != part0 || o < low || o > high) return SAMPLE_BINS;
                return (high - o) >> shift;
            };
            for (uint32_t i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS) count_s[i] = 0, weight_s[i] = 0;
            __syncthreads();
            each([&](uint32_t, float x) {
                const uint64_t w = weight(x);
                const uint32_t o = order_of(x);
                if (!w || o < cut) return;
                const uint32_t p = part(x, o);
                if (p >= SAMPLE_BINS) return;
                atomicAdd(&count_s[p], 1u);
                atomicAdd(&weight_s[p], (unsigned long long)w);
            });
            __syncthreads();
            // (tokens at the cut before beyond its ties are in the last part alone)
            uint64_t n[2], w[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                n[j] = count_s[2 * tid + j];
                w[j] = weight_s[2 * tid + j];
            }
            const uint64_t mine = number ? n[0] + n[1] : w[0] + w[1];
            unsigned long long upto = wave_upto((unsigned long long)mine);
            if (lane == 63) sums[wave] = upto;
            if (tid == 0) found_s[0] = SAMPLE_BINS;
            __syncthreads();
            uint64_t before = (number ? above_n : above_w) + upto - mine;
            for (uint32_t v = 0; v < wave; v++) before += sums[v];
            const uint64_t m0 = number ? n[0] : w[0], m1 = number ? n[1] : w[1];
            if (before < want && before + m0 >= want) found_s[0] = 2 * tid;
            else if (before + m0 < want && before + m0 + m1 >= want) found_s[0] = 2 * tid + 1;
            __syncthreads();
            const uint32_t in = (uint32_t)found_s[0];
            if (in >= SAMPLE_BINS) return;  // all together do not come to it: no tighter limit
            // what lies above the part
            uint64_t bn = 0, bw = 0;
#pragma unroll
            for (uint32_t j = 0; j < 2; j++)
                if (2 * tid + j < in) bn += n[j], bw += w[j];
#pragma unroll
            for (int y = 32; y; y >>= 1) bn += __shfl_xor((unsigned long long)bn, y), bw += __shfl_xor((unsigned long long)bw, y);
            __syncthreads();
            if (tid == 0) found_s[1] = found_s[2] = 0;
            __syncthreads();
            if (lane == 0) {
                atomicAdd(&found_s[1], (unsigned long long)bn);
                atomicAdd(&found_s[2], (unsigned long long)bw);
            }
            __syncthreads();
            above_n += found_s[1];
            above_w += found_s[2];
            if (level == 0) {
                part0 = in;
                // logits of the part, a little more on both sides
                // (one that reaches past what f32 holds: to the end)
                const bool whole = flat || !(scale > 0.0);
                const double from = (double)top - (double)in / scale, to = (double)top - (double)(in + 1) / scale;
                const double room = 1e-6 * (fabs((double)top) + fabs(from) + fabs(to));
                high = whole || !(from + room < 3.4e38) ? hi : min(hi, order_of((float)(from + room)));
                low = whole || in + 1 == SAMPLE_BINS || !(to - room > -3.4e38) ? 0u : min(high, order_of((float)(to - room)));
            } else {
                const uint32_t h = high - (in << shift);
                low = shift && h - low >= (1u << shift) ? h - ((1u << shift) - 1) : shift ? low : h;
                high = h;
                if (!shift) {
                    cut = h;
                    const uint64_t wt = weight(of_order(h)), left = want - (number ? above_n : above_w);
                    const uint32_t t = (uint32_t)min(number ? left : (left + wt - 1) / wt, (uint64_t)0xFFFFFFFEu);
                    ties = t;
                    return;
                }
            }
            const uint32_t width = high - low;
            shift = width >= SAMPLE_BINS ? 21 - __builtin_clz(width) : 0;
            __syncthreads();
        }
    };
    // what is kept, in all
    uint32_t tie_end = 0xFFFFFFFFu;  // ids at the cut are kept up to this one
    auto settle = [&]() {
        if (cut) tie_end = first_to(ties, [&](uint32_t, float x) { return (uint64_t)(order_of(x) == cut); });
    };
    auto kept = [&](uint32_t i, float x) -> uint64_t {
        const uint32_t o = order_of(x);
        return o > cut || (o == cut && i <= tie_end) ? weight(x) : 0;
    };
    auto sum_kept = [&]() {
        unsigned long long v = 0;
        each([&](uint32_t i, float x) { v += kept(i, x); });
#pragma unroll
        for (int y = 32; y; y >>= 1) v += __shfl_xor(v, y);
        __syncthreads();
        if (lane == 0) sums[wave] = v;
        __syncthreads();
        uint64_t all = 0;
        for (uint32_t w = 0; w < WAVES; w++) all += sums[w];
        return all;
    };
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, least = a.min_p ? a.min_p[row] : 0.0f;
    if (greedy) {
        cut = order_of(top);
        ties = 1;
        settle();
    } else {
        if (k > 0) {
            narrow(true, (uint32_t)k);
            settle();
        }
        if (p < 1.0f) {
            const double want = (double)p * (double)sum_kept();
            narrow(false, max((uint64_t)ceil(want), (uint64_t)1));
            settle();
        }
    }
    const double min_weight = least > 0.0f ? fmin((double)least, 1.0) * (double)one : 0.0;
    auto left = [&](uint32_t i, float x) -> uint64_t {
        const uint64_t w = kept(i, x);
        return (double)w >= min_weight ? w : 0;
    };
    unsigned long long v = 0;
    each([&](uint32_t i, float x) { v += left(i, x); });
#pragma unroll
    for (int y = 32; y; y >>= 1) v += __shfl_xor(v, y);
    __syncthreads();
    if (lane == 0) sums[wave] = v;
    __syncthreads();
    uint64_t all = 0;
    for (uint32_t w = 0; w < WAVES; w++) all += sums[w];
    __syncthreads();
    const double share = (double)u > 0.0 ? (double)u : 0.0;
    const uint64_t target = min((uint64_t)fmin(floor(share * (double)all), 0x1p63) + 1, all);
    const uint32_t token = first_to(target, left);
    if (tid == 0) {
        a.next[row] = (int32_t)token;
        if (a.logp) a.logp[row] = (float)log((double)weight(logit(token)) / (double)all);
    }
}

hipError_t launch_sample(const SampleArgs& args, bool bf16, hipStream_t s) {
    SampleArgs a = args;
    uint32_t bits = 0;
    while (((uint64_t)1 << bits) < a.vocab) bits++;
    a.unit = 62 - bits;
    if (bf16) sample_kernel<true><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
    else sample_kernel<false><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
