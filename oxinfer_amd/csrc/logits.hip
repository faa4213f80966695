// What a sampler does to a row of logits before it draws: penalties for tokens that have come, biases, the tokens that a grammar allows; and
// the best token that is left.
//
// A workgroup takes a slice of a row's vocabulary, its logits in LDS. The history is read once per slice, from L2, and only its tokens that lie in
// the slice are worked on: their counters are set to one, then counted up
// behind the prompt (integer atomics, whose order does not show), then taken, by whichever
// thread comes first for a token, which applies the penalties to that logit. No table of the vocabulary's size is kept, cleared or read. Biases
// go the same way, an id's last entry being a maximum of entry numbers. The logits are read and written once, which is the bound of a batch; a
// single row is bound by the chain of its latencies.
#include "logits.hpp"

namespace oxhip {

// Two f32 values as bf16 (to the nearest, halves to even), by the hardware's conversion.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, pair{(__bf16)a, (__bf16)b});
}
// An f32 as an integer in the same order; 0 and -0 alike.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
}
// The largest over a wave's lanes.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, shifted<0x111>(v));  // row_shr:1, 2, 4, 8
    v = max(v, shifted<0x112>(v));
    v = max(v, shifted<0x114>(v));
    v = max(v, shifted<0x118>(v));
    v = max(v, shifted<0x142, 0xA>(v));  // row_bcast:15, then :31
    v = max(v, shifted<0x143, 0xC>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

template <bool BF16>
__global__ __launch_bounds__(LOGIT_THREADS) void logits_kernel(LogitArgs a) {
    constexpr uint32_t SLICE = LOGIT_SLICE;
    constexpr int PER = LOGIT_SLICE / LOGIT_THREADS;
    constexpr int W = BF16 ? 8 : 4;  // values of a 16-byte access
    __shared__ __align__(16) float x_s[SLICE];
    __shared__ uint32_t count[SLICE];
    __shared__ uint64_t best_s[LOGIT_THREADS / 64];
    __shared__ uint32_t last_s;
    __shared__ uint32_t met_s[LOGIT_THREADS / 64];
    const uint32_t tid = threadIdx.x, slice = blockIdx.x / a.rows, row = blockIdx.x % a.rows, v0 = slice * SLICE;
    const uint32_t here = min(SLICE, a.vocab - v0);
    auto at = [&](int k) { return (uint32_t)(W * (tid + (k / W) * LOGIT_THREADS) + k % W); };  // of the slice: a thread's k-th logit
    const bool counted = a.history != nullptr, biased = a.bias_start != nullptr;
    // everything that depends on nothing is asked for first
    const int32_t len = counted ? a.history_len[row] : 0, prompt = counted && a.prompt_len ? a.prompt_len[row] : 0;
    const int32_t bias0 = biased ? a.bias_start[row] : 0, bias1 = biased ? a.bias_start[row + 1] : 0;
    const float rep = counted && a.repetition ? a.repetition[row] : 1.0f, pres = counted && a.presence ? a.presence[row] : 0.0f, freq = counted && a.frequency ? a.frequency[row] : 0.0f;
    const int32_t mrow = a.allowed ? (a.allowed_row ? a.allowed_row[row] : (int32_t)row) : -1;

    // the first tokens of the history, a register each: their places in the slice (one outside the vocabulary lies in no slice)
    constexpr uint32_t HELD = 8, NOWHERE = 0xFFFFFFFFu;
    const int32_t* hist = counted ? a.history + (size_t)row * a.history_stride : nullptr;
    uint32_t place[HELD];
#pragma unroll
    for (uint32_t k = 0; k < HELD; k++) place[k] = counted && tid + k * LOGIT_THREADS < a.history_stride ? (uint32_t)hist[tid + k * LOGIT_THREADS] - v0 : NOWHERE;

    float x[PER];
    const uint8_t* in = static_cast<const uint8_t*>(a.x) + ((size_t)row * a.x_stride + v0) * (BF16 ? 2 : 4);
#pragma unroll
    for (int k = 0; k < PER; k += W) {
        const uint32_t i = at(k);
        if ((a.vec & 1) && i + W <= here) {
            const uint4 u = *reinterpret_cast<const uint4*>(in + i * (BF16 ? 2 : 4));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < W; j++) x[k + j] = BF16 ? __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16) : __uint_as_float(w[j % 4]);
        } else {
#pragma unroll
            for (int j = 0; j < W; j++) {
                x[k + j] = 0.0f;
                if (i + j < here) x[k + j] = BF16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(in)[i + j]) : reinterpret_cast<const float*>(in)[i + j];
            }
        }
    }
    if (counted || biased) {
#pragma unroll
        for (int k = 0; k < PER; k += 4) *reinterpret_cast<float4*>(&x_s[at(k)]) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
    }
    // (what follows depends on what came first)
    const bool none = mrow >= 0 && (uint32_t)mrow >= a.n_allowed;  // (a mask that is not there allows nothing)
    const uint32_t* mask = mrow >= 0 && !none ? a.allowed + (size_t)mrow * a.allowed_stride : nullptr;
    uint32_t bits[PER / W];
#pragma unroll
    for (int k = 0; k < PER; k += W) {
        const uint32_t i = v0 + at(k);
        bits[k / W] = mask && at(k) < here ? mask[i / 32] >> (i % 32) : none ? 0u : 0xFFFFFFFFu;
    }
    const uint32_t b0 = (uint32_t)max(bias0, 0), b1 = biased ? min((uint32_t)max(bias1, 0), a.n_bias) : 0u;
    const bool mine = b0 + tid < b1;  // (the first biases, too)
    const uint32_t bias_place = mine ? (uint32_t)a.bias_id[b0 + tid] - v0 : NOWHERE;
    const float bias_value = mine ? a.bias[b0 + tid] : 0.0f;
    // f(place) for the history's tokens [from, to) that lie in the slice
    auto tokens = [&](uint32_t from, uint32_t to, auto f) {
#pragma unroll
        for (uint32_t k = 0; k < HELD; k++)
            if (place[k] < here && tid + k * LOGIT_THREADS >= from) f(place[k]);
        for (uint32_t i = max(from, HELD * LOGIT_THREADS) + tid; i < to; i += 4 * LOGIT_THREADS) {
            uint32_t t[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) t[k] = (uint32_t)hist[min(i + k * LOGIT_THREADS, to - 1)] - v0;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++)
                if (i + k * LOGIT_THREADS < to && t[k] < here) f(t[k]);
        }
    };
    // f(entry, its place, its value) for the biases that lie in the slice
    auto biases = [&](auto f) {
        if (bias_place < here) f(b0 + tid, bias_place, bias_value);
        for (uint32_t i = b0 + LOGIT_THREADS + tid; i < b1; i += LOGIT_THREADS) {
            const uint32_t t = (uint32_t)a.bias_id[i] - v0;
            if (t < here) f(i, t, a.bias[i]);
        }
    };
    const uint32_t n = counted ? (uint32_t)min((size_t)max(len, 0), a.history_stride) : 0u, said = min((uint32_t)max(prompt, 0), n);
    // What the slice has: bit 0 tokens of the history, bit 1 biases. Most slices have none of a few biases, and then none of their three barriers
    // (64 rows of 151936 bf16, 2000 tokens of history and up to 20 biases each: 28.2 -> 25.5 us; 25.7 with the bits always set).
    uint32_t met = 0;
    if (counted || biased) {
        bool any = n > HELD * LOGIT_THREADS;  // (those that no register holds are not looked at for this)
#pragma unroll
        for (uint32_t k = 0; k < HELD; k++) {
            place[k] = tid + k * LOGIT_THREADS < n ? place[k] : NOWHERE;
            any = any || place[k] < here;
        }
        const uint32_t flags = (__ballot(any) ? 1u : 0u) | (__ballot(bias_place < here || b1 > b0 + LOGIT_THREADS) ? 2u : 0u);
        if ((tid & 63) == 0) met_s[tid >> 6] = flags;
        tokens(0, n, [&](uint32_t t) { count[t] = 1; });
        __syncthreads();
#pragma unroll
        for (int w = 0; w < LOGIT_THREADS / 64; w++) met |= met_s[w];
        met = (uint32_t)__builtin_amdgcn_readfirstlane((int)met);
    }
    if (met & 1) {
        tokens(said, n, [&](uint32_t t) { atomicAdd(&count[t], 1u); });
        __syncthreads();
        tokens(0, n, [&](uint32_t t) {
            const uint32_t c = count[t] ? atomicExch(&count[t], 0u) : 0u;  // (most of a token's occurrences find it taken)
            if (!c) return;
            float v = x_s[t];
            v = v > 0.0f ? v / rep : v * rep;
            if (c > 1) v = (v - freq * (float)(c - 1)) - pres;
            x_s[t] = v;
        });
        __syncthreads();
    }
    if (met & 2) {
        biases([&](uint32_t, uint32_t t, float) { count[t] = 0; });
        __syncthreads();
        biases([&](uint32_t i, uint32_t t, float) { atomicMax(&count[t], i + 1); });
        __syncthreads();
        biases([&](uint32_t i, uint32_t t, float v) {
            if (count[t] == i + 1) x_s[t] = x_s[t] + v;  // (the last entry of its token)
        });
        __syncthreads();
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < PER; k += W) {
        const uint32_t i = at(k);
        if (i >= here) continue;
        if (met) {
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                const float4 f = *reinterpret_cast<const float4*>(&x_s[i + j]);
                x[k + j] = f.x; x[k + j + 1] = f.y; x[k + j + 2] = f.z; x[k + j + 3] = f.w;
            }
        }
        if constexpr (BF16) {
#pragma unroll
            for (int j = 0; j < W; j += 2) {
                const uint32_t w = bf16_pair(x[k + j], x[k + j + 1]);
                x[k + j] = __uint_as_float(w << 16);
                x[k + j + 1] = __uint_as_float(w & 0xFFFF0000u);
            }
        }
#pragma unroll
        for (int j = 0; j < W; j++) {
            if (!((bits[k / W] >> j) & 1) || (here < SLICE && i + j >= here)) x[k + j] = -__builtin_inff();
            top = fmaxf(top, x[k + j]);  // (passes NaN over)
        }
    }
    auto store = [&]() {
#pragma unroll
        for (int k = 0; k < PER; k += W) {
            const uint32_t i = at(k);
            if (i >= here) continue;
            uint8_t* to = static_cast<uint8_t*>(a.out) + ((size_t)row * a.out_stride + v0 + i) * (BF16 ? 2 : 4);
            if ((a.vec & 2) && i + W <= here) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = BF16 ? (__float_as_uint(x[k + (2 * j) % W]) >> 16) | (__float_as_uint(x[k + (2 * j + 1) % W]) & 0xFFFF0000u) : __float_as_uint(x[k + j]);
                *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int j = 0; j < W; j++)
                    if (i + j < here) {
                        if constexpr (BF16) reinterpret_cast<uint16_t*>(to)[j] = (uint16_t)(__float_as_uint(x[k + j]) >> 16);
                        else reinterpret_cast<float*>(to)[j] = x[k + j];
                    }
            }
        }
    };
    if (!a.next) {
        store();
        return;
    }
    // the best of the slice, then of the row: the last workgroup of a row to arrive looks at all of its slices. (The best value first, of equal ones the
    // lowest number; nothing is 0.)
    auto meet = [&](uint32_t v, auto number) {
        const uint32_t most = wave_max(v), lowest = most ? ~wave_max(v == most ? ~number() : 0u) : ~0u;
        __syncthreads();
        if ((tid & 63) == 0) best_s[tid >> 6] = (uint64_t)most << 32 | (uint32_t)~lowest;
        __syncthreads();
        uint64_t b = best_s[0];
#pragma unroll
        for (int w = 1; w < LOGIT_THREADS / 64; w++) b = best_s[w] > b ? best_s[w] : b;
        return b;
    };
    uint64_t best = meet(top > -__builtin_inff() ? ordered(top) : 0u, [&]() {
        uint32_t first = 0xFFFFFFFEu;
#pragma unroll
        for (int k = PER - 1; k >= 0; k--) first = at(k) < here && x[k] == top ? v0 + at(k) : first;  // (a thread's numbers ascend)
        return first;
    });
    if (a.slices > 1) {
        if (tid == 0) {
            __hip_atomic_store(&a.best[(size_t)row * a.slices + slice], best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const uint32_t seen = __hip_atomic_fetch_add(&a.counters[(size_t)row * CTR_STRIDE], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_s = seen == a.slices - 1;
            if (seen == a.slices - 1) __hip_atomic_store(&a.counters[(size_t)row * CTR_STRIDE], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (a.out) store();  // (behind the arrival, which would otherwise wait for it)
        __syncthreads();
        if (!last_s) return;
        best = 0;
        for (uint32_t i = tid; i < a.slices; i += LOGIT_THREADS) {
            const uint64_t o = __hip_atomic_load(&a.best[(size_t)row * a.slices + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            best = o > best ? o : best;
        }
        best = meet((uint32_t)(best >> 32), [&]() { return ~(uint32_t)best; });
    } else if (a.out) {
        store();
    }
    if (tid == 0) a.next[row] = best >> 32 ? (int32_t)~(uint32_t)best : -1;
}

hipError_t launch_logits(const LogitArgs& args, bool bf16, hipStream_t s) {
    LogitArgs a = args;
    const size_t size = bf16 ? 2 : 4;
    auto vec = [&](const void* p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
    a.vec = (vec(a.x, a.x_stride) ? 1u : 0u) | (vec(a.out, a.out_stride) ? 2u : 0u);
    a.slices = (uint32_t)logit_slices(a.vocab);
    const unsigned grid = a.slices * a.rows;
    if (bf16) logits_kernel<true><<<grid, LOGIT_THREADS, 0, s>>>(a);
    else logits_kernel<false><<<grid, LOGIT_THREADS, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
