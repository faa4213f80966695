// What a sampler does to a row of logits before it draws: penalties for tokens that have come, biases, the tokens that a grammar allows; and
// the best token that is left.
//
// A workgroup takes a slice of a row's vocabulary. It counts the history's tokens of that slice in LDS (integer atomics, whose order does not
// show), keeps for each token the last bias entry that names it (a maximum of entry numbers), and then passes over the slice's logits
// once. The history is read once per slice, from L2: no table of the vocabulary's size is kept or cleared in memory. The logits are read
// and written once, which is the bound of a batch; a single row is bound by the chain of its latencies.
#include "logits.hpp"

namespace oxhip {

constexpr uint32_t SEEN = 0x80000000u;  // the token occurs at all; below it, how often behind the prompt

// An f32 as an integer in the same order; 0 and -0 alike.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}

// PER: logits per thread, a multiple of 4 (bf16: 8).
template <bool BF16, int PER>
__global__ __launch_bounds__(256) void logits_kernel(LogitArgs a) {
    constexpr uint32_t SLICE = 256 * PER;
    constexpr int W = BF16 ? 8 : 4;  // values of a 16-byte access
    __shared__ uint32_t count[SLICE], entry[SLICE];
    __shared__ uint64_t best_s[4];
    __shared__ uint32_t last_s;
    const uint32_t tid = threadIdx.x, slice = blockIdx.x % a.slices, row = blockIdx.x / a.slices, v0 = slice * SLICE;
    const uint32_t here = min(SLICE, a.vocab - v0);
    auto at = [&](int k) { return (uint32_t)(W * (tid + (k / W) * 256) + k % W); };  // of the slice: a thread's k-th logit

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
    const bool counted = a.history != nullptr, biased = a.bias_start != nullptr;
    if (counted || biased) {
        for (uint32_t i = tid; i < SLICE; i += 256) count[i] = entry[i] = 0;
        __syncthreads();
        if (counted) {
            const int32_t* h = a.history + (size_t)row * a.history_stride;
            const uint32_t n = (uint32_t)min((size_t)max(a.history_len[row], 0), a.history_stride), said = a.prompt_len ? (uint32_t)max(a.prompt_len[row], 0) : 0u;
            for (uint32_t i = tid; i < n; i += 256) {
                const uint32_t t = (uint32_t)h[i] - v0;  // (an id outside the vocabulary is in no slice)
                if (t < here) {
                    if (i >= said) atomicAdd(&count[t], 1u);
                    else atomicOr(&count[t], SEEN);
                }
            }
        }
        if (biased) {
            const uint32_t b0 = (uint32_t)max(a.bias_start[row], 0), b1 = min((uint32_t)max(a.bias_start[row + 1], 0), a.n_bias);
            for (uint32_t i = b0 + tid; i < b1; i += 256) {
                const uint32_t t = (uint32_t)a.bias_id[i] - v0;
                if (t < here) atomicMax(&entry[t], i + 1);
            }
        }
        __syncthreads();
    }
    const float rep = counted && a.repetition ? a.repetition[row] : 1.0f, pres = counted && a.presence ? a.presence[row] : 0.0f, freq = counted && a.frequency ? a.frequency[row] : 0.0f;
    const int32_t mrow = a.allowed ? (a.allowed_row ? a.allowed_row[row] : (int32_t)row) : -1;
    const bool none = mrow >= 0 && (uint32_t)mrow >= a.n_allowed;  // (a mask that is not there allows nothing)
    const uint32_t* mask = mrow >= 0 && !none ? a.allowed + (size_t)mrow * a.allowed_stride : nullptr;
    uint64_t best = 0;
#pragma unroll
    for (int k = 0; k < PER; k += W) {
        const uint32_t i = at(k);
        if (i >= here) continue;
        const uint32_t bits = mask ? mask[(v0 + i) / 32] >> ((v0 + i) % 32) : none ? 0u : 0xFFFFFFFFu;
#pragma unroll
        for (int j = 0; j < W; j++) {
            float v = x[k + j];
            if (i + j < here) {
                if (counted) {
                    const uint32_t c = count[i + j], n = c & ~SEEN;
                    if (c) v = v > 0.0f ? v / rep : v * rep;
                    if (n) v = (v - freq * (float)n) - pres;
                }
                if (biased) {
                    const uint32_t b = entry[i + j];
                    if (b) v = v + a.bias[b - 1];
                }
                if (!((bits >> j) & 1)) v = -__builtin_inff();
                if constexpr (BF16) v = bf16_bits_to_f32(f32_to_bf16_bits(v));
                if (v > -__builtin_inff()) {
                    const uint64_t key = (uint64_t)ordered(v) << 32 | (0xFFFFFFFFu - (v0 + i + j));
                    best = key > best ? key : best;
                }
            }
            x[k + j] = v;
        }
        if (a.out) {
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
    }
    if (!a.next) return;
    // the best of the slice, then of the row: the last workgroup of a row to arrive looks at all of its slices
    auto meet = [&](uint64_t b) {
#pragma unroll
        for (int m = 32; m; m >>= 1) {
            const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)b, m);
            b = o > b ? o : b;
        }
        __syncthreads();
        if ((tid & 63) == 0) best_s[tid >> 6] = b;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++) b = best_s[w] > b ? best_s[w] : b;
        return b;
    };
    best = meet(best);
    if (a.slices > 1) {
        if (tid == 0) {
            __hip_atomic_store(&a.best[(size_t)row * a.slices + slice], best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const uint32_t seen = __hip_atomic_fetch_add(&a.counters[(size_t)row * CTR_STRIDE], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_s = seen == a.slices - 1;
            if (seen == a.slices - 1) __hip_atomic_store(&a.counters[(size_t)row * CTR_STRIDE], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_s) return;
        for (uint32_t i = tid; i < a.slices; i += 256) {
            const uint64_t o = __hip_atomic_load(&a.best[(size_t)row * a.slices + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            best = o > best ? o : best;
        }
        best = meet(best);
    }
    if (tid == 0) a.next[row] = best ? (int32_t)(0xFFFFFFFFu - (uint32_t)best) : -1;
}

hipError_t launch_logits(const LogitArgs& args, bool bf16, hipStream_t s) {
    LogitArgs a = args;
    const size_t size = bf16 ? 2 : 4;
    auto vec = [&](const void* p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
    a.vec = (vec(a.x, a.x_stride) ? 1u : 0u) | (vec(a.out, a.out_stride) ? 2u : 0u);
    a.slices = (uint32_t)logit_slices(a.vocab);
    if ((uint64_t)a.slices * a.rows > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const unsigned grid = a.slices * a.rows;
    if (bf16) logits_kernel<true, 16><<<grid, 256, 0, s>>>(a);
    else logits_kernel<false, 16><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
