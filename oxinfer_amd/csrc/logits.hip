// What a sampler does to a row of logits before it draws: penalties for tokens that have come, biases, the tokens that a grammar allows; and
// the best token that is left.
//
// A workgroup takes a slice of a row's vocabulary, its logits in LDS. The history is read once per slice, from L2, and only its tokens that lie in
// the slice are worked on: their counters are cleared, then counted up (integer atomics, whose order does not show), then taken, by whichever
// thread comes first for a token, which applies the penalties to that logit. No table of the vocabulary's size is kept, cleared or read. Biases
// go the same way, an id's last entry being a maximum of entry numbers. The logits are read and written once, which is the bound of a batch; a
// single row is bound by the chain of its latencies.
#include "logits.hpp"

namespace oxhip {

constexpr uint32_t SEEN = 0x80000000u;  // the token occurs at all; below it, how often behind the prompt

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

// PER: logits per thread, a multiple of 4 (bf16: 8).
template <bool BF16, int PER>
__global__ __launch_bounds__(256) void logits_kernel(LogitArgs a) {
    constexpr uint32_t SLICE = 256 * PER;
    constexpr int W = BF16 ? 8 : 4;  // values of a 16-byte access
    __shared__ __align__(16) float x_s[SLICE];
    __shared__ uint32_t count[SLICE];
    __shared__ uint64_t best_s[4];
    __shared__ uint32_t last_s;
    const uint32_t tid = threadIdx.x, slice = blockIdx.x % a.slices, row = blockIdx.x / a.slices, v0 = slice * SLICE;
    const uint32_t here = min(SLICE, a.vocab - v0);
    auto at = [&](int k) { return (uint32_t)(W * (tid + (k / W) * 256) + k % W); };  // of the slice: a thread's k-th logit
    const bool counted = a.history != nullptr, biased = a.bias_start != nullptr;
    // everything that depends on nothing is asked for first
    const int32_t len = counted ? a.history_len[row] : 0, prompt = counted && a.prompt_len ? a.prompt_len[row] : 0;
    const int32_t bias0 = biased ? a.bias_start[row] : 0, bias1 = biased ? a.bias_start[row + 1] : 0;
    const float rep = counted && a.repetition ? a.repetition[row] : 1.0f, pres = counted && a.presence ? a.presence[row] : 0.0f, freq = counted && a.frequency ? a.frequency[row] : 0.0f;
    const int32_t mrow = a.allowed ? (a.allowed_row ? a.allowed_row[row] : (int32_t)row) : -1;

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
    // f(entry, its place in the slice) for the entries [from, to) of a list of ids that lie in the slice (one outside the vocabulary lies in none)
    auto each = [&](const int32_t* ids, uint32_t from, uint32_t to, auto f) {
        for (uint32_t i = from + tid; i < to; i += 4 * 256) {
            uint32_t t[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) t[k] = (uint32_t)ids[min(i + k * 256, to - 1)] - v0;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++)
                if (i + k * 256 < to && t[k] < here) f(i + k * 256, t[k]);
        }
    };
    if (counted) {
        const int32_t* h = a.history + (size_t)row * a.history_stride;
        const uint32_t n = (uint32_t)min((size_t)max(len, 0), a.history_stride), said = (uint32_t)max(prompt, 0);
        each(h, 0, n, [&](uint32_t, uint32_t t) { count[t] = 0; });
        __syncthreads();
        each(h, 0, n, [&](uint32_t i, uint32_t t) {
            if (i >= said) atomicAdd(&count[t], 1u);
            else atomicOr(&count[t], SEEN);
        });
        __syncthreads();
        each(h, 0, n, [&](uint32_t, uint32_t t) {
            const uint32_t c = atomicExch(&count[t], 0u), times = c & ~SEEN;
            if (!c) return;  // (taken)
            float v = x_s[t];
            v = v > 0.0f ? v / rep : v * rep;
            if (times) v = (v - freq * (float)times) - pres;
            x_s[t] = v;
        });
        __syncthreads();
    }
    if (biased) {
        const uint32_t b0 = (uint32_t)max(bias0, 0), b1 = min((uint32_t)max(bias1, 0), a.n_bias);
        each(a.bias_id, b0, b1, [&](uint32_t, uint32_t t) { count[t] = 0; });
        __syncthreads();
        each(a.bias_id, b0, b1, [&](uint32_t i, uint32_t t) { atomicMax(&count[t], i + 1); });
        __syncthreads();
        each(a.bias_id, b0, b1, [&](uint32_t, uint32_t t) {
            const uint32_t last = atomicExch(&count[t], 0u);
            if (last) x_s[t] = x_s[t] + a.bias[last - 1];
        });
        __syncthreads();
    }
    const bool none = mrow >= 0 && (uint32_t)mrow >= a.n_allowed;  // (a mask that is not there allows nothing)
    const uint32_t* mask = mrow >= 0 && !none ? a.allowed + (size_t)mrow * a.allowed_stride : nullptr;
    uint32_t top = 0, top_at = 0;  // the best as an ordered integer, and its number of the vocabulary
#pragma unroll
    for (int k = 0; k < PER; k += W) {
        const uint32_t i = at(k);
        if (i >= here) continue;
        const uint32_t bits = mask ? mask[(v0 + i) / 32] >> ((v0 + i) % 32) : none ? 0u : 0xFFFFFFFFu;
        if (counted || biased) {
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                const float4 f = *reinterpret_cast<const float4*>(&x_s[i + j]);
                x[k + j] = f.x; x[k + j + 1] = f.y; x[k + j + 2] = f.z; x[k + j + 3] = f.w;
            }
        }
#pragma unroll
        for (int j = 0; j < W; j++) {
            float v = x[k + j];
            if (!((bits >> j) & 1)) v = -__builtin_inff();
            if constexpr (BF16) v = bf16_bits_to_f32(f32_to_bf16_bits(v));
            const uint32_t o = i + j < here && v > -__builtin_inff() ? ordered(v) : 0u;
            if (o > top) {  // (a thread's numbers ascend: the first of equal ones stays)
                top = o;
                top_at = v0 + i + j;
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
    // the best of the slice, then of the row: the last workgroup of a row to arrive looks at all of its slices. (Best value first, then the lowest number.)
    auto meet = [&](uint32_t v, uint32_t n) {
        const uint32_t most = wave_max(v), least = ~wave_max(v == most ? ~n : 0u);
        __syncthreads();
        if ((tid & 63) == 0) best_s[tid >> 6] = (uint64_t)most << 32 | (uint32_t)~least;
        __syncthreads();
        uint64_t b = best_s[0];
#pragma unroll
        for (int w = 1; w < 4; w++) b = best_s[w] > b ? best_s[w] : b;
        return b;
    };
    uint64_t best = meet(top, top_at);
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
        best = 0;
        for (uint32_t i = tid; i < a.slices; i += 256) {
            const uint64_t o = __hip_atomic_load(&a.best[(size_t)row * a.slices + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            best = o > best ? o : best;
        }
        best = meet((uint32_t)(best >> 32), ~(uint32_t)best);
    }
    if (tid == 0) a.next[row] = best >> 32 ? (int32_t)~(uint32_t)best : -1;
}

hipError_t launch_logits(const LogitArgs& args, bool bf16, hipStream_t s) {
    LogitArgs a = args;
    const size_t size = bf16 ? 2 : 4;
    auto vec = [&](const void* p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
    a.vec = (vec(a.x, a.x_stride) ? 1u : 0u) | (vec(a.out, a.out_stride) ? 2u : 0u);
    // Slices of 4096, or of 1024 where those would leave CUs idle: one row of 128256 XONE4096 and XONE1024 us, 64 rows of 151936 XB4096 and XB1024.
    const uint32_t slice = logit_slice(a.rows, a.vocab);
    a.slices = (a.vocab + slice - 1) / slice;
    if ((uint64_t)a.slices * a.rows > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const unsigned grid = a.slices * a.rows;
    if (bf16) slice == 4096 ? logits_kernel<true, 16><<<grid, 256, 0, s>>>(a) : logits_kernel<true, 8><<<grid, 256, 0, s>>>(a);
    else slice == 4096 ? logits_kernel<false, 16><<<grid, 256, 0, s>>>(a) : logits_kernel<false, 8><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace oxhip
