// The draw of a row's next token: of the weights w_i = exp((l_i - max l) / temperature), those that top-k, top-p and min-p leave, the first token, in the
// order of the ids, up to which they sum to more than u times their whole sum.
//
// Weights are made in f64 and kept as whole numbers of 2^-unit of the largest (44 bits for a vocabulary of 2^18): sums of them are exact whatever their order,
// so that neither the number of workgroups nor atomics decide a draw at a border.
//
// A row is read twice. The first launch takes each slice's largest logit and counts its tokens, and their weights in f32, by steps of a quarter of
// an octave; the row's last workgroup to arrive learns from that in which step a limit falls (with top-p, whose sums are only near, in which two). The second one
// forms the weights' exact sums, for each slice, and sets the tokens of these steps apart, in the order of their ids. The third, a workgroup a row, has but these to
// look at to find the limit: a few by their ranks, many by counting them, in parts of a range that shrinks to one value. Then it knows every slice's sum of
// what is kept, the slice that the draw falls into, and reads that one again. Tokens that do not fit the room set apart for them (steps that hold much of
// the vocabulary), and rows whose weights no f32 sorts (infinite logits, temperatures at the ends of f32), are looked at where they are, by a whole row's passes. (64 rows of 151936 bf16, normal
// logits of deviation 2, top-p 0.95: 90 us; 256 of them, whose slices have room for 256 tokens each, 915.)
//
// One row of 128256 f32 takes 21.6 us (8.0 + 5.2 + 9.5 traced: chains of loads, barriers and arrivals), 64 rows of 151936 bf16, 19 MB, 47 (17.5 + 24.0 + 8.7: counting in LDS,
// the f64 series, the third launch's chain). A workgroup of 512 threads with eight logits each: of 256 with sixteen they took 24.8 and 51.2.
#include "sample.hpp"

namespace oxhip {

// (Tokens held in LDS: as many as fit beside the rest. A CU then has one of the third launch's workgroups; with 8192 two of them may meet on one, and 64 rows of
// 151936 took 49.1 us instead of 46.1.)
constexpr uint32_t SAMPLE_BINS = 2048, SAMPLE_FEW = 2048, SAMPLE_HELD = 14336, SAMPLE_WITH = 256;
constexpr uint32_t WAVES = SAMPLE_THREADS / 64;
constexpr double LOG2E_D = 1.4426950408889634074;
enum { ROW_GREEDY = 1, ROW_EMPTY = 2, ROW_WHOLE = 4, ROW_K = 8, ROW_P = 16, ROW_SUMS = 32 };

__device__ __forceinline__ uint32_t order_of(float x) {  // in the same order, 0 and -0 alike
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// A value from another lane (0 from none), and sums over a wave's lanes: up to one's own, and of all.
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T lane_of(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, true), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, true);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, true));
    }
}
template <class T>
__device__ __forceinline__ T wave_upto(T v) {
    v += lane_of<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    v += lane_of<0x112, 0xF>(v);
    v += lane_of<0x114, 0xF>(v);
    v += lane_of<0x118, 0xF>(v);
    v += lane_of<0x142, 0xA>(v);  // row_bcast:15, then :31
    v += lane_of<0x143, 0xC>(v);
    return v;
}
template <class T>
__device__ __forceinline__ T of_lane(T v, int lane) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane));
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    }
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
    return of_lane(wave_upto(v), 63);
}
template <class T>
__device__ __forceinline__ void put(T* p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T get(const T* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Whether this workgroup is the last of a row's to arrive (by all of its threads); the counter returns to zero. What the workgroups leave for each other is
// stored and read at the device's scope, and has been stored before they arrive.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, uint32_t of) {
    __shared__ uint32_t last;
    if (of == 1) return true;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t seen = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = seen == of - 1;
        if (seen == of - 1) put(counter, 0u);
    }
    __syncthreads();
    return last != 0;
}

// Eight logits from `i` on; NaN and what lies behind the row are -infinity.
template <bool BF16>
__device__ __forceinline__ void load_eight(const SampleArgs& a, uint32_t row, uint32_t i, float* v) {
    const uint8_t* p = static_cast<const uint8_t*>(a.x) + ((size_t)row * a.stride + i) * (BF16 ? 2 : 4);
    if (a.vec && i + 8 <= a.vocab) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (BF16) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        } else {
            const uint4 u2 = *reinterpret_cast<const uint4*>(p + 16);
            const uint32_t w2[4] = {u2.x, u2.y, u2.z, u2.w};
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __uint_as_float(w[j]), v[4 + j] = __uint_as_float(w2[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[j] = -__builtin_inff();
            if (i + j < a.vocab) v[j] = BF16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[j]) : reinterpret_cast<const float*>(p)[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = v[j] != v[j] ? -__builtin_inff() : v[j];
}

// A row's rules.
struct Rules {
    float heat, p, least, u;
    int32_t k;
    bool greedy;
};
__device__ __forceinline__ Rules rules_of(const SampleArgs& a, uint32_t row) {
    Rules r;
    r.heat = a.temperature ? a.temperature[row] : 1.0f;
    r.greedy = !(r.heat > 0.0f);
    r.k = a.top_k ? a.top_k[row] : 0;
    if (r.k > 0 && (uint32_t)r.k >= a.vocab) r.k = 0;  // (none: top-p then has its steps' weights, which are not summed where tokens are counted for top-k)
    r.p = a.top_p ? a.top_p[row] : 1.0f;
    r.least = a.min_p ? a.min_p[row] : 0.0f;
    r.u = a.u[row];
    return r;
}
// A logit's step, by one rounding each: the same in all launches.
__device__ __forceinline__ float step_scale(float heat) { return 5.77078016355585362f / heat; }
__device__ __forceinline__ float step_of(float x, float scale) { return floorf(x * scale); }

// Weights: 2^y of y = (l - top) log2 e / temperature, in 2^-unit. 2^y by its Taylor series around the nearest whole number, 10 terms of |f ln 2| <= 0.35: the next is 2^-42
// of it. An addition of 2^52 rounds to a whole number. Of eight logits at a time, so that the series' numbers are brought once for eight (one by one, with
// a branch each, the second launch took 26.9 us of 64 rows of 151936, so 23.9).
struct Weigher {
    double top, by;
    float top_f;
    int unit;
    bool plain;  // only the largest weigh anything
    template <int N>
    __device__ __forceinline__ void of(const float (&x)[N], uint64_t (&w)[N]) const {
        constexpr double C[11] = {1.0, 0.69314718055994531, 0.24022650695910071, 0.055504108664821580, 0.0096181291076284772, 0.0013333558146428443, 1.5403530393381609e-4,
                                  1.5252733804059840e-5, 1.3215486790144309e-6, 1.0178086009239699e-7, 7.0549116208011233e-9};  // (ln 2)^n / n!
        double f[N], s[N];
        int n[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            double y = ((double)x[j] - top) * by;
            y = y > -1000.0 ? y : -1000.0;  // (also of a product of 0 and infinity)
            const double whole = rint(y);
            f[j] = y - whole;
            n[j] = (int)whole + unit;
            s[j] = C[10];
        }
#pragma unroll
        for (int k = 9; k >= 0; k--)
#pragma unroll
            for (int j = 0; j < N; j++) s[j] = fma(s[j], f[j], C[k]);
#pragma unroll
        for (int j = 0; j < N; j++) {
            w[j] = (uint64_t)__double_as_longlong(ldexp(s[j], n[j]) + 0x1p52) & ((1ull << 52) - 1);
            if (plain || x[j] == top_f) w[j] = x[j] == top_f ? 1ull << unit : 0;
        }
    }
    __device__ __forceinline__ uint64_t operator()(float x) const {
        const float v[1] = {x};
        uint64_t w[1];
        of(v, w);
        return w[0];
    }
};
__device__ __forceinline__ Weigher weigher(const SampleArgs& a, const Rules& r, float top) {
    return Weigher{(double)top, LOG2E_D / (double)r.heat, top, (int)a.unit, r.greedy || top == __builtin_inff()};
}

// ---- the first pass -------------------------------------------------------------------------------------------------------------------------

template <bool BF16>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_scan_kernel(SampleArgs a) {
    // Tokens are counted for top-k, their weights summed for top-p alone, as whole numbers of 2^-32 of the slice's largest. (Eight sums of a step side by side: tokens are
    // many and steps few, and 64 lanes' additions to one place go one after the other. The launch takes 17 us of 64 rows of 151936, 9 where no row has a limit; with one sum of
    // a step, in f32, 69, with sixteen 66: additions of floats in LDS are slow.)
    constexpr uint32_t COPIES = 8, GROUPS = 4;
    __shared__ __align__(16) unsigned long long step_s[SAMPLE_STEPS][COPIES];
    __shared__ uint32_t sum_s[GROUPS][SAMPLE_STEPS];
    __shared__ float top_s[WAVES], best_s[SAMPLE_SLICES], down_s[SAMPLE_SLICES];
    static_assert(GROUPS * (SAMPLE_STEPS / 2) <= SAMPLE_THREADS, "two steps a thread");
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slice = blockIdx.x / a.rows, at = blockIdx.x % a.rows, row = a.row0 + at;
    const Rules r = rules_of(a, row);
    float x[8];
    load_eight<BF16>(a, row, slice * SAMPLE_SLICE + 8 * tid, x);
    auto largest = [&](float v) {
#pragma unroll
        for (int y = 32; y; y >>= 1) v = fmaxf(v, __shfl_xor(v, y));
        if (lane == 0) top_s[wave] = v;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) v = fmaxf(v, top_s[w]);
        return v;
    };
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    for (uint32_t i = 2 * tid; i < SAMPLE_STEPS * COPIES; i += 2 * SAMPLE_THREADS) *reinterpret_cast<uint4*>(&step_s[0][0] + i) = make_uint4(0, 0, 0, 0);
    top = largest(top);
    const float scale = step_scale(r.heat);
    const bool sorted = !r.greedy && scale > 1e-30f && scale < 1e30f, number = r.k > 0, limits = sorted && (number || r.p < 1.0f);
    uint32_t* steps = a.step + ((size_t)at * a.slices + slice) * SAMPLE_STEPS;
    if (limits) {
        const float high = step_of(top, scale);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float down = high - step_of(x[j], scale);  // (of infinite ones NaN or infinite)
            if (!(down < (float)SAMPLE_STEPS)) continue;
            const uint32_t w = (uint32_t)(__builtin_amdgcn_exp2f((x[j] - top) * (0.25f * scale)) * 4294967040.0f);
            atomicAdd(&step_s[(int)down][lane % COPIES], number ? 1ull : (unsigned long long)w);
        }
        __syncthreads();
        if (tid < SAMPLE_STEPS) {
            unsigned long long v = 0;
#pragma unroll
            for (uint32_t c = 0; c < COPIES; c++) v += step_s[tid][(tid + c) % COPIES];
            put(&steps[tid], number ? (uint32_t)v : __float_as_uint((float)v * 0x1p-32f));
        }
    }
    if (tid == 0) put(&a.best[(size_t)at * a.slices + slice], top);
    if (!last_to_arrive(&a.counters[at * CTR_STRIDE], a.slices)) return;

    float mine = -__builtin_inff();
    for (uint32_t s = tid; s < a.slices; s += SAMPLE_THREADS) mine = fmaxf(mine, best_s[s] = get(&a.best[(size_t)at * a.slices + s]));
    __syncthreads();
    top = largest(mine);
    SampleRow out{top, 0.0f, 0.0f, 0};
    if (top == -__builtin_inff()) out.flags = ROW_EMPTY;
    else if (r.greedy) out.flags = ROW_GREEDY;
    else if (!sorted || !(fabsf(top * scale) < 1e30f)) out.flags = ROW_WHOLE;
    else if (limits && fabsf(step_of(top, scale)) >= 0x1p23f) {
        // Steps are whole numbers below 2^23 only: past that a token's may lie some ulps of them off (2^-23 of `high`, for it and the best one together), also past the last
        // one that is counted. What weighs anything is all looked at then: neighbouring logits are a step apart and more, so that it is of few different values.
        const float high = step_of(top, scale);
        out.low = high - (float)SAMPLE_STEPS - fabsf(high) * 0x1p-21f;
        out.high = __builtin_inff();
        out.flags = (number ? ROW_K : 0u) | (r.p < 1.0f ? ROW_P : 0u);
    } else if (limits) {
        // the row's steps from the slices', which begin each at its own largest logit
        const float high = step_of(top, scale);
        for (uint32_t s = tid; s < a.slices; s += SAMPLE_THREADS) {
            down_s[s] = high - step_of(best_s[s], scale);
            best_s[s] = __builtin_amdgcn_exp2f((best_s[s] - top) * (0.25f * scale));
        }
        __syncthreads();
        const uint32_t group = tid / (SAMPLE_STEPS / 2), j0 = tid % (SAMPLE_STEPS / 2);
        if (group < GROUPS) {
            uint32_t n[2] = {0, 0};
            float m[2] = {0.0f, 0.0f};
            constexpr uint32_t AHEAD = 8;  // (slices asked for at once: they lie in memory, past the L2)
            for (uint32_t s0 = group; s0 < a.slices; s0 += GROUPS * AHEAD) {
                uint32_t v[AHEAD][2];
                auto slice_of = [&](uint32_t i) { return min(s0 + GROUPS * i, a.slices - 1); };
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; i++)
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++) {
                        const uint32_t j = j0 + h * (SAMPLE_STEPS / 2), s = slice_of(i);
                        v[i][h] = get(a.step + ((size_t)at * a.slices + s) * SAMPLE_STEPS + (j - (uint32_t)fminf(down_s[s], (float)j)));
                    }
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; i++)
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++) {
                        const bool on = s0 + GROUPS * i < a.slices && down_s[slice_of(i)] <= (float)(j0 + h * (SAMPLE_STEPS / 2));
                        n[h] += on ? v[i][h] : 0;
                        m[h] += on ? __uint_as_float(v[i][h]) * best_s[slice_of(i)] : 0.0f;
                    }
            }
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) sum_s[group][j0 + h * (SAMPLE_STEPS / 2)] = number ? n[h] : __float_as_uint(m[h]);
        }
        __syncthreads();
        if (tid < 64) {  // PER steps a lane
            constexpr uint32_t PER = SAMPLE_STEPS / 64;
            static_assert(SAMPLE_STEPS % 64 == 0, "as many steps a lane");
            uint32_t n_to[PER];  // the sums up to and with a step
            float m_to[PER];
#pragma unroll
            for (uint32_t j = 0; j < PER; j++) {
                n_to[j] = j ? n_to[j ? j - 1 : 0] : 0;
                m_to[j] = j ? m_to[j ? j - 1 : 0] : 0.0f;
#pragma unroll
                for (uint32_t g = 0; g < GROUPS; g++) {
                    n_to[j] += sum_s[g][PER * lane + j];
                    m_to[j] += __uint_as_float(sum_s[g][PER * lane + j]);
                }
            }
            const uint32_t n_before = wave_upto(n_to[PER - 1]) - n_to[PER - 1];
            const float m_before = wave_upto(m_to[PER - 1]) - m_to[PER - 1];
#pragma unroll
            for (uint32_t j = 0; j < PER; j++) {
                n_to[j] += n_before;
                m_to[j] += m_before;
            }
            const uint32_t n_all = of_lane(n_to[PER - 1], 63);
            const float m_all = of_lane(m_to[PER - 1], 63);
            constexpr int NONE = 100000;
            auto first = [&](auto reached) {  // the first step j with reached(j)
                int at = NONE;
#pragma unroll
                for (uint32_t j = 0; j < PER; j++) {
                    const uint64_t m = __ballot(reached(j));
                    at = min(at, m ? (int)PER * (int)__builtin_ctzll(m) + (int)j : NONE);
                }
                return at;
            };
            constexpr float NEAR = 4e-5f;  // (weights in f32, cut off at 2^-32 of a slice's largest; the slices' sums in f32)
            int k_at = NONE, p_lo = 0, p_hi = SAMPLE_STEPS - 1;
            const bool k_on = number && (uint32_t)r.k < n_all;
            if (k_on) k_at = first([&](uint32_t j) { return n_to[j] >= (uint32_t)r.k; });
            bool p_on = r.p < 1.0f;
            if (p_on && !number) {
                const float want = fmaxf(r.p, 0.0f) * m_all;
                p_lo = first([&](uint32_t j) { return m_to[j] >= want * (1.0f - NEAR); });
                p_hi = min(first([&](uint32_t j) { return m_to[j] >= want * (1.0f + NEAR); }), (int)SAMPLE_STEPS - 1);
                p_lo = min(p_lo, p_hi);
            }
            // Tokens that min-p leaves lie within so many steps of the best: limits below them are none. (Four steps for a weight of half a unit, held as one; two for both steps' roundings.)
            bool k_in = k_on;
            if (r.least > 0.0f) {
                const int reach = (int)fminf(-4.0f * __builtin_amdgcn_logf(fminf(r.least, 1.0f)) + 6.5f, 10000.0f);
                if ((!p_on || p_lo > reach) && (!k_in || k_at > reach)) p_on = k_in = false;
            }
            if (k_in || p_on) {
                int from = p_on ? p_lo : k_at, to = p_on ? p_hi : k_at;
                if (k_in && p_on) from = 0, to = k_at;  // (top-p of what top-k leaves: all of that is looked at)
                out.low = high - (float)to;
                out.high = from == 0 ? __builtin_inff() : high - (float)from;
                out.flags = (k_in ? ROW_K : 0u) | (p_on ? ROW_P : 0u) | (k_in ? 0u : ROW_SUMS);
            }
        }
    }
    if (tid == 0) a.row[at] = out;  // (for the next launch)
}

// ---- what finds a limit, and a draw ---------------------------------------------------------------------------------------------------------

struct alignas(16) DrawShared {
    union {
        unsigned long long bins[SAMPLE_BINS];
        struct {
            unsigned long long token[SAMPLE_FEW], weight[SAMPLE_FEW + 1];
            uint32_t start[SAMPLE_BINS + 1];
        } few;
    };
    unsigned long long slice[SAMPLE_SLICES], sums[WAVES], found[3];
    uint32_t offset[SAMPLE_SLICES + 1];
};

// A limit: tokens above the logit `cut` (in order_of's order; 0: no limit) are kept, and the first `ties` of those at it.
struct Cut {
    uint32_t order, ties;
    bool all_ties;  // there are no more of them
};

// The first tokens, in the order of their logits, that come to `want` by number or by weight, of the tokens that each(f) gives to f(logits, ids) by eight a thread
// (-infinity: none), those of cut.order and above, `above` lying above them all; from_v .. to_v (falling): about where their logits lie. By parts of a range of
// order_of's numbers, until a part is one number; where the range is wide, by parts of the range of the logits themselves first. False: all together do not come
// to it.
template <bool BF16, class Each>
__device__ __forceinline__ bool narrow(DrawShared& sh, const Weigher& weight, Each each, bool number, uint64_t want, uint64_t above, double from_v, double to_v, Cut& cut) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr uint32_t PER = SAMPLE_BINS / SAMPLE_THREADS, ONE = BF16 ? 16 : 0;  // (a bf16 has 16 bits: that many numbers of order_of are one value)
    const double wide = from_v - to_v, scale = wide > 0.0 && wide < 1e300 ? (double)(SAMPLE_BINS - 1) / wide : 0.0;
    const uint32_t least = cut.order;
    auto order_near = [&](double v, double room) { return v + room < -3.4e38 ? 0u : v + room > 3.4e38 ? 0xFFFFFFFFu : order_of((float)(v + room)); };
    const double room0 = 1e-6 * (fabs(from_v) + fabs(to_v));
    uint32_t low = order_near(to_v, -room0), high = order_near(from_v, room0), shift = 0, part0 = 0;
    bool values = !(high > low && (high - low) >> 22 == 0);  // (two rounds of 2048 parts of numbers do otherwise)
    bool open = !values, of_part = false;  // what lies outside of low .. high counts to its ends; only logits of the part part0 of the first round count
    auto settle = [&]() {
        const uint32_t width = high - low;
        shift = max(ONE, width >= SAMPLE_BINS ? 21u - (uint32_t)__builtin_clz(width) : 0u);
    };
    settle();
    for (;;) {
        for (uint32_t i = 2 * tid; i < SAMPLE_BINS; i += 2 * SAMPLE_THREADS) *reinterpret_cast<ulonglong2*>(&sh.bins[i]) = ulonglong2{0, 0};
        __syncthreads();
        each([&](const float (&x)[8], const uint32_t (&)[8]) {
            uint32_t p[8];
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t o = order_of(x[j]);
                uint32_t v = 0;
                if (values || of_part) {
                    const double d = (from_v - (double)x[j]) * scale;
                    v = d > 0.0 ? (uint32_t)fmin(d, (double)(SAMPLE_BINS - 1)) : 0u;
                }
                const bool out = of_part && v != part0;
                p[j] = values ? v : open ? (o >= high ? 0u : min((high - o) >> shift, SAMPLE_BINS - 1)) : out || o < low || o > high ? SAMPLE_BINS : (high - o) >> shift;
                if (o < least || !(x[j] > -__builtin_inff())) p[j] = SAMPLE_BINS;
                any = any || p[j] < SAMPLE_BINS;
            }
            if (!__ballot(any)) return;
            uint64_t w[8];
            weight.of(x, w);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (p[j] < SAMPLE_BINS && w[j]) atomicAdd(&sh.bins[p[j]], number ? 1ull : (unsigned long long)w[j]);
        });
        __syncthreads();
        unsigned long long v[PER], mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) {
            v[j] = sh.bins[PER * tid + j];
            mine += v[j];
        }
        const unsigned long long upto = wave_upto(mine);
        if (lane == 63) sh.sums[wave] = upto;
        if (tid == 0) sh.found[0] = SAMPLE_BINS;
        __syncthreads();
        uint64_t before = above + upto - mine;
        for (uint32_t w = 0; w < wave; w++) before += sh.sums[w];
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) {
            if (before < want && before + v[j] >= want) {
                sh.found[0] = PER * tid + j;
                sh.found[1] = before;
                sh.found[2] = v[j];
            }
            before += v[j];
        }
        __syncthreads();
        const uint32_t in = (uint32_t)sh.found[0];
        if (in >= SAMPLE_BINS) return false;
        above = sh.found[1];
        if (values) {
            part0 = in;
            // The logits of the part, a little more on both sides; at the ends, and where they reach past what f32 holds, to the end.
            const double from = from_v - (double)in / scale, to = from_v - (double)(in + 1) / scale, room = 1e-6 * (fabs(from_v) + fabs(from) + fabs(to));
            high = in == 0 || !(scale > 0.0) ? 0xFFFFFFFFu : order_near(from, room);
            low = in + 1 == SAMPLE_BINS || !(scale > 0.0) ? 0u : min(high, order_near(to, -room));
            values = false;
            of_part = true;
        } else {
            const uint32_t h = high - (in << shift), span = (1u << shift) - 1, l = h - low >= span || open ? h - min(h, span) : low;
            const bool end = open && (in == 0 || in + 1 == SAMPLE_BINS);
            if (shift <= ONE && !end) {
                // the one value of the part
                const uint32_t o = !BF16 ? h : h & 0x80000000u ? h & 0xFFFF0000u : ((h + 1) & 0xFFFF0000u) - 1;
                const uint64_t wt = number ? 1 : weight(of_order(o)), left = want - above;
                cut.order = o;
                cut.ties = (uint32_t)((left + wt - 1) / wt);
                cut.all_ties = cut.ties >= sh.found[2] / wt;
                return true;
            }
            low = open && in + 1 == SAMPLE_BINS ? 0u : l;
            high = open && in == 0 ? 0xFFFFFFFFu : h;
            open = false;
        }
        settle();
        __syncthreads();
    }
}

// Of the slices' sums sh.slice the slice up to which they come to `target` and more; target becomes what is left for it.
__device__ __forceinline__ uint32_t slice_of(DrawShared& sh, uint32_t slices, uint64_t& target) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t at = 0;
    uint64_t before = 0;
    for (uint32_t s0 = 0; s0 < slices; s0 += 64) {  // (all waves do the same)
        const unsigned long long v = s0 + lane < slices ? sh.slice[s0 + lane] : 0, upto = wave_upto(v);
        const uint64_t m = __ballot(before + upto >= target && s0 + lane < slices);
        if (m) {
            const int l = __builtin_ctzll(m);
            target -= before + __shfl(upto, l) - __shfl(v, l);
            return s0 + l;
        }
        before += __shfl(upto, 63);
        at = min(s0 + 63, slices - 1);
    }
    target = ~0ull;
    return at;
}
// The first id of `per` logits from i0 on up to which what f(logits, first id, values) makes of them, eight a thread at a time, sums to `target`.
template <bool BF16, class F>
__device__ __forceinline__ uint32_t id_in(const SampleArgs& a, DrawShared& sh, uint32_t row, uint32_t i0, uint32_t per, uint64_t target, F f) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t end = min(i0 + per, a.vocab);
    __syncthreads();
    if (tid == 0) sh.found[0] = end - 1;
    for (uint32_t i = i0; i < end; i += SAMPLE_SLICE) {
        float x[8];
        load_eight<BF16>(a, row, i + 8 * tid, x);
        uint64_t v[8];
        unsigned long long mine = 0;
        f(x, i + 8 * tid, v);
#pragma unroll
        for (int j = 0; j < 8; j++) mine += v[j];
        const unsigned long long upto = wave_upto(mine);
        __syncthreads();
        if (lane == 63) sh.sums[wave] = upto;
        __syncthreads();
        uint64_t before = upto - mine, all = 0;
        for (uint32_t w = 0; w < WAVES; w++) {
            if (w < wave) before += sh.sums[w];
            all += sh.sums[w];
        }
        if (all < target) {
            target -= all;
            continue;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (before < target && before + v[j] >= target) sh.found[0] = i + 8 * tid + j;
            before += v[j];
        }
        break;
    }
    __syncthreads();
    return (uint32_t)sh.found[0];
}
__device__ __forceinline__ uint64_t sum_of(DrawShared& sh, uint64_t v) {  // over the workgroup
    v = wave_sum((unsigned long long)v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.sums[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t all = 0;
    for (uint32_t w = 0; w < WAVES; w++) all += sh.sums[w];
    return all;
}
// What the random number asks for of a sum.
__device__ __forceinline__ uint64_t share_of(float u, uint64_t all) {
    const double share = u > 0.0f ? (double)u : 0.0;
    const double want = floor(share * (double)all);
    return want < (double)all ? (uint64_t)want + 1 : all;
}

// The limits of a row and its draw, by a workgroup: the tokens among which the limits fall are given by each(f), and by by_slices(sums, f), which adds f(logits, ids) up for each
// slice (all of the row's: `everything`); sh.slice has the kept weights of all
// others, by slices of `per` ids. `all` and `above`: the weights of all tokens, and of those above; n_above: the number of these.
template <bool BF16, class Each, class BySlices>
__device__ __forceinline__ bool draw(const SampleArgs& a, DrawShared& sh, uint32_t row, const Rules& r, const Weigher& weight, uint32_t flags, Each each, BySlices by_slices, bool everything, uint32_t slices, uint32_t per,
                                     uint64_t all, uint64_t above, uint32_t n_above, double from_v, double to_v) {
    const uint32_t tid = threadIdx.x;
    Cut cut{0, 0, true};
    bool limited = false;
    if (flags & ROW_GREEDY) {
        cut = Cut{order_of(weight.top_f), 1, false};
    } else {
        if (flags & ROW_K) limited = narrow<BF16>(sh, weight, each, true, (uint64_t)(uint32_t)r.k, n_above, from_v, to_v, cut);
        if (flags & ROW_P) {
            if (limited) {
                uint64_t v = 0;
                each([&](const float (&x)[8], const uint32_t (&)[8]) {
                    uint64_t w[8];
                    weight.of(x, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) v += order_of(x[j]) > cut.order ? w[j] : 0;
                });
                all = above + sum_of(sh, v) + cut.ties * weight(of_order(cut.order));
            }
            const uint64_t want = max((uint64_t)ceil(fmax((double)r.p, 0.0) * (double)all), (uint64_t)1);
            if (above >= want) return false;  // (the first launch's sums were further off than it allows for)
            if (!narrow<BF16>(sh, weight, each, false, want, above, from_v, to_v, cut) && !limited) return false;
        }
    }
    const double least = r.least > 0.0f ? fmin((double)r.least, 1.0) * (double)(1ull << a.unit) : 0.0;
    uint32_t tie_end = 0xFFFFFFFFu;  // ids at the cut are kept up to this one
    if (cut.order && !cut.all_ties) {
        unsigned long long* n = sh.bins;  // (the slices' numbers of ties, in the place of the bins)
        __syncthreads();
        for (uint32_t s = tid; s < slices; s += SAMPLE_THREADS) n[s] = 0;
        __syncthreads();
        by_slices(n, [&](const float (&x)[4], const uint32_t (&)[4]) {
            uint64_t v = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) v += order_of(x[j]) == cut.order ? 1 : 0;
            return v;
        });
        __syncthreads();
        uint64_t left = cut.ties;
        uint32_t s = 0;
        while (s + 1 < slices && n[s] < left) left -= n[s++];
        tie_end = id_in<BF16>(a, sh, row, s * per, per, left, [&](const float (&x)[8], uint32_t, uint64_t (&v)[8]) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = order_of(x[j]) == cut.order ? 1 : 0;
        });
    }
    auto left = [&](float x, uint32_t i, uint64_t w) -> uint64_t {
        const uint32_t o = order_of(x);
        return (o > cut.order || (o == cut.order && i <= tie_end)) && (double)w >= least ? w : 0;
    };
    __syncthreads();
    if (cut.order || everything || (flags & ROW_K))  // (also of a top-k past all tokens that weigh anything, which keeps those set apart)
        by_slices(sh.slice, [&](const float (&x)[4], const uint32_t (&i)[4]) {
            uint64_t w[4], v = 0;
            weight.of(x, w);
#pragma unroll
            for (int j = 0; j < 4; j++) v += left(x[j], i[j], w[j]);
            return v;
        });
    __syncthreads();
    uint64_t total = 0;
    for (uint32_t s = tid; s < slices; s += SAMPLE_THREADS) total += sh.slice[s];
    total = sum_of(sh, total);
    uint64_t target = share_of(r.u, total);
    const uint32_t s = slice_of(sh, slices, target);
    const uint32_t token = id_in<BF16>(a, sh, row, s * per, per, target, [&](const float (&x)[8], uint32_t i, uint64_t (&v)[8]) {
        weight.of(x, v);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = left(x[j], i + j, v[j]);
    });
    if (tid == 0) {
        a.next[row] = (int32_t)token;
        const uint8_t* p = static_cast<const uint8_t*>(a.x) + ((size_t)row * a.stride + token) * (BF16 ? 2 : 4);
        const float x = BF16 ? bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(p)) : *reinterpret_cast<const float*>(p);
        if (a.logp) a.logp[row] = (float)log((double)weight(x) / (double)total);
    }
    return true;
}
// The same of n tokens (order_of << 32 | id, by ids) that are all that may be kept, four a thread: by their ranks. A token's rank is the number of tokens in the higher
// ones of 2048 parts of the range top .. to_v, and of those of its own part that come before it.
template <bool BF16>
__device__ __forceinline__ void draw_few(const SampleArgs& a, DrawShared& sh, uint32_t row, const Rules& r, const Weigher& weight, uint32_t flags, const unsigned long long* tokens, uint32_t n,
                                         uint64_t all, float to_v) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr uint32_t PER = SAMPLE_FEW / SAMPLE_THREADS, BINS = SAMPLE_BINS / SAMPLE_THREADS;
    static_assert(PER == 4 && BINS == 4, "four tokens and four parts a thread");
    const float scale = (float)(SAMPLE_BINS - 1) / fmaxf(weight.top_f - to_v, 1e-30f);
    float x[PER];
    uint32_t id[PER], part[PER], slot[PER], rank[PER];
    for (uint32_t i = tid; i <= SAMPLE_BINS; i += SAMPLE_THREADS) sh.few.start[i] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
        const uint32_t k = PER * tid + j;
        const unsigned long long t = tokens[min(k, n - 1)];
        x[j] = k < n ? of_order((uint32_t)(t >> 32)) : -__builtin_inff();
        id[j] = (uint32_t)t;
        part[j] = (uint32_t)fminf((weight.top_f - x[j]) * scale, (float)(SAMPLE_BINS - 1));
        if (k < n) slot[j] = atomicAdd(&sh.few.start[part[j]], 1u);
    }
    __syncthreads();
    // sums over the workgroup, up to a thread's own
    auto upto = [&](auto v, auto& total) {
        const auto u = wave_upto(v);
        __syncthreads();
        if (lane == 63) sh.sums[wave] = u;
        __syncthreads();
        auto before = u - v;
        total = 0;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) {
            const auto s = (decltype(v))sh.sums[w];
            if (w < wave) before += s;
            total += s;
        }
        return before;
    };
    {
        uint32_t c[BINS], mine = 0, total;
#pragma unroll
        for (uint32_t j = 0; j < BINS; j++) mine += c[j] = sh.few.start[BINS * tid + j];
        uint32_t before = upto(mine, total);
#pragma unroll
        for (uint32_t j = 0; j < BINS; j++) {
            sh.few.start[BINS * tid + j] = before;
            before += c[j];
        }
        if (tid == 0) sh.few.start[SAMPLE_BINS] = n;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < PER; j++)
        if (PER * tid + j < n) sh.few.token[sh.few.start[part[j]] + slot[j]] = (unsigned long long)order_of(x[j]) << 32 | (0xFFFFFFFFu - id[j]);
    __syncthreads();
    uint64_t w[PER];
    weight.of(x, w);
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
        if (PER * tid + j >= n) continue;
        const unsigned long long mine = (unsigned long long)order_of(x[j]) << 32 | (0xFFFFFFFFu - id[j]);
        const uint32_t from = sh.few.start[part[j]], to = sh.few.start[part[j] + 1];
        rank[j] = from;
        for (uint32_t i = from; i < to; i++) rank[j] += sh.few.token[i] > mine ? 1u : 0u;
        sh.few.weight[rank[j]] = w[j];
    }
    __syncthreads();
    // the weights before each rank
    {
        unsigned long long c[PER], mine = 0, total;
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) mine += c[j] = PER * tid + j < n ? sh.few.weight[PER * tid + j] : 0;
        unsigned long long before = upto(mine, total);
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) {
            if (PER * tid + j < n) sh.few.weight[PER * tid + j] = before;
            before += c[j];
        }
        if (tid == 0) sh.few.weight[n] = total;
    }
    __syncthreads();
    const uint32_t k = flags & ROW_K ? min((uint32_t)r.k, n) : n;
    if (flags & ROW_K) all = sh.few.weight[k];
    const uint64_t want = flags & ROW_P ? max((uint64_t)ceil(fmax((double)r.p, 0.0) * (double)all), (uint64_t)1) : ~0ull;
    const double least = r.least > 0.0f ? fmin((double)r.least, 1.0) * (double)(1ull << a.unit) : 0.0;
    unsigned long long kept[PER], mine = 0, total;
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
        kept[j] = 0;
        if (PER * tid + j < n && rank[j] < k && sh.few.weight[rank[j]] < want && (double)w[j] >= least) kept[j] = w[j];
        mine += kept[j];
    }
    unsigned long long before = upto(mine, total);
    const uint64_t target = share_of(r.u, total);
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
        if (before < target && before + kept[j] >= target) {
            a.next[row] = (int32_t)id[j];
            if (a.logp) a.logp[row] = (float)log((double)kept[j] / (double)total);
        }
        before += kept[j];
    }
}

// ---- the second pass ------------------------------------------------------------------------------------------------------------------------

template <bool BF16>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_sums_kernel(SampleArgs a) {
    __shared__ unsigned long long sums_s[WAVES][3];
    __shared__ uint32_t counts_s[WAVES][2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slice = blockIdx.x / a.rows, at = blockIdx.x % a.rows, row = a.row0 + at;
    float x[8];
    load_eight<BF16>(a, row, slice * SAMPLE_SLICE + 8 * tid, x);
    const SampleRow info = a.row[at];
    const Rules r = rules_of(a, row);
    if (info.flags & (ROW_EMPTY | ROW_GREEDY | ROW_WHOLE)) return;
    const Weigher weight = weigher(a, r, info.top);
    const float scale = step_scale(r.heat);
    const bool limits = info.flags & (ROW_K | ROW_P);
    const double least = r.least > 0.0f ? fmin((double)r.least, 1.0) * (double)(1ull << a.unit) : 0.0;
    unsigned long long all = 0, above = 0, kept = 0;
    uint32_t named = 0, higher = 0;  // tokens of the thread among which the limits fall, and those above, a bit each
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float o = limits ? step_of(x[j], scale) : 0.0f;
        if (!limits || o > info.high) higher |= 1u << j;
        else if (o >= info.low) named |= 1u << j;
    }
    if (__ballot((info.flags & ROW_SUMS) || higher || named)) {
        uint64_t w[8];
        weight.of(x, w);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (!w[j]) named &= ~(1u << j);
            all += w[j];
            if (higher >> j & 1) {
                above += w[j];
                kept += (double)w[j] >= least ? w[j] : 0;
            }
        }
    }
    // (where those above are few, they are set apart with the others, if all of them fit: a row that has few of both is done by their ranks)
    if (!limits) higher = 0;
    const uint32_t n = __popc(named), n_upto = wave_upto(n), both = __popc(named | higher), both_upto = wave_upto(both);
    kept = wave_sum(kept);
    if (limits) {
        all = wave_sum(all);
        above = wave_sum(above);
    }
    if (lane == 63) {
        sums_s[wave][0] = all;
        sums_s[wave][1] = above;
        sums_s[wave][2] = kept;
        counts_s[wave][0] = both_upto;
        counts_s[wave][1] = n_upto;
    }
    __syncthreads();
    uint32_t n_both = 0, n_named = 0, both_before = 0, named_before = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) {
        if (w == wave) both_before = n_both, named_before = n_named;
        n_both += counts_s[w][0];
        n_named += counts_s[w][1];
    }
    const bool with = n_both - n_named <= SAMPLE_WITH && n_both <= a.room;
    const uint32_t set = with ? named | higher : named;
    uint32_t to = with ? both_before + both_upto - both : named_before + n_upto - n;
    const size_t place = (size_t)at * a.slices + slice;
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (set >> j & 1) {
            if (to < a.room) a.token[place * a.room + to] = (unsigned long long)order_of(x[j]) << 32 | (slice * SAMPLE_SLICE + 8 * tid + j);
            to++;
        }
    if (tid == 0) {
        SampleSlice o{0, 0, 0, (uint16_t)(n_both - n_named), (uint16_t)(with ? n_both : n_named), with};
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) {
            o.all += sums_s[w][0];
            o.above += sums_s[w][1];
            o.kept += sums_s[w][2];
        }
        a.slice[place] = o;
    }
}

// ---- the draw -------------------------------------------------------------------------------------------------------------------------------

// A workgroup a row. WHOLE: without the passes before, of a vocabulary of more slices than are kept count of.
template <bool BF16, bool WHOLE>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_pick_kernel(SampleArgs a) {
    __shared__ DrawShared sh;
    __shared__ unsigned long long held_s[WHOLE ? 1 : SAMPLE_HELD];
    __shared__ float top_s[WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, at = blockIdx.x, row = a.row0 + at;
    const Rules r = rules_of(a, row);
    SampleRow info;
    if constexpr (WHOLE) {
        float top = -__builtin_inff();
        for (uint32_t i = 8 * tid; i < a.vocab; i += SAMPLE_SLICE) {
            float x[8];
            load_eight<BF16>(a, row, i, x);
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, x[j]);
        }
#pragma unroll
        for (int y = 32; y; y >>= 1) top = fmaxf(top, __shfl_xor(top, y));
        if (lane == 0) top_s[wave] = top;
        __syncthreads();
        for (uint32_t w = 0; w < WAVES; w++) top = fmaxf(top, top_s[w]);
        info = SampleRow{top, 0.0f, 0.0f, top == -__builtin_inff() ? ROW_EMPTY : ROW_WHOLE};
    } else {
        info = a.row[at];
    }
    if (info.flags & ROW_EMPTY) {
        if (tid == 0) {
            a.next[row] = -1;
            if (a.logp) a.logp[row] = -__builtin_inff();
        }
        return;
    }
    if (!WHOLE && r.greedy) {  // the first of the best
        uint32_t from = a.slices;
        for (uint32_t s = tid; s < a.slices; s += SAMPLE_THREADS)
            if (a.best[(size_t)at * a.slices + s] == info.top) from = min(from, s);
#pragma unroll
        for (int y = 32; y; y >>= 1) from = min(from, (uint32_t)__shfl_xor(from, y));
        if (lane == 0) sh.offset[wave] = from;
        __syncthreads();
        for (uint32_t w = 0; w < WAVES; w++) from = min(from, sh.offset[w]);
        const uint32_t token = id_in<BF16>(a, sh, row, from * SAMPLE_SLICE, SAMPLE_SLICE, 1, [&](const float (&x)[8], uint32_t, uint64_t (&v)[8]) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = x[j] == info.top ? 1 : 0;
        });
        if (tid == 0) {
            a.next[row] = (int32_t)token;
            if (a.logp) a.logp[row] = 0.0f;
        }
        return;
    }
    const Weigher weight = weigher(a, r, info.top);
    uint64_t all = 0, above = 0;
    uint32_t n_above = 0, total = 0;
    bool whole = WHOLE || (info.flags & ROW_WHOLE), with = false;  // (all tokens above the limits' steps are set apart as well)
    const bool limits = info.flags & (ROW_K | ROW_P);
    const unsigned long long* tokens = a.token + (size_t)at * a.slices * a.room;
    if (!whole) {  // what the slices have, together
        bool over = false, without = false;
        for (uint32_t s = tid; s < a.slices; s += SAMPLE_THREADS) {
            const SampleSlice p = a.slice[(size_t)at * a.slices + s];
            all += p.all;
            above += p.above;
            n_above += p.n_above;
            sh.slice[s] = p.kept;
            sh.offset[s] = p.n;
            over = over || p.n > a.room;
            without = without || !p.with;
        }
        whole = __syncthreads_or(over);
        with = !__syncthreads_or(without);
        if (wave == 0) {  // the slices' tokens, one behind the other
            uint32_t from = 0;
            for (uint32_t s0 = 0; s0 < a.slices; s0 += 64) {
                const uint32_t c = s0 + lane < a.slices ? sh.offset[s0 + lane] : 0, upto = wave_upto(c);
                if (s0 + lane < a.slices) sh.offset[s0 + lane] = from + upto - c;
                from += __shfl(upto, 63);
            }
            if (lane == 0) sh.offset[a.slices] = from;
        }
        if (limits) {
            all = sum_of(sh, all);
            above = sum_of(sh, above);
            n_above = (uint32_t)sum_of(sh, n_above);
        } else {
            __syncthreads();
        }
        total = sh.offset[a.slices];
    }
    if (!whole && total <= SAMPLE_HELD) {
        for (uint32_t s = wave; s < a.slices; s += WAVES) {
            const uint32_t from = sh.offset[s], many = sh.offset[s + 1] - from;
            for (uint32_t i = lane; i < many; i += 64) held_s[from + i] = tokens[(size_t)s * a.room + i];
        }
        __syncthreads();
        if (limits && with && total <= SAMPLE_FEW) {
            draw_few<BF16>(a, sh, row, r, weight, info.flags, held_s, total, all, info.low / step_scale(r.heat));
            return;
        }
    }
    const uint32_t pieces = (a.vocab + SAMPLE_SLICE - 1) / SAMPLE_SLICE, per = WHOLE ? (pieces + SAMPLE_SLICES - 1) / SAMPLE_SLICES * SAMPLE_SLICE : SAMPLE_SLICE;
    const uint32_t slices = (uint32_t)(((uint64_t)a.vocab + per - 1) / per);
    // (tokens above the limits' steps that are set apart with them are known to be kept: their weights are in the slices' sums)
    auto token = [&](unsigned long long t, bool here, float& x, uint32_t& id) {
        x = of_order((uint32_t)(t >> 32));
        id = (uint32_t)t;
        if (!here || step_of(x, step_scale(r.heat)) > info.high) x = -__builtin_inff();
    };
    // The tokens among which the limits fall: held here, where the second pass has left them, or the whole row where it is.
    auto each = [&](auto f) {
        float x[8];
        uint32_t id[8];
        if (whole) {
            for (uint32_t p = 0; p < pieces; p++) {
                const uint32_t i = p * SAMPLE_SLICE + 8 * tid;
                load_eight<BF16>(a, row, i, x);
#pragma unroll
                for (int j = 0; j < 8; j++) id[j] = i + j;
                f(x, id);
            }
        } else if (total <= SAMPLE_HELD) {
            for (uint32_t i = 0; i < total; i += 8 * SAMPLE_THREADS) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t k = i + j * SAMPLE_THREADS + tid;
                    token(held_s[min(k, total - 1)], k < total, x[j], id[j]);
                }
                f(x, id);
            }
        } else {
            for (uint32_t s = wave; s < slices; s += WAVES) {
                const uint32_t many = sh.offset[s + 1] - sh.offset[s];
                for (uint32_t i = 0; i < many; i += 8 * 64) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t k = i + j * 64 + lane;
                        token(tokens[(size_t)s * a.room + min(k, many - 1)], k < many, x[j], id[j]);
                    }
                    f(x, id);
                }
            }
        }
    };
    auto by_slices = [&](unsigned long long* sums, auto f) {
        float x[4];
        uint32_t id[4];
        if (whole) {
            for (uint32_t p = 0; p < 2 * pieces; p++) {  // (half of what each takes at a time)
                const uint32_t i = p / 2 * SAMPLE_SLICE + 8 * tid;
                float y[8];
                load_eight<BF16>(a, row, i, y);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[j] = p & 1 ? y[4 + j] : y[j];
                    id[j] = i + (p & 1) * 4 + j;
                }
                const unsigned long long v = wave_sum((unsigned long long)f(x, id));
                if (lane == 0 && v) atomicAdd(&sums[p / 2 * SAMPLE_SLICE / per], v);
            }
        } else {
            for (uint32_t s = wave; s < slices; s += WAVES) {
                const uint32_t from = sh.offset[s], many = sh.offset[s + 1] - from;
                unsigned long long v = 0;
                for (uint32_t i = 0; i < many; i += 4 * 64) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t k = i + j * 64 + lane, at = min(k, many - 1);
                        token(total <= SAMPLE_HELD ? held_s[from + at] : tokens[(size_t)s * a.room + at], k < many, x[j], id[j]);
                    }
                    v += f(x, id);
                }
                v = wave_sum(v);
                if (lane == 0) sums[s] += v;
            }
        }
    };
    for (;;) {
        uint32_t flags = info.flags;
        // (the logits that steps `low` .. `high` stand for, falling)
        const float scale = step_scale(r.heat);
        double from_v = info.high < __builtin_inff() ? fmin((double)info.top, ((double)info.high + 1.0) / (double)scale) : (double)info.top, to_v = (double)info.low / (double)scale;
        if (whole) {
            flags = r.greedy ? ROW_GREEDY : (r.k > 0 ? ROW_K : 0u) | (r.p < 1.0f ? ROW_P : 0u);
            from_v = (double)info.top;
            to_v = from_v - 44.0 * (double)r.heat;
            __syncthreads();
            for (uint32_t s = tid; s < slices; s += SAMPLE_THREADS) sh.slice[s] = 0;
            all = above = 0;
            n_above = 0;
            if (flags & ROW_P) {
                each([&](const float (&x)[8], const uint32_t (&)[8]) {
                    uint64_t w[8];
                    weight.of(x, w);
#pragma unroll
                    for (int j = 0; j < 8; j++) all += w[j];
                });
                all = sum_of(sh, all);
            }
        }
        if (draw<BF16>(a, sh, row, r, weight, flags, each, by_slices, whole, slices, per, all, above, n_above, from_v, to_v) || whole) return;
        whole = true;
    }
}

template <bool BF16>
static hipError_t launch(SampleArgs a, const DecodeScratch& sc, hipStream_t s) {
    if (a.slices > SAMPLE_SLICES) {
        sample_pick_kernel<BF16, true><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
        return hipGetLastError();
    }
    // As many rows at a time as the scratch holds, with room for 256 tokens of a slice at least.
    constexpr size_t LEAST = SAMPLE_SLICE / 16;
    const uint32_t rows = a.rows;
    const size_t bytes = sc.partial_floats * 4, fixed = sizeof(SampleRow) + (size_t)a.slices * (SAMPLE_STEPS * 4 + sizeof(float) + sizeof(SampleSlice)) + 64;
    uint32_t most = (uint32_t)(bytes / (fixed + a.slices * LEAST * 8));
    if (most > sc.ncounters / CTR_STRIDE) most = (uint32_t)(sc.ncounters / CTR_STRIDE);
    if (!most) return hipErrorInvalidValue;
    if (most > rows) most = rows;
    const size_t room = (bytes - most * fixed) / ((size_t)most * a.slices * 8);
    a.room = (uint32_t)(room < SAMPLE_SLICE ? room : SAMPLE_SLICE);
    uint8_t* p = reinterpret_cast<uint8_t*>(sc.partial);
    auto take = [&](size_t n) {
        uint8_t* q = p;
        p += (n + 15) / 16 * 16;
        return q;
    };
    a.step = reinterpret_cast<uint32_t*>(take((size_t)most * a.slices * SAMPLE_STEPS * 4));
    a.slice = reinterpret_cast<SampleSlice*>(take((size_t)most * a.slices * sizeof(SampleSlice)));
    a.best = reinterpret_cast<float*>(take((size_t)most * a.slices * sizeof(float)));
    a.row = reinterpret_cast<SampleRow*>(take((size_t)most * sizeof(SampleRow)));
    a.token = reinterpret_cast<unsigned long long*>(p);
    a.counters = sc.counters;
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        a.rows = rows - a.row0 < most ? rows - a.row0 : most;
        sample_scan_kernel<BF16><<<a.rows * a.slices, SAMPLE_THREADS, 0, s>>>(a);
        sample_sums_kernel<BF16><<<a.rows * a.slices, SAMPLE_THREADS, 0, s>>>(a);
        sample_pick_kernel<BF16, false><<<a.rows, SAMPLE_THREADS, 0, s>>>(a);
    }
    return hipGetLastError();
}

hipError_t launch_sample(const SampleArgs& args, bool bf16, const DecodeScratch& sc, hipStream_t s) {
    SampleArgs a = args;
    uint32_t bits = 0;
    while (((uint64_t)1 << bits) < a.vocab) bits++;
    a.unit = 62 - bits < 46 ? 62 - bits : 46;
    a.slices = (a.vocab + SAMPLE_SLICE - 1) / SAMPLE_SLICE;
    a.vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.stride * (bf16 ? 2 : 4) % 16 == 0;
    return bf16 ? launch<true>(a, sc, s) : launch<false>(a, sc, s);
}

}  // namespace oxhip
