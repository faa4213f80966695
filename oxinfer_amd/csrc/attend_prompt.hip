// Attention over the 8-bit cache for many rows of a sequence (attend.hip has the mathematics): what a prompt needs, bound by the matrix cores
// and by the exponentials beside them.
//
// A tile is 32 query entries (rows x heads of a group) of one key head a wave, for four or eight waves. The workgroup turns a block of 32 keys and
// values into f16 operands in LDS once for all of them, and a wave reads every operand once:
//   S^T = K Q^T    32 keys x 32 entries x 16 channels an instruction; a lane gets 16 scores of one entry
//   O^T += V^T P^T 32 channels x 32 entries x 16 keys
// The loop is a pipeline over blocks, so that matrix instructions and exponentials of one step do not wait for each other: step i multiplies
// the values of block i - 1 while it looks for the largest score of block i, then the keys of block i + 1 while it makes block i's weights; keys
// of block i + 2 and values of block i become operands meanwhile, from codes asked for two steps before.
#include <type_traits>

#include "attend.hpp"

namespace oxhip {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mma32(half8 a, half8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// Over the two lanes that hold an entry's scores, 32 apart.
__device__ __forceinline__ float half_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Two waves on a SIMD, where half of its registers hold what a wave keeps, cover each other's barriers and exponentials (a prompt of 4096 rows, 32
// heads of 128 channels over 8: one wave of 64 entries a SIMD 225 us, two of 32 in workgroups of four waves 177, of eight 157; 0.88 PFLOP/s).
// KD = d / 32; PLACES: waves on a SIMD.
template <int KD, int WAVES, int PLACES, bool F32, bool RULES>
__global__ __launch_bounds__(64 * WAVES, PLACES) void attend_prompt_kernel(AttendArgs a) {
    constexpr int THREADS = 64 * WAVES, ENTRIES = 32 * WAVES, UNITS = 4 * KD * 32, REGS = (UNITS + THREADS - 1) / THREADS;  // 16-byte units of a block's keys and values
    constexpr uint32_t d = KD * 32;
    __shared__ half8 k_s[2][KD * 2][64], v_s[2][KD * 2][64];
    __shared__ int32_t span_s[WAVES][3];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5, g = a.g;
    const uint32_t kvh = blockIdx.x % a.kv.n_kv, place = blockIdx.x / a.kv.n_kv;

    const int32_t s = kv_find(a.b, place, g, ENTRIES, 1);
    const KvSeq seq = kv_seq(a.b, s, a.kv.shift);
    const uint64_t entries = (uint64_t)(uint32_t)seq.n * g;
    const uint32_t tiles = (uint32_t)((entries + ENTRIES - 1) / ENTRIES);
    const int64_t at_place = (int64_t)place - (int64_t)kv_first_place((uint64_t)(uint32_t)max(a.b.row_start[s], 0) * g, s, ENTRIES, 1);
    if (at_place < 0 || at_place >= tiles || entries < a.prompt) return;
    const uint64_t e0 = (uint64_t)(tiles - 1 - (uint32_t)at_place) * ENTRIES + wave * 32;  // (the last rows, which see most, first)

    // what the entries see: keys below `pre`, and [lo, hi)
    int32_t lo = 0, hi = 0, pre = 0;
    int32_t lo_min = INT32_MAX, hi_max = 0, lo_max = 0, hi_min = INT32_MAX, pre_max = 0;
    const uint64_t e = e0 + n;
    const bool live = e < entries;
    const uint32_t i = live ? (uint32_t)(e / g) : 0u, head = kvh * g + (live ? (uint32_t)(e - (uint64_t)i * g) : 0u);
    const size_t row = (size_t)seq.row0 + i;
    const int32_t pos = seq.len - seq.n + (int32_t)i;
    if (live) {
        hi = max(pos + 1, 0);
        if (a.window && pos >= (int32_t)a.window) lo = pos - (int32_t)a.window + 1;
        if (a.first) lo = max(lo, a.first[row]);
        if (hi <= lo) lo = hi = 0;
        if (a.prefix) pre = min(max(a.prefix[s], 0), seq.len);
        if (hi > lo) lo_min = lo;
        hi_max = hi_min = hi;
        lo_max = lo;
        pre_max = pre;
    }
    auto wave_fold = [&](int32_t v, auto f) {
        v = f(v, (int32_t)__builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false)[h ? 0 : 1]);
        v = f(v, __shfl_xor(v, 16));
        return tile_fold(v, f);
    };
    auto least = [](int32_t x, int32_t y) { return min(x, y); };
    auto most = [](int32_t x, int32_t y) { return max(x, y); };
    lo_min = wave_fold(lo_min, least);
    hi_max = wave_fold(hi_max, most);
    lo_max = wave_fold(lo_max, most);
    hi_min = wave_fold(hi_min, least);
    pre_max = wave_fold(pre_max, most);
    if (lane == 0) {
        span_s[wave][0] = lo_min;
        span_s[wave][1] = hi_max;
        span_s[wave][2] = pre_max;
    }
    // (values that no step has brought yet are multiplied with weights of zero)
    for (uint32_t x = tid; x < KD * 2 * 64; x += THREADS) v_s[1][x / 64][x % 64] = half8{0, 0, 0, 0, 0, 0, 0, 0};
    __syncthreads();
    KvSpan span;
    {
        int32_t l0 = span_s[0][0], h0 = span_s[0][1], p0 = span_s[0][2];
#pragma unroll
        for (int w = 1; w < WAVES; w++) {
            l0 = min(l0, span_s[w][0]);
            h0 = max(h0, span_s[w][1]);
            p0 = max(p0, span_s[w][2]);
        }
        span = kv_span(__builtin_amdgcn_readfirstlane(p0), __builtin_amdgcn_readfirstlane(l0), __builtin_amdgcn_readfirstlane(h0));
    }
    const uint32_t steps = span.count;

    // queries as operands, scaled to 2^14 at most
    half8 qh[KD * 2], ql[F32 ? KD * 2 : 1];
    int power;  // of their scores' factor
    {
        float v[KD * 2][8], top = 0.0f;
#pragma unroll
        for (int x = 0; x < KD * 2; x++) {
            if (live) {
                load_query<F32>(a.q, row * a.q_stride + (size_t)head * d + x * 16 + h * 8, a.vec & 1, v[x]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[x][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(v[x][j]));
        }
        top = half_max(top);
        const int down = row_power(top);
        power = a.power + down;
#pragma unroll
        for (int x = 0; x < KD * 2; x++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float q = ldexpf(v[x][j], -down);
                qh[x][j] = (_Float16)q;
                if constexpr (F32) ql[x][j] = (_Float16)(q - (float)qh[x][j]);
            }
    }
    const float slope = RULES && a.slopes && live ? a.slopes[head] * LOG2E : 0.0f, cap = a.cap * LOG2E, cap_inv = a.cap > 0.0f ? 1.0f / cap : 0.0f;

    // Where blocks lie, and their scales: 64 blocks at a time, a lane a block; past the last block, the last one again.
    int32_t where_l = -1;
    float ksc_l = 1.0f, lvs_l = 0.0f;
    float m = NO_MAX, bar;
    bool watch = false;  // a block without values is among the wave's
    auto look = [&](uint32_t from) {
        float vsc = 1.0f;
        where_l = -1;
        ksc_l = 1.0f;
        if (from + lane < steps) {
            const uint32_t blk = kv_span_block(span, from + lane);
            const int32_t page = kv_page(a.b, a.kv, s, blk);
            if (page >= 0) {
                where_l = (int32_t)kv_block_index(a.kv, page, kvh, blk);
                ksc_l = key_scale(a.kv.k_scale[where_l]) * a.scale;
                vsc = a.kv.v_scale[where_l];
            }
        }
        lvs_l = value_log(vsc);  // (log2)
        watch = watch || __builtin_amdgcn_ballot_w64(no_values(lvs_l));
        bar = bar_of(m, watch);
    };
    // A block's codes, by 16 bytes a thread: unit u of its keys, then of its values.
    uint4 raw[2][REGS];
    auto ask = [&](uint4* to, int32_t k_where, int32_t v_where) {
#pragma unroll
        for (int x = 0; x < REGS; x++) {
            const uint32_t u = min(tid + x * THREADS, (uint32_t)UNITS - 1);
            const bool values = u >= UNITS / 2;
            const uint8_t* from = (values ? a.kv.v : a.kv.k) + (size_t)(uint32_t)max(values ? v_where : k_where, 0) * (KV_BLOCK * d);
            to[x] = gload<uint4>(as_global(from) + (values ? u - UNITS / 2 : u) * 16);
        }
    };
    auto put = [&](const uint4* from, half8 (*k)[64], half8 (*v)[64]) {
#pragma unroll
        for (int x = 0; x < REGS; x++) {
            const uint32_t u = tid + x * THREADS;
            if (UNITS % THREADS && u >= (uint32_t)UNITS) continue;
            const bool values = u >= UNITS / 2;
            const uint32_t i = values ? u - UNITS / 2 : u;  // KiB i / 64, lane i % 64 = 16 g + n: operands 4 (i / 64) + g, lanes n and 16 + n
            half8* to = (values ? &v[0][0] : &k[0][0]) + (i / 16) * 32 + i % 16;
            to[0] = code_values(from[x].x, from[x].y);
            to[16] = code_values(from[x].z, from[x].w);
        }
    };
    f32x16 acc[KD], sc;
    half8 ph[2], pl[2];
    float l = 0.0f;
    ph[0] = ph[1] = half8{0, 0, 0, 0, 0, 0, 0, 0};
    if constexpr (F32) pl[0] = pl[1] = half8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < KD; c++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[c][r] = 0.0f;
    auto keys = [&](const half8 (*k)[64], f32x16& to) {
#pragma unroll
        for (int r = 0; r < 16; r++) to[r] = 0.0f;
#pragma unroll
        for (int x = 0; x < KD * 2; x++) {
            const half8 op = k[x][lane];
            to = mma32(op, qh[x], to);
            if constexpr (F32) to = mma32(op, ql[x], to);
        }
    };
    auto values = [&](const half8 (*v)[64]) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int c = 0; c < KD; c++) {
                const half8 op = v[c * 2 + u][lane];
                acc[c] = mma32(op, ph[u], acc[c]);
                if constexpr (F32) acc[c] = mma32(op, pl[u], acc[c]);
            }
    };

    if (steps) {
        // Blocks' places as scalars, for the steps ahead: keys go two blocks ahead of the values. (The lanes' 64 blocks are looked up anew as the
        // furthest of them passes a multiple of 64; what a step needs of blocks before it has in scalars by then.)
        int32_t w_next[5];   // blocks i .. i + 4
        float ks_next[5], lv_next[5];
        auto fetch = [&](uint32_t i, int32_t& w, float& ks, float& lv) {
            const uint32_t b = min(i, steps - 1);
            if ((i & 63) == 0 && i < steps) look(i);
            w = __builtin_amdgcn_readlane(where_l, b & 63);
            ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksc_l), b & 63));
            lv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs_l), b & 63));
        };
#pragma unroll
        for (uint32_t i = 0; i < 5; i++) fetch(i, w_next[i], ks_next[i], lv_next[i]);
        {
            uint4 first[REGS];
            ask(first, w_next[0], w_next[0]);
            put(first, k_s[0], v_s[0]);
            ask(first, w_next[1], w_next[0]);
            ask(raw[0], w_next[2], w_next[0]);
            ask(raw[1], w_next[3], w_next[1]);
            put(first, k_s[1], v_s[0]);
        }
        __syncthreads();
        keys(k_s[0], sc);
        __syncthreads();  // (the first step puts other keys there)
        // (two steps' code, one after the other: a copy of codes on their way from one register to another would wait for them)
        auto step = [&](uint32_t i, auto parity) {
            constexpr int odd = decltype(parity)::value;
            const int32_t k0 = (int32_t)(kv_span_block(span, i) * KV_BLOCK);
            const float lv = lv_next[0], ks = ks_next[0];
            // values of block i - 1; the step's codes (keys of block i + 2, values of block i), and the next ones on their way
            values(v_s[odd ^ 1]);
            put(raw[odd], k_s[odd], v_s[odd]);
            ask(raw[odd], w_next[4], w_next[2]);
            // the largest scores of block i
            const int32_t end = k0 + (int32_t)KV_BLOCK;
            const bool whole = (k0 >= lo_max && end <= hi_min) || end <= pre_max;
            float f = score_factor<RULES>(ks, power);
            if (w_next[0] < 0 && ((k0 < hi && end > lo) || k0 < pre)) l = __builtin_nanf("");  // no page of the cache
            if constexpr (RULES) {
#pragma unroll
                for (int r = 0; r < 16; r++) sc[r] *= f;
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int r = 0; r < 16; r++) sc[r] = cap * tanh_of(sc[r] * cap_inv);
                }
                if (a.slopes) {
                    const float far = (float)(pos - (k0 + 4 * (int32_t)h));
#pragma unroll
                    for (int r = 0; r < 16; r++) sc[r] = fmaf(-slope, fabsf(far - (float)((r >> 2) * 8 + (r & 3))), sc[r]);
                }
            }
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int32_t j = k0 + (r >> 2) * 8 + 4 * (int32_t)h + (r & 3);
                    sc[r] = (j >= lo && j < hi) || j < pre ? sc[r] : -__builtin_inff();
                }
            }
            float top = sc[0];
#pragma unroll
            for (int r = 1; r < 16; r++) top = fmaxf(top, sc[r]);
            if constexpr (!RULES) top *= f;
            float shift = lv + HEAD_ROOM - m;
            if (__builtin_amdgcn_ballot_w64(top + lv > bar)) {
                // (an entry whose own scores need it: another row's do not change a row's bits)
                const float own = half_max(top) + lv, before = m, to = own > m + (MOST_ROOM - HEAD_ROOM) ? own : m, down = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l = lowered(l, before - to);
#pragma unroll
                for (int c = 0; c < KD; c++) acc[c] *= down;
                shift = lv + HEAD_ROOM - m;
                bar = bar_of(m, watch);
                if (__builtin_amdgcn_ballot_w64(is_far(m))) {  // (the scores become exponents)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const float apart = ((RULES ? sc[r] : sc[r] * f) - m) + (lv + HEAD_ROOM), near = RULES ? sc[r] + shift : fmaf(sc[r], f, shift);
                        sc[r] = !is_far(m) ? near : apart > F16_ROOM ? F16_ROOM : apart;
                    }
                    f = 1.0f;
                    shift = 0.0f;
                }
                if (no_values(lv)) {  // (weights for the sum alone)
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        sum += __builtin_amdgcn_exp2f((RULES ? sc[r] + shift : fmaf(sc[r], f, shift)) - lv);
                        sc[r] = -__builtin_inff();
                    }
                    l += sum;
                }
            }
            // keys of block i + 1; the weights of block i
            f32x16 ahead;
            // (the wave that has matrix instructions to issue goes before the one that has exponentials)
            __builtin_amdgcn_s_setprio(1);
            keys(k_s[odd ^ 1], ahead);
            __builtin_amdgcn_s_setprio(0);
            const float unscale = __builtin_amdgcn_exp2f(-lv);
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int r = (j < 4 ? u * 4 : (u + 2) * 4) + (j & 3);  // (keys 8 u + 4 h + j, then 16 + 8 u + 4 h + j - 4: a value operand's)
                    const float p = __builtin_amdgcn_exp2f(RULES ? sc[r] + shift : fmaf(sc[r], f, shift));
                    sum += p;
                    ph[u][j] = (_Float16)p;
                    if constexpr (F32) pl[u][j] = (_Float16)(p - (float)ph[u][j]);
                }
            l += sum * unscale;
            sc = ahead;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                w_next[x] = w_next[x + 1];
                ks_next[x] = ks_next[x + 1];
                lv_next[x] = lv_next[x + 1];
            }
            fetch(i + 5, w_next[4], ks_next[4], lv_next[4]);
            __syncthreads();
        };
        for (uint32_t i = 0; i < steps; i += 2) {
            step(i, std::integral_constant<int, 0>{});
            if (i + 1 < steps) step(i + 1, std::integral_constant<int, 1>{});
        }
        values(v_s[(steps - 1) & 1]);
    }
    const float sum = half_sum(l), whole = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that sees nothing: zeros)
    if (!live) return;
    const size_t to = row * a.out_stride + (size_t)head * d;
#pragma unroll
    for (int c = 0; c < KD; c++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = acc[c][r + j] * whole;
            const size_t at = to + c * 32 + r * 2 + h * 4;
            if constexpr (F32) {
                float* p = static_cast<float*>(a.out) + at;
                if (a.vec & 2) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
                else p[0] = x[0], p[1] = x[1], p[2] = x[2], p[3] = x[3];
            } else {
                uint16_t* p = static_cast<uint16_t*>(a.out) + at;
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = f32_to_bf16_bits(x[j]);
                if (a.vec & 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
                else p[0] = (uint16_t)w[0], p[1] = (uint16_t)w[1], p[2] = (uint16_t)w[2], p[3] = (uint16_t)w[3];
            }
        }
}

template <int KD, int WAVES, bool F32, bool RULES>
static hipError_t launch_waves(const AttendArgs& a, hipStream_t s) {
    constexpr int PLACES = (F32 && KD > 4) || KD > 5 ? 1 : 2;  // waves on a SIMD: two where half of its registers do
    const uint64_t grid = kv_places((uint64_t)a.b.rows * a.g, a.b.n_seqs, 32 * WAVES, 1) * a.kv.n_kv;
    if (!kv_launch_fits(grid, 64 * WAVES)) return hipErrorInvalidValue;
    attend_prompt_kernel<KD, WAVES, (WAVES == 8 ? 2 : PLACES), F32, RULES><<<(unsigned)grid, 64 * WAVES, 0, s>>>(a);
    return hipGetLastError();
}
// Eight waves turn the codes into operands half as often as four, where their tiles still fill the chip and are filled themselves: prompts of 2048
// and 4096 rows (32 heads over 8, bf16) 68 and 187 us with four, 76 and 173 with eight; 4096 rows behind 8192 tokens 741 and 683.
template <int KD, bool F32, bool RULES>
static hipError_t launch_prompt(const AttendArgs& a, hipStream_t s) {
    const uint64_t entries = (uint64_t)a.b.rows * a.g;
    if constexpr (KD <= (F32 ? 4 : 5))
        if (entries * a.kv.n_kv >= 1024 * 128 && entries >= (uint64_t)a.b.n_seqs * 1024) return launch_waves<KD, 8, F32, RULES>(a, s);
    return launch_waves<KD, 4, F32, RULES>(a, s);
}
template <bool F32, bool RULES>
static hipError_t launch_d(const AttendArgs& a, hipStream_t s) {
    switch (a.kv.d / 32) {
        case 1: return launch_prompt<1, F32, RULES>(a, s);
        case 2: return launch_prompt<2, F32, RULES>(a, s);
        case 3: return launch_prompt<3, F32, RULES>(a, s);
        case 4: return launch_prompt<4, F32, RULES>(a, s);
        case 5: return launch_prompt<5, F32, RULES>(a, s);
        case 6: return launch_prompt<6, F32, RULES>(a, s);
        case 7: return launch_prompt<7, F32, RULES>(a, s);
        default: return launch_prompt<8, F32, RULES>(a, s);
    }
}
hipError_t launch_attend_prompt(const AttendArgs& a, bool bf16, bool rules, hipStream_t s) {
    if (bf16) return rules ? launch_d<false, true>(a, s) : launch_d<false, false>(a, s);
    return rules ? launch_d<true, true>(a, s) : launch_d<true, false>(a, s);
}

}  // namespace oxhip
