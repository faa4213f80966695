// Attention of many rows over chosen spans (attend_lists.hip), a wave a row and key head: short lists, so many of them that the chip is full without sharing one.
//
// A group of heads that chose together is often four or fewer, eight here at most, and a matrix instruction has 16 columns. The columns are SLOTS sets of the entries,
// each with every SLOTS-th block of the list, a maximum and a sum of its own: of SLOTS blocks a column takes the scores of its own block, so that all lanes
// make weights of scores that count (with one set, a row of 48 blocks and 3 heads spends four fifths of its exponentials on columns that are none), and the products with a
// block's values get the weights of its set alone, zeros elsewhere. The sets meet behind the last block, by lane shifts. The mathematics is attend.hip's.
//
// 1018 rows of two sequences, 48 spans of 32 each, 4 key heads of 96 with 3 heads each, f32, capped, distance bias: 115 us, 150 by attend_split.hpp's kernel. What the rows read,
// 1.1 GB, comes from the L2 (93 % hits) at 10 TB/s (the rate seen; not shown to be a limit); of about 160 vector instructions a block 96 turn codes into f16 values, for 3 entries of 16.
#include <cmath>
#include <type_traits>

#include "attend.hpp"

namespace oxhip {

constexpr uint32_t ROW_WAVES = 4;
constexpr uint32_t NOWHERE = (1u << 26) - 2;  // a block's number past any sequence's (kv_plan.hpp): none of it is seen

// Over the SLOTS lanes of an entry (16 / SLOTS apart in a row of 16).
template <int SLOTS, class F>
__device__ __forceinline__ float slots_fold(float v, F f) {
    v = f(v, __int_as_float(lanes_of<0x128>(__float_as_int(v))));  // row_ror:8, then :4
    if constexpr (SLOTS == 4) v = f(v, __int_as_float(lanes_of<0x124>(__float_as_int(v))));
    return v;
}

template <int KD, bool F32, bool RULES, int SLOTS>
__global__ __launch_bounds__(64 * ROW_WAVES, KD <= 4 ? 2 : 1) void attend_rows_kernel(AttendArgs a) {
    constexpr int PLANES = F32 ? 2 : 1, P = 16 / SLOTS;
    constexpr uint32_t d = KD * 32;
    const uint32_t lane = threadIdx.x & 63, n = lane & 15, grp = lane >> 4, slot = n / P, g = a.g;
    // Workgroups go round the eight XCDs: each takes an eighth of the units, neighbouring rows of one key head after the other, so that what these rows read of a sequence
    // finds its place in the XCD's own L2 (two sequences of 20001 tokens, 4 key heads of 96: 121 us with the heads side by side).
    const uint32_t place = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
    const uint32_t unit = place * ROW_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= a.units) return;
    const uint32_t kvh = unit / a.b.rows, row = unit - kvh * a.b.rows;
    const bool live = n % P < g;
    const uint32_t head = kvh * g + (live ? n % P : 0u);
    const int32_t s = kv_find(a.b, row, 1, 1, 0);
    const KvSeq seq = kv_seq(a.b, s, a.kv.shift);
    const int64_t within = (int64_t)row - seq.row0;
    if (within < 0 || within >= seq.n) return;  // (a row behind the last sequence)
    const int32_t pos = seq.len - seq.n + (int32_t)within;
    const int32_t* chosen = a.chosen + ((size_t)row * a.kv.n_kv + kvh) * a.count;
    uint32_t total = 0;
    for (uint32_t x = 0; x < a.count; x += 64) {
        const uint64_t named = __ballot(x + lane < a.count && chosen[min(x + lane, a.count - 1)] >= 0);
        if (named) total = x + 64 - (uint32_t)__builtin_clzll(named);
    }
    total <<= a.span_shift;
    // what the row sees: keys below `pre`, and [lo, hi)
    int32_t lo = 0, hi = max(pos + 1, 0), pre = 0;
    if (a.window && pos >= (int32_t)a.window) lo = pos - (int32_t)a.window + 1;
    if (a.first) lo = max(lo, a.first[row]);
    if (hi <= lo) lo = hi = 0;
    if (a.prefix) pre = min(max(a.prefix[s], 0), seq.len);

    // 64 blocks of the list, a lane a block: numbers, places, scales
    uint32_t name = NOWHERE;
    int32_t at = -1;
    float ksc = 1.0f, lvs = 0.0f;
    struct Ahead {
        uint32_t name;
        int32_t page;
    };
    auto names = [&](uint32_t from) {
        const uint32_t x = from + lane;
        Ahead v{NOWHERE, -1};
        if (x < total) {
            // (numbers ascend; one that does not, or that the row's sequence does not have, names nothing; nor is a block read of which the row sees nothing)
            const uint32_t i = x >> a.span_shift;
            const int32_t c = chosen[i], before = i ? chosen[i - 1] : -1;
            if (c > before && c >= 0 && c <= (pos >> 5) >> a.span_shift) {
                const uint32_t blk = ((uint32_t)c << a.span_shift) + (x & ((1u << a.span_shift) - 1));
                const int32_t k0 = (int32_t)(blk * KV_BLOCK);
                if ((k0 < hi && k0 + (int32_t)KV_BLOCK > lo) || k0 < pre) {
                    v.name = blk;
                    v.page = kv_page(a.b, a.kv, s, blk);
                }
            }
        }
        return v;
    };
    float m = NO_MAX, l = 0.0f, bar = bar_of(NO_MAX, false);
    bool watch = false;  // a block without values is among those looked up
    auto settle = [&](const Ahead& v) {
        float vsc = 1.0f;
        name = v.name;
        at = -1;
        ksc = 1.0f;
        if (v.page >= 0) {
            at = (int32_t)kv_block_index(a.kv, v.page, kvh, v.name);
            ksc = key_scale(a.kv.k_scale[at]) * a.scale;
            vsc = a.kv.v_scale[at];
        }
        lvs = value_log(vsc);  // (log2)
        watch = watch || __builtin_amdgcn_ballot_w64(no_values(lvs));
        bar = bar_of(m, watch);
    };
    auto request = [&](const uint8_t* codes, int32_t where, uint4* to) {
        const gbytes p = as_global(codes + (size_t)(uint32_t)max(where, 0) * (KV_BLOCK * d)) + lane * 16;
#pragma unroll
        for (int x = 0; x < KD; x++) to[x] = gload<uint4>(p + x * 1024);
    };
    auto where_of = [&](uint32_t i) { return __builtin_amdgcn_readlane(at, i & 63); };

    settle(names(0));
    uint4 kq[2][KD], vq[2][KD];
    request(a.kv.k, where_of(0), kq[0]);

    // the entries' queries as operands, the same for every set
    half8 qh[KD], ql[F32 ? KD : 1];
    int power;
    {
        float v[KD][8], top = 0.0f;
#pragma unroll
        for (int x = 0; x < KD; x++) {
            if (live) {
                load_query<F32>(a.q, (size_t)row * a.q_stride + (size_t)head * d + x * 32 + grp * 8, a.vec & 1, v[x]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[x][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(v[x][j]));
        }
        const int down = row_power(entry_max(top));
        power = a.power + down;
#pragma unroll
        for (int x = 0; x < KD; x++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float q = ldexpf(v[x][j], -down);
                qh[x][j] = (_Float16)q;
                if constexpr (F32) ql[x][j] = (_Float16)(q - (float)qh[x][j]);
            }
    }
    const float slope = RULES && a.slopes && live ? a.slopes[head] * LOG2E : 0.0f, cap = a.cap * LOG2E, cap_inv = a.cap > 0.0f ? 1.0f / cap : 0.0f;

    f32x4 acc[2 * KD];
#pragma unroll
    for (int t = 0; t < 2 * KD; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    Ahead next{NOWHERE, -1};
    for (uint32_t i = 0; i < total; i += SLOTS) {
        if ((i & 63) == 0 && i + 64 < total) next = names(i + 64);  // (on its way while these 64 are worked on)
        // scores of SLOTS blocks; keys and values one block ahead
        f32x4 sc[SLOTS][2];
#pragma unroll
        for (int b = 0; b < SLOTS; b++) {
            if (b + 1 < SLOTS) request(a.kv.k, where_of(i + b + 1), kq[(b + 1) & 1]);
            else request(a.kv.v, where_of(i), vq[0]);
            sc[b][0] = sc[b][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < KD; x++) {
                const uint4 c = kq[b & 1][x];
                const half8 k_lo = code_values(c.x, c.y), k_hi = code_values(c.z, c.w);
                sc[b][0] = mma(k_lo, qh[x], sc[b][0]);
                sc[b][1] = mma(k_hi, qh[x], sc[b][1]);
                if constexpr (F32) {
                    sc[b][0] = mma(k_lo, ql[x], sc[b][0]);
                    sc[b][1] = mma(k_hi, ql[x], sc[b][1]);
                }
            }
        }
        // the lane's set: its block's number and scales, its scores
        const int from = (int)((i & 63) + slot);
        const int32_t k0 = (int32_t)((uint32_t)__shfl((int)name, from) * KV_BLOCK);
        const float ks_b = __shfl(ksc, from), lv = __shfl(lvs, from);
        const bool none = __shfl(at, from) < 0;
        l = none && ((k0 < hi && k0 + (int32_t)KV_BLOCK > lo) || k0 < pre) ? __builtin_nanf("") : l;  // (no page of the cache)
        float f = score_factor<RULES>(ks_b, power);
        float x[8];
        const int32_t key0 = k0 + 4 * (int32_t)grp, end = k0 + (int32_t)KV_BLOCK;
#pragma unroll
        for (int r = 0; r < 8; r++) {
            x[r] = sc[0][r >> 2][r & 3];
#pragma unroll
            for (int b = 1; b < SLOTS; b++) x[r] = slot == (uint32_t)b ? sc[b][r >> 2][r & 3] : x[r];
            if constexpr (RULES) x[r] *= f;
        }
        if constexpr (RULES) {
            if (a.cap > 0.0f) {
#pragma unroll
                for (int r = 0; r < 8; r++) x[r] = cap * tanh_of(x[r] * cap_inv);
            }
            if (a.slopes) {
                const float far = (float)(pos - key0);
#pragma unroll
                for (int r = 0; r < 8; r++) x[r] = fmaf(-slope, fabsf(far - (float)(16 * (r >> 2) + (r & 3))), x[r]);
            }
        }
        if (__builtin_amdgcn_ballot_w64(!((k0 >= lo && end <= hi) || end <= pre))) {
#pragma unroll
            for (int r = 0; r < 8; r++) {
                const int32_t j = key0 + 16 * (r >> 2) + (r & 3);
                x[r] = (j >= lo && j < hi) || j < pre ? x[r] : -__builtin_inff();
            }
        }
        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if constexpr (!RULES) top *= f;
        float shift = lv + HEAD_ROOM - m;
        if (__builtin_amdgcn_ballot_w64(top + lv > bar)) {
            // (an entry whose own scores need it: another row's do not change a row's bits)
            const float own = entry_max(top) + lv, before = m, to = own > m + (MOST_ROOM - HEAD_ROOM) ? own : m, down = __builtin_amdgcn_exp2f(m - to);
            m = to;
            l = lowered(l, before - to);
#pragma unroll
            for (int c = 0; c < 2 * KD; c++) acc[c] *= down;
            shift = lv + HEAD_ROOM - m;
            bar = bar_of(m, watch);
            if (__builtin_amdgcn_ballot_w64(is_far(m))) {  // (the scores become exponents)
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    const float apart = ((RULES ? x[r] : x[r] * f) - m) + (lv + HEAD_ROOM), near = RULES ? x[r] + shift : fmaf(x[r], f, shift);
                    x[r] = !is_far(m) ? near : apart > F16_ROOM ? F16_ROOM : apart;
                }
                f = 1.0f;
                shift = 0.0f;
            }
            if (__builtin_amdgcn_ballot_w64(no_values(lv))) {  // (weights for the sum alone)
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    sum += __builtin_amdgcn_exp2f((RULES ? x[r] + shift : fmaf(x[r], f, shift)) - lv);
                    x[r] = no_values(lv) ? -__builtin_inff() : x[r];
                }
                l += no_values(lv) ? sum : 0.0f;
            }
        }
        half8 ph, pl;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const float p = __builtin_amdgcn_exp2f(RULES ? x[r] + shift : fmaf(x[r], f, shift));
            sum += p;
            ph[r] = (_Float16)p;
            if constexpr (F32) pl[r] = (_Float16)(p - (float)ph[r]);
        }
        l += sum * __builtin_amdgcn_exp2f(-lv);
        // the values' products; the keys of the next step are asked for behind its places, which may be those of the next 64 blocks
        int32_t wheres[SLOTS];
#pragma unroll
        for (int b = 0; b < SLOTS; b++) wheres[b] = where_of(i + b);
        if ((i & 63) == 64 - SLOTS) {
            settle(next);
            next = Ahead{NOWHERE, -1};
        }
#pragma unroll
        for (int b = 0; b < SLOTS; b++) {
            if (b + 1 < SLOTS) request(a.kv.v, wheres[b + 1 < SLOTS ? b + 1 : b], vq[(b + 1) & 1]);
            else request(a.kv.k, where_of(i + SLOTS), kq[0]);  // (past the last block: some block, or the cache's first)
            const half8 nothing = {0, 0, 0, 0, 0, 0, 0, 0};
            const half8 wh = slot == (uint32_t)b ? ph : nothing;
            half8 wl;
            if constexpr (F32) wl = slot == (uint32_t)b ? pl : nothing;
#pragma unroll
            for (int c = 0; c < KD; c++) {
                const uint4 u = vq[b & 1][c];
                const half8 v_lo = code_values(u.x, u.y), v_hi = code_values(u.z, u.w);
                acc[2 * c] = mma(v_lo, wh, acc[2 * c]);
                acc[2 * c + 1] = mma(v_hi, wh, acc[2 * c + 1]);
                if constexpr (F32) {
                    acc[2 * c] = mma(v_lo, wl, acc[2 * c]);
                    acc[2 * c + 1] = mma(v_hi, wl, acc[2 * c + 1]);
                }
            }
        }
    }
    // the sets meet
    const float most = slots_fold<SLOTS>(m, [](float x, float y) { return fmaxf(x, y); });
    const float sum = slots_fold<SLOTS>(lowered(entry_sum(l), m - most), [](float x, float y) { return x + y; });
    const float down = __builtin_amdgcn_exp2f(m - most) * (sum == 0.0f ? 0.0f : 1.0f / sum);  // (a row that sees nothing: zeros)
#pragma unroll
    for (int c = 0; c < 2 * KD; c++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[c][j] = slots_fold<SLOTS>(acc[c][j] * down, [](float x, float y) { return x + y; });
    if (slot || !live) return;
    const size_t to = (size_t)row * a.out_stride + (size_t)head * d + grp * 4;
#pragma unroll
    for (int c = 0; c < 2 * KD; c++) {
        if constexpr (F32) {
            float* p = static_cast<float*>(a.out) + to + c * 16;
            if (a.vec & 2) *reinterpret_cast<float4*>(p) = make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]);
            else p[0] = acc[c][0], p[1] = acc[c][1], p[2] = acc[c][2], p[3] = acc[c][3];
        } else {
            uint16_t* p = static_cast<uint16_t*>(a.out) + to + c * 16;
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = f32_to_bf16_bits(acc[c][j]);
            if (a.vec & 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
            else p[0] = (uint16_t)w[0], p[1] = (uint16_t)w[1], p[2] = (uint16_t)w[2], p[3] = (uint16_t)w[3];
        }
    }
}

template <int KD, bool F32, bool RULES>
static hipError_t launch_slots(const AttendArgs& a, hipStream_t s) {
    const unsigned grid = ((a.units + ROW_WAVES - 1) / ROW_WAVES + 7) / 8 * 8;
    if (a.g <= 4) attend_rows_kernel<KD, F32, RULES, 4><<<grid, 64 * ROW_WAVES, 0, s>>>(a);
    else attend_rows_kernel<KD, F32, RULES, 2><<<grid, 64 * ROW_WAVES, 0, s>>>(a);
    return hipGetLastError();
}
template <bool F32, bool RULES>
static hipError_t launch_d(const AttendArgs& a, hipStream_t s) {
    switch (a.kv.d / 32) {
        case 1: return launch_slots<1, F32, RULES>(a, s);
        case 2: return launch_slots<2, F32, RULES>(a, s);
        case 3: return launch_slots<3, F32, RULES>(a, s);
        case 4: return launch_slots<4, F32, RULES>(a, s);
        case 5: return launch_slots<5, F32, RULES>(a, s);
        case 6: return launch_slots<6, F32, RULES>(a, s);
        case 7: return launch_slots<7, F32, RULES>(a, s);
        default: return launch_slots<8, F32, RULES>(a, s);
    }
}
hipError_t launch_attend_rows(const AttendArgs& a, bool bf16, bool rules, hipStream_t s) {
    if (bf16) return rules ? launch_d<false, true>(a, s) : launch_d<false, false>(a, s);
    return rules ? launch_d<true, true>(a, s) : launch_d<true, false>(a, s);
}

}  // namespace oxhip
