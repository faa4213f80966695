// Attention of a ragged batch of query rows over the 8-bit key / value cache:
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s),   s_j = cap tanh(scale q k_j / cap) - slope |position - j|
// over the keys that the row sees. One pass over the cache; the maximum and the sum run along.
//
// A tile is 16 query rows of one key head: row i of the tile's sequence and query head h of the group are entry i g + h, so that all heads
// of a group share what is read. A wave takes a block of 32 keys at a time:
//   S^T = K Q^T   2 x d / 32 matrix instructions (16 keys x 16 entries x 32 channels); a lane gets 8 scores of one entry
//   O^T += V^T P^T   d / 16 of them (16 channels x 16 entries x 32 keys), the P^T operand being the lane's 8 weights where they are
// The codes become f16 exactly (1024 + u by a byte permute, less 1152). The key scale joins the score's own factor. The value scale joins
// the weight's exponent, p' = 2^(s + log2 v_scale - m), at no cost, m being the running maximum of s + log2 v_scale; the sum of weights
// is formed of p' / v_scale. p' is at most 2^15 (2^11 when the maximum is set, and the maximum is set anew only when a weight would pass 2^15:
// hardly ever behind a wave's first blocks): of weights rounded to f16, small ones keep as many bits as there are.
// f32 rows: q and p' go in as two f16 values each (value and residual, 22 bits), twice the matrix instructions, which the reads hide.
// bf16 rows: as one (11 bits, where the rows and results have 8); the rows are scaled by a power of two each, so that nothing overflows.
#include <cmath>
#include <type_traits>

#include "attend.hpp"

namespace oxhip {

// Waves of a workgroup, and workgroups on a CU.
constexpr int split_waves(int) { return 8; }
constexpr int split_places(int kd) { return kd <= 4 ? 2 : 1; }

// KD = d / 32; F32: f32 rows; RULES: capped or biased scores, or a factor outside the range that the plain path takes; ONCE: codes pass
// the L2 by, as bytes that are read once.
template <int KD, bool F32, bool RULES, bool ONCE>
__global__ __launch_bounds__(64 * split_waves(KD), 2 * split_places(KD)) void attend_split_kernel(AttendArgs a) {
    constexpr int NW = split_waves(KD), PLANES = F32 ? 2 : 1, CHUNK = KD >= 2 ? 64 : 32;  // channels whose sums the waves exchange at a time
    constexpr int RED = NW * 16 * (CHUNK + 1) > NW * 4 * (KD * 32 + 1) ? NW * 16 * (CHUNK + 1) : NW * 4 * (KD * 32 + 1), JOIN = 16 * MOST_SPLITS + NW * 128;
    __shared__ __align__(16) float lds[RED > JOIN ? RED : JOIN];
    __shared__ float m_s[NW][16], l_s[NW][16];
    __shared__ uint32_t last_s;
    __shared__ half8 q_s[PLANES][KD][64];
    __shared__ float top_s[KD][16];
    constexpr uint32_t d = KD * 32;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = a.g;
    uint32_t tid = threadIdx.x, lane = tid & 63, n = lane & 15, grp = lane >> 4;
    // The compiler takes the thread's number as new: the addresses that it makes of it for one part of a tile's work would otherwise stay in
    // registers through all the others.
    auto anew = [&]() {
        asm volatile("" : "+v"(tid));
        lane = tid & 63;
        n = lane & 15;
        grp = lane >> 4;
    };

    // Which tile, and which part of its blocks, is this workgroup's (kv_weight): a wave adds the sequences' weights up, a lane a sequence, 64 of them
    // at a time, for the others too, so that what decides how many barriers a wave passes is read once.
    __shared__ int32_t seq_s[4][64];
    KvSeq mine{};                              // the lane's sequence of the 64 from s0 on
    uint32_t mine_weight, mine_units, s0 = 0;  // its tiles' weight each; its tiles x key heads
    auto load = [&](uint32_t from) {
        s0 = from;
        __syncthreads();
        if (wave == 0) {
            KvSeq q{};
            uint32_t w = 1;
            bool falls = false;
            if (s0 + lane < a.b.n_seqs) {
                falls = a.b.row_start && a.b.row_start[s0 + lane + 1] < a.b.row_start[s0 + lane];
                q = kv_seq(a.b, (int32_t)(s0 + lane), a.kv.shift);
                if ((uint32_t)q.n * (uint64_t)g >= a.prompt) q.n = 0;  // (attend_prompt_kernel's)
                w = kv_weight(q, a.window, a.window && a.prefix ? a.prefix[s0 + lane] : 0, a.quantum);
            }
            seq_s[0][lane] = q.row0;
            seq_s[1][lane] = q.n;
            seq_s[2][lane] = q.len;
            seq_s[3][lane] = __ballot(falls) ? 0 : (int32_t)w;  // (a weight is 1 at least)
        }
        __syncthreads();
        mine.row0 = seq_s[0][lane];
        mine.n = seq_s[1][lane];
        mine.len = seq_s[2][lane];
        mine_weight = (uint32_t)seq_s[3][lane];
        mine_units = kv_tiles(mine, g) * a.kv.n_kv;
    };
    auto last = [&](uint32_t upto) { return (uint32_t)__builtin_amdgcn_readlane((int)upto, 63); };
    uint32_t total = 0;
    for (uint32_t from = 0; from < a.b.n_seqs; from += 64) {
        load(from);
        // Row numbers that do not ascend may come to more tiles than the launch has workgroups for, and parts that never arrive would leave their
        // counters behind for later calls: nothing is done then.
        if (!last(mine_weight)) return;
        total += last(lanes_upto(mine_units * mine_weight));
    }
    const uint32_t size = max(scalar(divide(total + a.many - 1, a.many)), a.least);
    uint32_t at_wg = 0, at_part = 0;  // workgroups, and parts that workgroups leave for each other, of the sequences before these 64
    uint32_t k, upto, parts_upto, from;
    if (a.b.n_seqs > 64) load(0);
    for (;;) {
        k = divide(mine_weight + size - 1, size);
        upto = lanes_upto(mine_units * k);
        parts_upto = lanes_upto(k > 1 ? mine_units * k : 0);
        const uint64_t behind = __ballot(at_wg + upto > blockIdx.x);  // sequences that end behind this workgroup
        if (behind) {
            from = (uint32_t)__builtin_ctzll(behind);
            break;
        }
        if (s0 + 64 >= a.b.n_seqs) return;
        at_wg += last(upto);
        at_part += last(parts_upto);
        load(s0 + 64);
    }
    const uint32_t s = s0 + from, active = (uint32_t)__builtin_amdgcn_readlane((int)k, from);  // workgroups that share a tile
    const KvSeq seq{(int32_t)s, __builtin_amdgcn_readlane(mine.row0, from), __builtin_amdgcn_readlane(mine.n, from), __builtin_amdgcn_readlane(mine.len, from)};
    const uint32_t units = (uint32_t)__builtin_amdgcn_readlane((int)mine_units, from);
    const uint32_t own = blockIdx.x - (at_wg + (uint32_t)__builtin_amdgcn_readlane((int)upto, from) - units * active);  // of the sequence's workgroups
    const uint32_t unit = scalar(divide(own, active)), part = own - unit * active;
    const int32_t tile = (int32_t)scalar(divide(unit, a.kv.n_kv));
    const uint32_t kvh = unit - (uint32_t)tile * a.kv.n_kv;
    // (where the tile's parts lie in the scratch)
    const uint32_t first_part = active > 1 ? at_part + (uint32_t)__builtin_amdgcn_readlane((int)parts_upto, from) - (units - unit) * active : 0;
    const int64_t entries = (int64_t)seq.n * g;
    const uint32_t e = (uint32_t)tile * 16 + n, cols = (uint32_t)min((int64_t)16, entries - (int64_t)tile * 16);
    const bool live = n < cols;
    const uint32_t i = live ? divide(e, g) : 0u, head = kvh * g + (live ? e - i * g : 0u);
    const size_t row = (size_t)seq.row0 + i;
    const int32_t pos = seq.len - seq.n + (int32_t)i;

    // what the entry sees: keys below `pre`, and [lo, hi)
    int32_t lo = 0, hi = 0, pre = 0;
    if (live) {
        hi = max(pos + 1, 0);
        if (a.window && pos >= (int32_t)a.window) lo = pos - (int32_t)a.window + 1;
        if (a.first) lo = max(lo, a.first[row]);
        if (hi <= lo) lo = hi = 0;
        if (a.prefix) pre = min(max(a.prefix[s], 0), seq.len);
    }
    const int32_t lo_min = tile_min(hi > lo ? lo : INT32_MAX), hi_max = tile_max(hi), lo_max = tile_max(live ? lo : 0), hi_min = tile_min(live ? hi : INT32_MAX);
    const int32_t pre_max = tile_max(pre);
    const KvSpan span = kv_span(pre_max, lo_min, hi_max);
    const uint32_t b0 = part ? (uint32_t)((uint64_t)span.count * part / active) : 0u, b1 = part + 1 < active ? (uint32_t)((uint64_t)span.count * (part + 1) / active) : span.count;

    // The entry's query as operands: in LDS, where all waves read it for each block (kept in registers, it would cost a wave in two its place on
    // the CU). Wave ks brings the channels 32 ks .. 32 ks + 31. What depends on memory goes in an order that keeps the chain short: queries and
    // page numbers are asked for together, the first keys and the scales before the queries are converted.
    float v[8];
    if (wave < KD) {
        const size_t at = row * a.q_stride + (size_t)head * d + wave * 32 + grp * 8;
        if (!live) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 0.0f;
        } else {
            load_query<F32>(a.q, at, a.vec & 1, v);
        }
    }
    const float slope = RULES && a.slopes && live ? a.slopes[head] * LOG2E : 0.0f, cap = a.cap * LOG2E, cap_inv = a.cap > 0.0f ? 1.0f / cap : 0.0f;
    const uint32_t steps = b1 > b0 + wave ? (b1 - b0 - wave + NW - 1) / NW : 0;  // of this wave: blocks b0 + wave, + NW, ...
    // Where the wave's blocks lie, and their scales: for 64 of them at a time, a lane a block. A block's number and scales as scalars, one
    // block ahead of its use; a block of no page reads the cache's first (nothing is made of it).
    int32_t at = -1;
    float ksc = 1.0f, lvs = 0.0f;
    float m = NO_MAX, l = 0.0f, bar;
    bool watch = false;  // a block without values is among the wave's
    auto page_of = [&](uint32_t t) { return t + lane < steps ? kv_page(a.b, a.kv, (int32_t)s, kv_span_block(span, b0 + wave + (t + lane) * NW)) : -1; };
    auto scales_of = [&](uint32_t t, int32_t page) {
        float vsc = 1.0f;
        at = -1;
        ksc = 1.0f;  // (of a block of no page, too: what rows do not see of it is -infinity times this)
        if (page >= 0) {
            at = (int32_t)kv_block_index(a.kv, page, kvh, kv_span_block(span, b0 + wave + (t + lane) * NW));
            ksc = key_scale(a.kv.k_scale[at]) * a.scale;
            vsc = a.kv.v_scale[at];
        }
        return vsc;
    };
    auto look_out = [&]() {
        watch = watch || __builtin_amdgcn_ballot_w64(no_values(lvs));
        bar = bar_of(m, watch);
    };
    auto locate = [&](uint32_t t, int32_t& where, float& ks_b, float& lv) {
        if ((t & 63) == 0) {
            lvs = value_log(scales_of(t, page_of(t)));  // (log2)
            look_out();
        }
        const uint32_t from = t & 63;
        where = __builtin_amdgcn_readlane(at, from);
        ks_b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksc), from));
        lv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs), from));
    };
    auto request = [&](const uint8_t* codes, int32_t where, uint4* to) {
        const gbytes p = as_global(codes + (size_t)(uint32_t)max(where, 0) * (KV_BLOCK * d)) + lane * 16;
#pragma unroll
        for (int x = 0; x < KD; x++) to[x] = ONCE ? gload_once<uint4>(p + x * 1024) : gload<uint4>(p + x * 1024);
    };
    const int32_t page0 = page_of(0);
    if (wave < KD) {
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(v[j]));
        top = entry_max(top);
        if (lane < 16) top_s[wave][lane] = top;
    }
    __syncthreads();
    uint4 kq[KD], vq[KD];
    const float vsc0 = scales_of(0, page0);
    int32_t where = __builtin_amdgcn_readlane(at, 0);
    request(a.kv.k, where, kq);
    float top = top_s[0][n];
#pragma unroll
    for (int ks = 1; ks < KD; ks++) top = fmaxf(top, top_s[ks][n]);
    const int down = row_power(top), power = a.power + down;
    if (wave < KD) {
        half8 hi8, lo8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = ldexpf(v[j], -down);
            hi8[j] = (_Float16)x;
            if constexpr (F32) lo8[j] = (_Float16)(x - (float)hi8[j]);
        }
        q_s[0][wave][lane] = hi8;
        if constexpr (F32) q_s[PLANES - 1][wave][lane] = lo8;
    }
    __syncthreads();

    f32x4 acc[2 * KD];
#pragma unroll
    for (int t = 0; t < 2 * KD; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // keys are on request from the block before, values from before the scores
    {
        lvs = value_log(vsc0);
        look_out();
        int32_t where_next;
        float ks_b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksc), 0)), lv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs), 0)), ks_next, lv_next;
        for (uint32_t t = 0; t < steps; t++) {
            const uint32_t blk = kv_span_block(span, b0 + wave + t * NW);
            const int32_t k0 = (int32_t)(blk * KV_BLOCK);
            request(a.kv.v, where, vq);
            asm volatile("" ::: "memory");  // (the queries are to be read anew, not kept)
            f32x4 sc[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int x = 0; x < KD; x++) {
                const half8 k_lo = code_values(kq[x].x, kq[x].y), k_hi = code_values(kq[x].z, kq[x].w);
#pragma unroll
                for (int plane = 0; plane < PLANES; plane++) {
                    const half8 q = q_s[plane][x][lane];
                    sc[0] = mma(k_lo, q, sc[0]);
                    sc[1] = mma(k_hi, q, sc[1]);
                }
            }
            const bool none = where < 0;
            where_next = where;
            ks_next = ks_b;
            lv_next = lv;
            if (t + 1 < steps) locate(t + 1, where_next, ks_next, lv_next);
            request(a.kv.k, where_next, kq);
            // no page of the cache: rows that would see it come out as NaN
            l = none && ((k0 < hi && k0 + (int32_t)KV_BLOCK > lo) || k0 < pre) ? __builtin_nanf("") : l;
            // scores: of keys k0 + 4 grp + r and k0 + 16 + 4 grp + r
            float f = score_factor<RULES>(ks_b, power);
            float x[8];  // scores times log2 e; without rules, what the products gave: their factor is above 0 and joins the exponent
            const int32_t key0 = k0 + 4 * (int32_t)grp;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                x[r] = sc[r >> 2][r & 3];
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
            const int32_t end = k0 + (int32_t)KV_BLOCK;
            if (!((k0 >= lo_max && end <= hi_min) || end <= pre_max)) {
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
                const float own = entry_max(top) + lv, to = own > m + (MOST_ROOM - HEAD_ROOM) ? own : m, down = __builtin_amdgcn_exp2f(m - to);
                m = to;
                l *= down;
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
                if (no_values(lv)) {  // (weights for the sum alone)
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        sum += __builtin_amdgcn_exp2f(RULES ? x[r] + shift : fmaf(x[r], f, shift));
                        x[r] = -__builtin_inff();
                    }
                    l += sum * __builtin_amdgcn_exp2f(-lv);
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
#pragma unroll
            for (int c = 0; c < KD; c++) {
                const half8 v_lo = code_values(vq[c].x, vq[c].y), v_hi = code_values(vq[c].z, vq[c].w);
                acc[2 * c] = mma(v_lo, ph, acc[2 * c]);
                acc[2 * c + 1] = mma(v_hi, ph, acc[2 * c + 1]);
                if constexpr (F32) {
                    acc[2 * c] = mma(v_lo, pl, acc[2 * c]);
                    acc[2 * c + 1] = mma(v_hi, pl, acc[2 * c + 1]);
                }
            }
            where = where_next;
            ks_b = ks_next;
            lv = lv_next;
        }
    }
    // the waves' parts meet
    anew();
    l = entry_sum(l);
    if (lane < 16) {
        m_s[wave][lane] = m;
        l_s[wave][lane] = l;
    }
    __syncthreads();
    auto meet = [&](uint32_t entry, float& top, float& sum) {
        float mw[NW], lw[NW];
#pragma unroll
        for (int w = 0; w < NW; w++) {
            mw[w] = m_s[w][entry];
            lw[w] = l_s[w][entry];
        }
        top = mw[0];
#pragma unroll
        for (int w = 1; w < NW; w++) top = fmaxf(top, mw[w]);
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) sum += lw[w] * __builtin_amdgcn_exp2f(mw[w] - top);
    };
    auto store = [&](uint32_t entry, uint32_t c, float x) {
        const uint32_t at = (uint32_t)tile * 16 + entry;
        const size_t to = ((size_t)seq.row0 + at / g) * a.out_stride + (size_t)(kvh * g + at % g) * d + c;
        if constexpr (F32) static_cast<float*>(a.out)[to] = x;
        else static_cast<uint16_t*>(a.out)[to] = f32_to_bf16_bits(x);
    };
    const size_t stride = (size_t)a.cols * (d + 2);
    float* mine_part = a.partial + (size_t)(first_part + part) * stride;  // [cols][d], then the maxima, then the sums
    {
        float top, sum;
        meet(n, top, sum);
        const float whole = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that sees nothing: zeros)
        const float down = __builtin_amdgcn_exp2f(m - top) * (active == 1 ? whole : 1.0f);
#pragma unroll
        for (int c = 0; c < 2 * KD; c++) acc[c] *= down;
        if (active > 1 && wave == 0 && lane < cols) {
            __hip_atomic_store(mine_part + (size_t)a.cols * d + lane, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(mine_part + (size_t)a.cols * (d + 1) + lane, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    auto exchange = [&](auto rows, auto channels) {  // so many entries and channels at a time
        constexpr uint32_t ROWS = decltype(rows)::value, C = decltype(channels)::value;
        float* r = lds;  // [NW][ROWS][C + 1]
#pragma unroll
        for (uint32_t c0 = 0; c0 < d; c0 += C) {
            if (c0) __syncthreads();
            if (n < ROWS) {
#pragma unroll
                for (uint32_t c = 0; c < C / 16; c++)
                    if (c0 / 16 + c < 2 * KD)
#pragma unroll
                        for (int x = 0; x < 4; x++) r[(wave * ROWS + n) * (C + 1) + c * 16 + grp * 4 + x] = acc[c0 / 16 + c < 2 * KD ? c0 / 16 + c : 0][x];
            }
            __syncthreads();
            for (uint32_t idx = tid; idx < cols * C; idx += NW * 64) {
                const uint32_t entry = idx / C, c = idx % C;
                if (c0 + c >= d) continue;
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; w++) x += r[(w * ROWS + entry) * (C + 1) + c];
                if (active > 1) __hip_atomic_store(mine_part + (size_t)entry * d + c0 + c, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                else store(entry, c0 + c, x);
            }
        }
    };
    if (cols <= 4) exchange(std::integral_constant<uint32_t, 4>{}, std::integral_constant<uint32_t, d>{});
    else exchange(std::integral_constant<uint32_t, 16>{}, std::integral_constant<uint32_t, CHUNK>{});
    if (active == 1) return;
    // The parts meet through memory: the last workgroup to arrive adds them, in their order; the counter returns to zero for the next
    // launch. (Device-scope accesses throughout and a wait for this thread's stores before the arrival: no cache is written back or emptied.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const uint32_t seen = __hip_atomic_fetch_add(&a.counters[(size_t)first_part * CTR_STRIDE], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_s = seen == active - 1;
        if (seen == active - 1) __hip_atomic_store(&a.counters[(size_t)first_part * CTR_STRIDE], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last_s) return;
    anew();
    const float* all = a.partial + (size_t)first_part * stride;
    float* weight = lds;                        // [16][MOST_SPLITS]: what a split's part counts
    float* sums = lds + 16 * MOST_SPLITS;       // [512][2]
    for (uint32_t entry = wave; entry < cols; entry += NW) {  // an entry a wave, a split a lane
        float mz[MOST_SPLITS / 64], lz[MOST_SPLITS / 64], top = NO_MAX, sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < MOST_SPLITS / 64; i++) {
            const uint32_t z = min(lane + 64 * i, active - 1);
            mz[i] = __hip_atomic_load(all + z * stride + (size_t)a.cols * d + entry, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            lz[i] = __hip_atomic_load(all + z * stride + (size_t)a.cols * (d + 1) + entry, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (uint32_t i = 0; i < MOST_SPLITS / 64; i++) top = fmaxf(top, mz[i]);
#pragma unroll
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
#pragma unroll
        for (uint32_t i = 0; i < MOST_SPLITS / 64; i++) {
            mz[i] = __builtin_amdgcn_exp2f(mz[i] - top);
            sum += lane + 64 * i < active ? mz[i] * lz[i] : 0.0f;
        }
#pragma unroll
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
#pragma unroll
        for (uint32_t i = 0; i < MOST_SPLITS / 64; i++)
            if (lane + 64 * i < active) weight[entry * MOST_SPLITS + lane + 64 * i] = sum == 0.0f ? 0.0f : mz[i] / sum;
    }
    __syncthreads();
    // two channels a thread, and the splits in as many groups as there are threads for
    const uint32_t twos = cols * d / 2, groups = max(1u, (uint32_t)(NW * 64) / twos);
    for (uint32_t i0 = 0; i0 < twos; i0 += NW * 64) {
        const uint32_t idx = groups > 1 ? tid % twos : i0 + tid, group = groups > 1 ? tid / twos : 0u, entry = idx * 2 / d;
        float y0 = 0.0f, y1 = 0.0f;
        if (idx < twos && group < groups) {
            const uint32_t z0 = active * group / groups, z1 = active * (group + 1) / groups;
            const uint64_t* p = reinterpret_cast<const uint64_t*>(all) + idx;  // (a part begins at a multiple of 8 bytes)
            for (uint32_t z = z0; z < z1; z += 8) {
                uint64_t v[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) v[i] = __hip_atomic_load(p + (size_t)min(z + i, z1 - 1) * (stride / 2), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    const float w = z + i < z1 ? weight[entry * MOST_SPLITS + min(z + i, z1 - 1)] : 0.0f;
                    y0 = fmaf(w, __uint_as_float((uint32_t)v[i]), y0);
                    y1 = fmaf(w, __uint_as_float((uint32_t)(v[i] >> 32)), y1);
                }
            }
        }
        if (groups > 1) {
            sums[2 * tid] = y0;
            sums[2 * tid + 1] = y1;
            __syncthreads();
            for (uint32_t j = 1; j < groups && tid < twos; j++) {
                y0 += sums[2 * (tid + j * twos)];
                y1 += sums[2 * (tid + j * twos) + 1];
            }
        }
        if (idx < twos && group == 0) {
            store(entry, idx * 2 % d, y0);
            store(entry, idx * 2 % d + 1, y1);
        }
    }
}

template <bool F32, bool RULES, bool ONCE>
static hipError_t launch_split(const AttendArgs& a, unsigned grid, hipStream_t s) {
    switch (a.kv.d / 32) {
        case 1: attend_split_kernel<1, F32, RULES, ONCE><<<grid, 64 * split_waves(1), 0, s>>>(a); break;
        case 2: attend_split_kernel<2, F32, RULES, ONCE><<<grid, 64 * split_waves(2), 0, s>>>(a); break;
        case 3: attend_split_kernel<3, F32, RULES, ONCE><<<grid, 64 * split_waves(3), 0, s>>>(a); break;
        case 4: attend_split_kernel<4, F32, RULES, ONCE><<<grid, 64 * split_waves(4), 0, s>>>(a); break;
        case 5: attend_split_kernel<5, F32, RULES, ONCE><<<grid, 64 * split_waves(5), 0, s>>>(a); break;
        case 6: attend_split_kernel<6, F32, RULES, ONCE><<<grid, 64 * split_waves(6), 0, s>>>(a); break;
        case 7: attend_split_kernel<7, F32, RULES, ONCE><<<grid, 64 * split_waves(7), 0, s>>>(a); break;
        default: attend_split_kernel<8, F32, RULES, ONCE><<<grid, 64 * split_waves(8), 0, s>>>(a); break;
    }
    return hipGetLastError();
}

hipError_t launch_attend(const KvView& kv, const KvBatchView& b, const AttendCall& call, const DecodeScratch& sc, hipStream_t s) {
    AttendArgs a{};
    a.kv = kv;
    a.b = b;
    a.q = call.q;
    a.out = call.out;
    a.q_stride = call.q_stride;
    a.out_stride = call.out_stride;
    a.slopes = call.slopes;
    a.prefix = call.prefix;
    a.first = call.first;
    a.partial = sc.partial;
    a.counters = sc.counters;
    int power;
    a.scale = std::frexp(call.scale, &power) * LOG2E;
    a.power = power;
    a.cap = call.cap;
    a.g = call.n_q / kv.n_kv;
    a.window = call.window;
    const size_t size = call.bf16 ? 2 : 4;
    auto vec = [&](const void* p, size_t stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0; };
    a.vec = (vec(call.q, call.q_stride) ? 1u : 0u) | (vec(call.out, call.out_stride) ? 2u : 0u);
    const bool rules = call.cap > 0.0f || call.slopes || !(call.scale >= 0x1p-10f && call.scale <= 0x1p40f);
    // Sequences of many query entries go to the kernel that is bound by the matrix cores, those of few to this file's; which of them a batch
    // has is known on the device alone, but where all rows together are few, or all one sequence's.
    // It has tiles of 128 entries and takes a tile's keys one after the other, so it pays where its tiles fill the chip: 1024 rows alone or behind 8192
    // tokens (32 heads of 128 over 8, bf16: 256 tiles) 36 and 216 us, here 43 and 291; 512 rows 22 and 198, here 21 and 153; of heads of 64 channels
    // (8 over 4) 4096 rows 82 and 232, here 58 and 205. The same 1024 rows in f32: 50 and 309, here 48 and 368; capped bf16: 80 and 624, here 50 and 362
    // (2048 rows: 128 and 590, here 131 and 733): for capped scores the border lies too low.
    const uint64_t all = (uint64_t)b.rows * a.g, fill = all * kv.n_kv / 128;
    const bool prompts = b.row_start && all >= PROMPT_ENTRIES && fill >= 256 && fill * kv.d >= 256 * 128;
    a.prompt = !prompts ? 0xFFFFFFFFu : b.n_seqs > 1 ? PROMPT_ENTRIES : 1;
    if (prompts) {
        const hipError_t e = launch_attend_prompt(a, call.bf16, rules, s);
        if (e != hipSuccess || b.n_seqs == 1) return e;
    }
    a.cols = b.row_start ? 16u : min(16u, a.g);
    const uint64_t units = kv_units(b.row_start, b.rows, b.n_seqs, a.g, kv.n_kv), most = (uint64_t)b.max_pages << kv.shift;  // (at most that many)
    a.quantum = kv_quantum(units, most);
    if (!a.quantum) return hipErrorInvalidValue;
    a.many = 256 * split_places((int)kv.d / 32);
    // (blocks of wide heads hold more: 16 x 5 drafted rows of d = 256 24.9 us in parts of 16 blocks and more, 26.2 of 32)
    const uint32_t least = kv.d > 128 ? KV_LEAST / 2 : KV_LEAST;
    a.least = a.quantum < least ? least / a.quantum : 1;
    const uint64_t weight = (most + a.quantum - 1) / a.quantum, parts = (weight + a.least - 1) / a.least;  // of a tile, at most
    uint64_t grid = units * parts < units + a.many ? units * parts : units + a.many;
    if (a.many > MOST_SPLITS || 2 * a.many * CTR_STRIDE > sc.ncounters || 2 * (uint64_t)a.many * a.cols * (kv.d + 2) > sc.partial_floats || !kv_launch_fits(grid, 64 * split_waves((int)kv.d / 32))) return hipErrorInvalidValue;
    // Where a sequence's entries make one tile (all sequences' on average), a block is read once; a second tile finds it in the L2. 64 sequences of
    // 8 heads to a key head, 8192 tokens at most: 74.5 us through the L2, 69.1 past it; 16 sequences of 8 rows of 4: 36.5 and 42.7.
    const bool once = b.row_start ? (uint64_t)b.rows * a.g <= (uint64_t)b.n_seqs * 16 : a.g <= 16;
    const auto go = [&](auto f32, auto ruled) {
        constexpr bool F32 = decltype(f32)::value, RULES = decltype(ruled)::value;
        return once ? launch_split<F32, RULES, true>(a, (unsigned)grid, s) : launch_split<F32, RULES, false>(a, (unsigned)grid, s);
    };
    const std::true_type yes;
    const std::false_type no;
    if (call.bf16) return rules ? go(no, yes) : go(no, no);
    return rules ? go(yes, yes) : go(yes, no);
}

}  // namespace oxhip
