// The attention kernel for few rows a sequence (attend.hip has the mathematics), over what a tile reads: the keys that its sequence's rows see (PLAIN), the
// shared tokens of a group's sequences and each sequence's own (SHARED), or the spans that were chosen for a row (CHOSEN).
#pragma once
#include <type_traits>

#include "attend.hpp"

namespace oxhip {

enum { PLAIN, SHARED, CHOSEN };
constexpr uint32_t BLOCK_BITS = 26, BLOCK_MASK = (1u << BLOCK_BITS) - 1, NO_BLOCK = BLOCK_MASK - 1;  // (a sequence has at most 2^26 - 2 blocks: none of its rows sees keys of this one)

// Waves of a workgroup, and workgroups on a CU.
constexpr int split_waves(int) { return 8; }
constexpr int split_places(int kd) { return kd <= 4 ? 2 : 1; }

// KD = d / 32; F32: f32 rows; RULES: capped or biased scores, or a factor outside the range that the plain path takes; ONCE: codes pass
// the L2 by, as bytes that are read once; KIND: which blocks a tile reads.
template <int KD, bool F32, bool RULES, bool ONCE, int KIND>
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

    KvSeq seq;                                // the entry's sequence (its number also one of the batch's tables)
    uint32_t kvh, part, active, first_part;   // key head; this part of the tile's blocks, of so many; where the parts lie in the scratch
    uint32_t cols, e0, i, head, per, head0;   // entries; entry e is query head head0 + (e0 + e) % per of row first_row + (e0 + e) / per
    size_t first_row;
    bool live;
    int32_t pos = 0;
    uint32_t total = 0;  // blocks of the tile
    // what only a shared prefix has, and what only chosen spans have
    __shared__ uint32_t run_end[KIND == SHARED ? 32 : 1], run_pre[KIND == SHARED ? 32 : 1], run_base[KIND == SHARED ? 32 : 1], run_lo[KIND == SHARED ? 32 : 1];
    __shared__ int32_t run_table[KIND == SHARED ? 32 : 1], live_s[KIND == SHARED ? 16 : 1];
    int32_t common = 0;                      // tokens that the entry's sequence shares
    uint32_t run_common = 0, run_own = 0;    // the runs of blocks that the entry sees
    const int32_t* chosen = nullptr;         // the row's spans
    auto last_lane = [&](uint32_t upto) { return (uint32_t)__builtin_amdgcn_readlane((int)upto, 63); };
    if constexpr (KIND == PLAIN) {
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
        uint32_t weights = 0;
        for (uint32_t from = 0; from < a.b.n_seqs; from += 64) {
            load(from);
            // Row numbers that do not ascend may come to more tiles than the launch has workgroups for, and parts that never arrive would leave their
            // counters behind for later calls: nothing is done then.
            if (!last_lane(mine_weight)) return;
            weights += last_lane(lanes_upto(mine_units * mine_weight));
        }
        const uint32_t size = max(scalar(divide(weights + a.many - 1, a.many)), a.least);
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
            at_wg += last_lane(upto);
            at_part += last_lane(parts_upto);
            load(s0 + 64);
        }
        active = (uint32_t)__builtin_amdgcn_readlane((int)k, from);  // workgroups that share a tile
        seq = KvSeq{(int32_t)(s0 + from), __builtin_amdgcn_readlane(mine.row0, from), __builtin_amdgcn_readlane(mine.n, from), __builtin_amdgcn_readlane(mine.len, from)};
        const uint32_t units = (uint32_t)__builtin_amdgcn_readlane((int)mine_units, from);
        const uint32_t own = blockIdx.x - (at_wg + (uint32_t)__builtin_amdgcn_readlane((int)upto, from) - units * active);  // of the sequence's workgroups
        const uint32_t unit = scalar(divide(own, active));
        part = own - unit * active;
        const uint32_t tile = scalar(divide(unit, a.kv.n_kv));
        kvh = unit - tile * a.kv.n_kv;
        // (where the tile's parts lie in the scratch)
        first_part = active > 1 ? at_part + (uint32_t)__builtin_amdgcn_readlane((int)parts_upto, from) - (units - unit) * active : 0;
        const int64_t entries = (int64_t)seq.n * g;
        e0 = tile * 16;
        cols = (uint32_t)min((int64_t)16, entries - (int64_t)e0);
        per = g;
        head0 = kvh * g;
        first_row = (size_t)seq.row0;
        live = n < cols;
        i = live ? divide(e0 + n, g) : 0u;
        head = head0 + (live ? e0 + n - i * g : 0u);
    } else {
        // Tiles of a.tile_rows rows of the batch (of one row, or 16 heads of its group, where KIND is CHOSEN), each in a.parts parts at most.
        const uint32_t unit = blockIdx.x % a.units, heads = (g + 15) / 16;
        part = blockIdx.x / a.units;
        kvh = unit % a.kv.n_kv;
        const uint32_t tile = unit / a.kv.n_kv / heads, h16 = unit / a.kv.n_kv % heads;
        per = min(16u, g - 16 * h16);
        const uint32_t rows_of = KIND == SHARED ? a.tile_rows : 1, row0 = tile * rows_of, rows = min(rows_of, a.b.rows - row0);
        first_row = row0;
        e0 = 0;
        head0 = kvh * g + 16 * h16;
        cols = rows * per;
        first_part = unit * a.parts;
        live = n < cols;
        i = live ? divide(n, per) : 0u;
        head = head0 + (live ? n - i * per : 0u);
        // the sequence of the tile's row `mine`: lane n's
        const uint32_t mine = min(n, rows - 1);
        int32_t s_mine = (int32_t)(row0 + mine);
        if (a.b.row_start) {
            const int32_t s0 = kv_find(a.b, row0, 1, 1, 0);
            const int32_t ends = a.b.row_start[min((uint32_t)s0 + lane, a.b.n_seqs - 1) + 1];
            for (uint32_t r = 0; r < rows; r++) {
                const uint64_t before = __ballot(ends <= (int32_t)(row0 + r));  // (sequences that end before this row)
                const int32_t s = ~before ? min(s0 + __builtin_ctzll(~before), (int32_t)a.b.n_seqs - 1) : kv_find(a.b, row0 + r, 1, 1, 0);
                s_mine = mine == r ? s : s_mine;
            }
        }
        seq = kv_seq(a.b, s_mine, a.kv.shift);
        const int64_t within = (int64_t)row0 + mine - seq.row0;
        const bool in = within >= 0 && within < seq.n;
        if constexpr (KIND == CHOSEN) {
            if (!in) return;  // (a row behind the last sequence)
            pos = seq.len - seq.n + (int32_t)within;
            chosen = a.chosen + ((size_t)row0 * a.kv.n_kv + kvh) * a.count;
            for (uint32_t x = 0; x < a.count; x += 64) {
                const uint64_t named = __ballot(x + lane < a.count && chosen[min(x + lane, a.count - 1)] >= 0);
                if (named) total = x + 64 - (uint32_t)__builtin_clzll(named);
            }
            total <<= a.span_shift;
        } else {
            // The tile's blocks come in runs: what the rows of a group see of its shared tokens (run r, of the first row r of the group that is in the
            // tile), then what the rows of a sequence see of its own (run 16 + r). Lane 16 x + r makes runs r and 16 + r of row r.
            int32_t gi = 0;
            {
                int32_t to = (int32_t)a.n_groups + 1;  // the last group that begins at the sequence or before it
                while (gi < to) {
                    const int32_t mid = (gi + to) / 2;
                    if (a.group_start[mid] <= seq.s) gi = mid + 1;
                    else to = mid;
                }
                gi--;
            }
            int32_t leader = -1;
            common = 0;
            if (in && gi >= 0 && gi < (int32_t)a.n_groups) {
                leader = a.group_start[gi];
                if (leader >= 0 && leader <= seq.s) common = (int32_t)min((int64_t)max(a.common[gi], 0), (int64_t)a.b.max_pages * KV_BLOCK << a.kv.shift);
            }
            const int32_t p = seq.len - seq.n + (int32_t)within;
            int32_t r_hi = in ? max(p + 1, 0) : 0, r_lo = a.window && p >= (int32_t)a.window ? p - (int32_t)a.window + 1 : 0;
            if (in && a.first) r_lo = max(r_lo, a.first[row0 + mine]);
            if (r_hi <= r_lo) r_lo = r_hi = 0;
            const int32_t r_pre = in && a.prefix ? min(max(a.prefix[seq.s], 0), seq.len) : 0;
            const int32_t r_s = in ? seq.s : -1 - (int32_t)mine, r_g = common > 0 ? gi : -1 - (int32_t)mine;  // (what has none is alone)
            int32_t lo_min = INT32_MAX, hi_max = 0, pre_max = 0, first_g = 16, first_s = 16, s_lo = INT32_MAX, s_hi = 0;
            for (uint32_t r = 0; r < rows; r++) {
                const int32_t hi = __builtin_amdgcn_readlane(r_hi, r), lo = __builtin_amdgcn_readlane(r_lo, r), pre = __builtin_amdgcn_readlane(r_pre, r);
                if (__builtin_amdgcn_readlane(r_g, r) == r_g) {
                    first_g = min(first_g, (int32_t)r);
                    const int32_t end = min(hi, common);
                    if (end > lo) {
                        lo_min = min(lo_min, lo);
                        hi_max = max(hi_max, end);
                    }
                    pre_max = max(pre_max, min(pre, common));
                }
                if (__builtin_amdgcn_readlane(r_s, r) == r_s) {
                    first_s = min(first_s, (int32_t)r);
                    if (hi > max(lo, common)) {
                        s_lo = min(s_lo, max(lo, common));
                        s_hi = max(s_hi, hi);
                    }
                }
            }
            const bool own_run = (lane & 16) != 0, first = n < rows && (own_run ? first_s : first_g) == (int32_t)n;
            // (a sequence's own: from the block that its first own token is in)
            const uint32_t base = own_run ? (uint32_t)common / KV_BLOCK : 0u;
            KvSpan run = own_run ? kv_span_from(base, r_pre > common ? r_pre : 0, s_lo, s_hi) : kv_span(pre_max, lo_min, hi_max);
            if (!first || (!own_run && common <= 0) || (own_run && !in)) run.count = 0;
            const uint32_t upto = lanes_upto(lane < 32 ? run.count : 0u);
            if (wave == 0 && lane < 32) {
                run_end[lane] = upto;
                run_pre[lane] = run.pre;
                run_base[lane] = base;
                run_lo[lane] = run.lo;
                run_table[lane] = own_run ? seq.s : leader;
            }
            total = last_lane(upto);
            // (from the row's lane to the entry's)
            const int32_t mine_in = __shfl((int)in, (int)i);
            seq = KvSeq{__shfl(seq.s, (int)i), __shfl(seq.row0, (int)i), __shfl(seq.n, (int)i), __shfl(seq.len, (int)i)};
            pos = __shfl(p, (int)i);
            common = __shfl(common, (int)i);
            run_common = (uint32_t)__shfl(first_g, (int)i);
            run_own = 16 + (uint32_t)__shfl(first_s, (int)i);
            live = live && mine_in;
            if (wave == 0 && lane < 16) live_s[lane] = live;
            __syncthreads();
        }
        // (a part is a.least blocks at least)
        active = min(a.parts, max(1u, (total + a.least - 1) / a.least));
        if (part >= active) return;
    }
    const size_t row = first_row + i;

    // what the entry sees: keys below `pre`, and [lo, hi)
    int32_t lo = 0, hi = 0, pre = 0;
    if constexpr (KIND == PLAIN) pos = seq.len - seq.n + (int32_t)i;
    if (live) {
        hi = max(pos + 1, 0);
        if (a.window && pos >= (int32_t)a.window) lo = pos - (int32_t)a.window + 1;
        if (a.first) lo = max(lo, a.first[row]);
        if (hi <= lo) lo = hi = 0;
        if (a.prefix) pre = min(max(a.prefix[seq.s], 0), seq.len);
    }
    const int32_t lo_min = tile_min(hi > lo ? lo : INT32_MAX), hi_max = tile_max(hi), lo_max = tile_max(live ? lo : 0);
    int32_t hi_min = tile_min(live ? hi : INT32_MAX), pre_max = tile_max(pre);
    KvSpan span{};
    if constexpr (KIND == PLAIN) {
        span = kv_span(pre_max, lo_min, hi_max);
        total = span.count;
    }
    // Of a shared prefix: of the shared tokens [lo, hi_c) and those below pre_c, of the sequence's own [lo_o, hi_o) and [common, pre_o). All entries
    // see the whole of a shared block that ends at hi_min, or at pre_max (here the least), if all of them are of one group.
    int32_t hi_c = 0, pre_c = 0, lo_o = 0, hi_o = 0, pre_o = 0;
    if constexpr (KIND == SHARED) {
        hi_c = min(hi, common) > lo ? min(hi, common) : 0;
        pre_c = min(pre, common);
        lo_o = max(lo, common);
        hi_o = hi > lo_o ? hi : 0;
        pre_o = pre > common ? pre : 0;
        const bool one = !__builtin_amdgcn_ballot_w64(live && run_common != 0);
        hi_min = one ? tile_min(live ? hi_c : INT32_MAX) : 0;
        pre_max = one ? tile_min(live ? pre_c : INT32_MAX) : 0;
    }
    const uint32_t b0 = part ? (uint32_t)((uint64_t)total * part / active) : 0u, b1 = part + 1 < active ? (uint32_t)((uint64_t)total * (part + 1) / active) : total;

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
    // (a block's number, and above it the run that it is of)
    uint32_t name = NO_BLOCK;
    auto page_of = [&](uint32_t t) {
        if (t + lane >= steps) return -1;
        const uint32_t x = b0 + wave + (t + lane) * NW;
        if constexpr (KIND == PLAIN) {
            return kv_page(a.b, a.kv, seq.s, kv_span_block(span, x));
        } else if constexpr (KIND == SHARED) {
            uint32_t run = 0;
#pragma unroll
            for (uint32_t r = 0; r < 31; r++) run += x >= run_end[r] ? 1u : 0u;
            const uint32_t y = run ? x - run_end[run - 1] : x, blk = y < run_pre[run] ? run_base[run] + y : run_lo[run] + (y - run_pre[run]);
            name = blk | run << BLOCK_BITS;
            return kv_page(a.b, a.kv, run_table[run], blk);
        } else {
            // (numbers ascend; one that does not, or that the row's sequence does not have, names nothing)
            const uint32_t at = x >> a.span_shift;
            const int32_t c = chosen[at], before = at ? chosen[at - 1] : -1;
            const bool named = c > before && c >= 0 && c <= (pos >> 5) >> a.span_shift;
            name = named ? ((uint32_t)c << a.span_shift) + (x & ((1u << a.span_shift) - 1)) : NO_BLOCK;
            // (nor is a block read of which the row sees nothing: what the cache holds there may be anything)
            const int32_t k0 = (int32_t)(name * KV_BLOCK);
            if (!((k0 < hi_max && k0 + (int32_t)KV_BLOCK > lo_min) || k0 < pre_max)) name = NO_BLOCK;
            return name == NO_BLOCK ? -1 : kv_page(a.b, a.kv, seq.s, name);
        }
    };
    auto scales_of = [&](uint32_t t, int32_t page) {
        float vsc = 1.0f;
        at = -1;
        ksc = 1.0f;  // (of a block of no page, too: what rows do not see of it is -infinity times this)
        if (page >= 0) {
            at = (int32_t)kv_block_index(a.kv, page, kvh, KIND == PLAIN ? kv_span_block(span, b0 + wave + (t + lane) * NW) : name & BLOCK_MASK);
            ksc = key_scale(a.kv.k_scale[at]) * a.scale;
            vsc = a.kv.v_scale[at];
        }
        return vsc;
    };
    auto look_out = [&]() {
        watch = watch || __builtin_amdgcn_ballot_w64(no_values(lvs));
        bar = bar_of(m, watch);
    };
    auto locate = [&](uint32_t t, int32_t& where, float& ks_b, float& lv, uint32_t& named) {
        if ((t & 63) == 0) {
            lvs = value_log(scales_of(t, page_of(t)));  // (log2)
            look_out();
        }
        const uint32_t from = t & 63;
        where = __builtin_amdgcn_readlane(at, from);
        if constexpr (KIND != PLAIN) named = (uint32_t)__builtin_amdgcn_readlane((int)name, from);
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
        uint32_t named = KIND != PLAIN ? (uint32_t)__builtin_amdgcn_readlane((int)name, 0) : 0u, named_next = named;
        float ks_b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ksc), 0)), lv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lvs), 0)), ks_next, lv_next;
        for (uint32_t t = 0; t < steps; t++) {
            const uint32_t blk = KIND == PLAIN ? kv_span_block(span, b0 + wave + t * NW) : named & BLOCK_MASK;
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
            if (t + 1 < steps) locate(t + 1, where_next, ks_next, lv_next, named_next);
            request(a.kv.k, where_next, kq);
            // what the entry sees of this block's run: keys [v_lo, v_hi), and [v_base, v_pre)
            int32_t v_lo = lo, v_hi = hi, v_base = 0, v_pre = pre;
            if constexpr (KIND == SHARED) {
                const uint32_t run = named >> BLOCK_BITS;
                const bool of_group = run == run_common, of_own = run == run_own;
                v_lo = of_own ? lo_o : lo;
                v_hi = of_group ? hi_c : of_own ? hi_o : 0;
                v_base = of_own ? common : 0;
                v_pre = of_group ? pre_c : of_own ? pre_o : 0;
            }
            // no page of the cache: rows that would see it come out as NaN
            l = none && ((k0 < v_hi && k0 + (int32_t)KV_BLOCK > v_lo) || (k0 < v_pre && (KIND != SHARED || k0 + (int32_t)KV_BLOCK > v_base))) ? __builtin_nanf("") : l;
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
            if (!((k0 >= lo_max && end <= hi_min) || end <= pre_max) || (KIND == SHARED && named >> BLOCK_BITS >= 16)) {
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    const int32_t j = key0 + 16 * (r >> 2) + (r & 3);
                    x[r] = (j >= v_lo && j < v_hi) || (j < v_pre && (KIND != SHARED || j >= v_base)) ? x[r] : -__builtin_inff();
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
                if (no_values(lv)) {  // (weights for the sum alone)
                    float sum = 0.0f;
#pragma unroll
                    for (int r = 0; r < 8; r++) {
                        sum += __builtin_amdgcn_exp2f((RULES ? x[r] + shift : fmaf(x[r], f, shift)) - lv);
                        x[r] = -__builtin_inff();
                    }
                    l += sum;
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
            named = named_next;
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
        for (int w = 0; w < NW; w++) sum += lowered(lw[w], mw[w] - top);
    };
    auto store = [&](uint32_t entry, uint32_t c, float x) {
        if constexpr (KIND == SHARED)
            if (!live_s[entry]) return;  // (a row behind the last sequence)
        const uint32_t at = e0 + entry;
        const size_t to = (first_row + at / per) * a.out_stride + (size_t)(head0 + at % per) * d + c;
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
            sum += lane + 64 * i < active ? lowered(lz[i], mz[i] - top) : 0.0f;
            mz[i] = __builtin_amdgcn_exp2f(mz[i] - top);
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

template <bool F32, bool RULES, bool ONCE, int KIND>
static hipError_t launch_split(const AttendArgs& a, unsigned grid, hipStream_t s) {
    switch (a.kv.d / 32) {
        case 1: attend_split_kernel<1, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(1), 0, s>>>(a); break;
        case 2: attend_split_kernel<2, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(2), 0, s>>>(a); break;
        case 3: attend_split_kernel<3, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(3), 0, s>>>(a); break;
        case 4: attend_split_kernel<4, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(4), 0, s>>>(a); break;
        case 5: attend_split_kernel<5, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(5), 0, s>>>(a); break;
        case 6: attend_split_kernel<6, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(6), 0, s>>>(a); break;
        case 7: attend_split_kernel<7, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(7), 0, s>>>(a); break;
        default: attend_split_kernel<8, F32, RULES, ONCE, KIND><<<grid, 64 * split_waves(8), 0, s>>>(a); break;
    }
    return hipGetLastError();
}

}  // namespace oxhip
