// Which parts of a long cache a row's attention is to read: the mean key of every span of the cache in 8 bits, and for each row and key head the
// spans that score best.
//
// A span is a power of two of tokens of one page and key head. Its mean key m over the tokens that the cache holds of it is kept as signed bytes c with one f32
// scale, s = max |m| / 127, c = rint(m / s). A query is made bytes in the same way for the score (its scale being max |q| times the f32 nearest to 1 / 127),
//   score(span) = max over the heads of the group of (sum of products of bytes) * s_span * s_query:
// the sum is exact (int8 matrix instructions, 32-bit sums), the product of the three is formed in f64, so that which spans are chosen does not depend on the
// order of any sum. A span costs d + 4 bytes to score, 1 / (2 span) of what its keys and values take.
//
// What has to be read is little (2.3 MB for a token over 131072, 14 for 64 sequences of up to 32768): the choice is bound by the chain from page numbers to scores to counts, and
// takes 18 and 14 us of the 24 and 20 that the mean keys, reading back and the choice take together; 1018 rows over 20001 tokens 24 of 29, of which the instructions
// that turn sums into scores and count them are the larger part.
#include <algorithm>

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

constexpr uint32_t WAVE_BINS = 256, ALL_BINS = 1024;

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_of(uint32_t v) {  // another lane's, or 0
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t most_with(uint64_t v) {
    return max(v, (uint64_t)lane_of<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | lane_of<CTRL, ROWS>((uint32_t)v));
}
__device__ __forceinline__ uint64_t wave_most(uint64_t v) {
    v = most_with<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    v = most_with<0x112, 0xF>(v);
    v = most_with<0x114, 0xF>(v);
    v = most_with<0x118, 0xF>(v);
    v = most_with<0x142, 0xA>(v);  // row_bcast:15, then :31
    v = most_with<0x143, 0xC>(v);
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
    v += lane_of<0x111, 0xF>(v);
    v += lane_of<0x112, 0xF>(v);
    v += lane_of<0x114, 0xF>(v);
    v += lane_of<0x118, 0xF>(v);
    v += lane_of<0x142, 0xA>(v);
    v += lane_of<0x143, 0xC>(v);
    return v;
}

// Of the spans first .. last - 1 of a row `need` are taken by their scores, those before and behind them always (n in all); their numbers are written, ascending. The
// score of the last one taken is found by counting: how many scores fall into each of BINS equal parts of the range from the lowest to the highest. The part that
// the count falls into is taken as a whole, or its scores are ranked if they are a wave's lanes at most, or it becomes the range (of scores that are much alike).
// By a wave (WAVES 1), without barriers, or by WAVES waves that share their counts, each of which does the rest for itself: a barrier of eight waves costs more
// than to read 1024 counts. `bins` are zeros, `list` has room for 64 scores, and a number that is 0.
template <uint32_t WAVES, uint32_t BINS>
__device__ __forceinline__ void choose(const uint64_t* score, uint32_t* bins, uint64_t* list, uint32_t* listed, uint32_t n, uint32_t first, uint32_t last, uint32_t need, int32_t* out) {
    constexpr uint32_t THREADS = 64 * WAVES, PER = BINS / 64, BATCH = 4;
    __shared__ unsigned long long range_s[WAVES][2];
    __shared__ uint32_t taken_s[WAVES][2];
    const uint32_t tid = threadIdx.x % THREADS, lane = tid & 63, wave = tid >> 6;
    // what the threads have stored in LDS is read by others behind this
    auto meet = [&]() {
        if constexpr (WAVES > 1) {
            __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    auto each = [&](auto f) {  // f(score) of those that are chosen among, four of a thread at a time
        for (uint32_t x0 = first; x0 < last; x0 += BATCH * THREADS) {
            uint64_t u[BATCH];
#pragma unroll
            for (uint32_t j = 0; j < BATCH; j++) u[j] = score[min(x0 + j * THREADS + tid, last - 1)];
#pragma unroll
            for (uint32_t j = 0; j < BATCH; j++)
                if (x0 + j * THREADS + tid < last) f(u[j]);
        }
    };
    auto widest = [&](uint64_t& lo, uint64_t& hi) {  // over all threads
        lo = ~wave_most(~lo);
        hi = wave_most(hi);
        if constexpr (WAVES > 1) {
            if (lane == 0) range_s[wave][0] = lo, range_s[wave][1] = hi;
            __syncthreads();
#pragma unroll
            for (uint32_t w = 0; w < WAVES; w++) {
                lo = min(lo, (uint64_t)range_s[w][0]);
                hi = max(hi, (uint64_t)range_s[w][1]);
            }
        }
    };
    uint64_t lo = ~0ull, hi = 0;
    each([&](uint64_t u) {
        lo = min(lo, u);
        hi = max(hi, u);
    });
    widest(lo, hi);
    uint32_t above = 0;  // spans that score more than the range
    bool whole = false;
    while (need && lo != hi) {
        // A part of the range: by value where both ends are finite values of a sum that is one too, else by the integers themselves.
        const double top = unordered(hi), wide = top - unordered(lo), by = (double)(BINS - 1) / wide;
        const bool values = lo && wide > 0.0 && wide < __builtin_inf() && by < __builtin_inf();
        constexpr int BITS = 31 - __builtin_clz(BINS);
        const int shift = max(0, 64 - BITS - (int)__builtin_clzll(hi - lo));  // (by integers: as many parts)
        auto part = [&](uint64_t u) { return values ? min((uint32_t)((top - unordered(u)) * by), BINS - 1) : min((uint32_t)((hi - u) >> shift), BINS - 1); };
        each([&](uint64_t u) {
            if (u >= lo && u <= hi) atomicAdd(&bins[part(u)], 1u);
        });
        meet();
        uint32_t c[PER], mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < PER; j += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(&bins[PER * lane + j]);
            c[j] = v.x, c[j + 1] = v.y, c[j + 2] = v.z, c[j + 3] = v.w;
            mine += v.x + v.y + v.z + v.w;
        }
        uint32_t before = above + wave_upto(mine) - mine, in = BINS, in_before = 0, in_it = 0;
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) {
            if (before < need && before + c[j] >= need) in = PER * lane + j, in_before = before, in_it = c[j];
            before += c[j];
        }
        const uint64_t has = __ballot(in < BINS);  // (one lane)
        const int from = has ? (int)__builtin_ctzll(has) : 0;
        in = (uint32_t)__builtin_amdgcn_readlane((int)in, from);
        above = (uint32_t)__builtin_amdgcn_readlane((int)in_before, from);
        in_it = (uint32_t)__builtin_amdgcn_readlane((int)in_it, from);
        whole = above + in_it == need;
        if (in_it <= 64) {
            each([&](uint64_t u) {
                if (u >= lo && u <= hi && part(u) == in) list[atomicAdd(listed, 1u)] = u;
            });
            meet();
            const uint64_t own = lane < in_it ? list[lane] : 0;
            if (whole) {
                lo = hi = ~wave_most(lane < in_it ? ~own : 0);
            } else {
                uint32_t more = 0, as_much = 0;
                for (uint32_t j = 0; j < in_it; j++) {
                    const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(own >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)own, j);
                    more += u > own ? 1u : 0u;
                    as_much += u == own ? 1u : 0u;
                }
                const uint64_t who = __ballot(lane < in_it && above + more < need && above + more + as_much >= need);
                const int at = who ? (int)__builtin_ctzll(who) : 0;
                lo = hi = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(own >> 32), at) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)own, at);
                above += (uint32_t)__builtin_amdgcn_readlane((int)more, at);
            }
            break;
        }
        uint64_t l = ~0ull, h = 0;
        each([&](uint64_t u) {
            if (u >= lo && u <= hi && part(u) == in) {
                l = min(l, u);
                h = max(h, u);
            }
        });
        meet();
        for (uint32_t i = tid; i < BINS; i += THREADS) bins[i] = 0;
        lo = l;
        hi = h;
        widest(lo, hi);
        meet();
        whole = false;
    }
    // All that score more than `lo`, and the first of those that score as much (all of them, if their part is taken as a whole). A wave writes those of its share of
    // the spans behind those of the waves before.
    const uint32_t ties = whole ? 0xFFFFFFFFu : need - above, share = WAVES == 1 ? n : ((n + WAVES - 1) / WAVES + 63) / 64 * 64, x_from = min(wave * share, n), x_to = min(x_from + share, n);
    const uint64_t below = (1ull << lane) - 1;
    auto look = [&](uint32_t x, bool& always, bool& more, bool& equal) {
        always = x < x_to && (x < first || x >= last);
        const bool choice = x < x_to && !always && need;
        const uint64_t u = choice ? score[x] : 0;
        more = choice && u > lo;
        equal = choice && u == lo;
    };
    uint32_t equal_before = 0, to = 0;
    if constexpr (WAVES > 1) {
        uint32_t sure = 0, equals = 0;
        for (uint32_t x0 = x_from; x0 < x_to; x0 += 64) {
            bool always, more, equal;
            look(x0 + lane, always, more, equal);
            sure += (uint32_t)__popcll(__ballot(always || more));
            equals += (uint32_t)__popcll(__ballot(equal));
        }
        if (lane == 0) taken_s[wave][0] = sure, taken_s[wave][1] = equals;
        __syncthreads();
        for (uint32_t w = 0; w < wave; w++) {
            to += taken_s[w][0] + min(taken_s[w][1], ties - min(ties, equal_before));
            equal_before += taken_s[w][1];
        }
    }
    for (uint32_t x0 = x_from; x0 < x_to; x0 += 64) {
        bool always, more, equal;
        look(x0 + lane, always, more, equal);
        const uint64_t equals = __ballot(equal);
        const bool taken = always || more || (equal && equal_before + (uint32_t)__popcll(equals & below) < ties);
        const uint64_t all = __ballot(taken);
        if (taken) out[to + (uint32_t)__popcll(all & below)] = (int32_t)(x0 + lane);
        to += (uint32_t)__popcll(all);
        equal_before += (uint32_t)__popcll(equals);
    }
}

// A workgroup chooses the spans of up to rows_of rows of a sequence for one key head: rows_of times the group's heads are 16 query entries at most (one row of a larger
// group, 16 heads at a time). Scores of 16 spans x 16 entries come from d / 64 matrix instructions, spans as columns; a wave takes four such tiles (of wide heads two) at a time, so that
// their page numbers and scales, then their codes are on their way together (one tile at a time, one row over 131072 tokens took 27 us). Where the entries are 4 or 8,
// four tiles or two share the 16 rows of a result, each adding to rows of its own (the other rows of its operand are zeros), so that no lane works on a row that is none. All
// spans' scores lie in LDS, as integers in their order; then a wave chooses for a row of several, or eight waves for one.
// KD = (d + 63) / 64.
template <bool BF16, uint32_t WAVES, uint32_t KD>
__global__ __launch_bounds__(64 * WAVES, 4) void kv_select_kernel(SelectArgs a) {
    extern __shared__ uint64_t score_s[];  // [rows_of][spans]
    constexpr uint32_t THREADS = 64 * WAVES, TILES = KD <= 2 ? 4 : 2, CHOOSE = 8;  // (a wave's four tiles of wide heads: more registers than there are)
    __shared__ __align__(16) int8_t q_s[17][KD * 64 + 16];  // (the last row is zeros)
    __shared__ double q_scale[16];
    __shared__ __align__(16) uint32_t bins[CHOOSE * WAVE_BINS];
    __shared__ uint64_t list[CHOOSE][64];
    __shared__ uint32_t listed[CHOOSE];
    static_assert(ALL_BINS <= CHOOSE * WAVE_BINS, "");
    const uint32_t d = a.kv.d, tid = threadIdx.x, lane = tid & 63, n = lane & 15, grp = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t head = blockIdx.x % a.kv.n_kv, place = blockIdx.x / a.kv.n_kv, tokens = KV_BLOCK << a.span_shift;
    int32_t s = (int32_t)place, at_place = 0;
    if (a.b.row_start) {
        s = kv_find(a.b, place, 1, a.rows_of, 1);
        at_place = (int32_t)(place - (uint32_t)kv_first_place((uint32_t)max(a.b.row_start[s], 0), s, a.rows_of, 1));
    }
    const KvSeq q = kv_seq(a.b, s, a.kv.shift);
    if (at_place < 0 || (uint64_t)(uint32_t)at_place * a.rows_of >= (uint32_t)q.n) return;
    const uint32_t i0 = (uint32_t)at_place * a.rows_of, rows = min(a.rows_of, (uint32_t)q.n - i0);
    const size_t row0 = (size_t)(uint32_t)q.row0 + i0;
    const int32_t pos0 = q.len - q.n + (int32_t)i0, pos_last = pos0 + (int32_t)rows - 1;
    auto spans_at = [&](int32_t pos) { return pos < 0 ? 0u : (uint32_t)pos / tokens + 1; };
    const uint32_t spans = spans_at(pos_last);
    if (spans > a.count) {
        // a lane's span of the four tiles from t0 on: where its summary lies (-1: nowhere), and its scale
        auto ask = [&](uint32_t t0, int32_t& at, float& scale) {
            const uint32_t x = (t0 + grp) * 16 + n;
            at = -1;
            scale = 0.0f;
            if (grp < TILES && x < spans) {
                const uint32_t block = x << a.span_shift;
                const int32_t page = kv_page(a.b, a.kv, s, block);
                if (page >= 0) {
                    at = (int32_t)(kv_block_index(a.kv, page, head, block) >> a.span_shift);
                    scale = a.scale[at];
                }
            }
        };
        int32_t at_first;
        float scale_first;
        ask(wave * TILES, at_first, scale_first);
        const uint32_t heads_of = min(a.g, 16u);
        for (uint32_t g0 = 0; g0 < a.g; g0 += 16) {  // (one row where there are more than 16)
            const uint32_t heads = min(heads_of, a.g - g0), entries = rows * heads, pad = entries <= 4 && TILES == 4 ? 4u : entries <= 8 ? 8u : 16u;
            if (g0) __syncthreads();
            for (uint32_t e = wave; e < 17; e += WAVES) {
                float v[KD];
                float top = 0.0f;
#pragma unroll
                for (uint32_t j = 0; j < KD; j++) {
                    const uint32_t c = j * 64 + lane;
                    v[j] = 0.0f;
                    if (e < entries && c < d) {
                        const size_t at = (row0 + e / heads) * a.q_stride + (size_t)(head * a.g + g0 + e % heads) * d + c;
                        v[j] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(a.q)[at]) : static_cast<const float*>(a.q)[at];
                        v[j] = v[j] != v[j] ? 0.0f : fminf(fmaxf(v[j], -3.40282347e38f), 3.40282347e38f);  // (NaN counts as 0, infinity as the largest value)
                    }
                    top = fmaxf(top, fabsf(v[j]));
                }
                top = __uint_as_float((uint32_t)wave_most(__float_as_uint(top)));
                const float scale = top * (1.0f / 127.0f);
#pragma unroll
                for (uint32_t j = 0; j < KD; j++) q_s[e][j * 64 + lane] = scale > 0.0f ? (int8_t)(int)fmin(fmax(rint((double)v[j] / (double)scale), -127.0), 127.0) : (int8_t)0;
                if (lane == 0 && e < 16) q_scale[e] = (double)scale;
            }
            if (rows > 1)
                for (uint32_t x = tid; x < rows * a.spans; x += THREADS) score_s[x] = 0;
            if (g0 == 0) {
                for (uint32_t x = tid; x < CHOOSE * WAVE_BINS; x += THREADS) bins[x] = 0;
                if (tid < CHOOSE) listed[tid] = 0;
            }
            __syncthreads();
            // the entries of a lane's four results: their rows and scales
            const uint32_t e0 = grp * 4 % pad;
            double by[4];
            uint32_t of[4];
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                of[r] = (e0 + r) / heads;
                by[r] = q_scale[e0 + r];
            }
            int32_t at_next = at_first;
            float scale_next = scale_first;
            for (uint32_t t0 = wave * TILES; t0 * 16 < spans; t0 += WAVES * TILES) {
                const int32_t at = at_next;
                const float scale = scale_next;
                i32x4 key[TILES][KD];
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    const int32_t where = __shfl(at, (int)(t * 16 + n));
#pragma unroll
                    for (uint32_t j = 0; j < KD; j++) {
                        const uint32_t c = j * 64 + grp * 16;
                        key[t][j] = i32x4{0, 0, 0, 0};
                        if (c < d && where >= 0) key[t][j] = *reinterpret_cast<const i32x4*>(a.code + (size_t)where * d + c);
                    }
                }
                ask(t0 + WAVES * TILES, at_next, scale_next);
                i32x4 dot = {0, 0, 0, 0};
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    // (an operand's row: the entry, where the tile's rows of the result are this one's)
                    const uint32_t e = t % (16 / pad) == n / pad ? n % pad : 16;
#pragma unroll
                    for (uint32_t j = 0; j < KD; j++) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(&q_s[e][j * 64 + grp * 16]), key[t][j], dot, 0, 0, 0);
                    if ((t + 1) % (16 / pad)) continue;
                    // the lane's tile, and its span
                    const uint32_t tile = t + 1 - 16 / pad + grp * 4 / pad, x = (t0 + tile) * 16 + n;
                    const double by_span = (double)(pad == 4 ? scale : __shfl(scale, (int)(tile * 16 + n)));
                    const bool there = (pad == 4 ? at : __shfl(at, (int)(tile * 16 + n))) >= 0;
                    double y[4];
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) y[r] = (double)dot[r] * by_span * by[r];
                    dot = i32x4{0, 0, 0, 0};
                    if (rows == 1) {
                        double best = e0 < entries ? y[0] : -__builtin_inf();
#pragma unroll
                        for (uint32_t r = 1; r < 4; r++) best = e0 + r < entries ? fmax(best, y[r]) : best;  // (passes NaN over)
                        if (pad > 4) best = fmax(best, __shfl_xor(best, 16));
                        if (pad > 8) best = fmax(best, __shfl_xor(best, 32));
                        const uint64_t u = there ? ordered(best) : 0;
                        if (x < spans && e0 == 0) score_s[x] = g0 && score_s[x] > u ? score_s[x] : u;
                    } else if (x < spans && there) {
                        double best = y[0];
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++) {
                            if (e0 + r < entries && (r == 3 || of[r < 3 ? r + 1 : r] != of[r] || e0 + r + 1 >= entries))
                                atomicMax(reinterpret_cast<unsigned long long*>(&score_s[of[r] * a.spans + x]), (unsigned long long)ordered(best));
                            if (r < 3) best = of[r < 3 ? r + 1 : r] == of[r] ? fmax(best, y[r < 3 ? r + 1 : r]) : y[r < 3 ? r + 1 : r];
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    // (those that are taken whatever they score are out of the count; first + last <= count < n_r)
    const uint32_t need = a.count - a.first - a.last;
    if (rows == 1 && spans > a.count) {
        if (wave >= CHOOSE) return;
        choose<CHOOSE, ALL_BINS>(score_s, bins, list[0], listed, spans, a.first, spans - a.last, need, a.out + (row0 * a.kv.n_kv + head) * a.count);
        return;
    }
    for (uint32_t r = wave; r < rows; r += WAVES) {  // (eight at most)
        const uint32_t n_r = spans_at(pos0 + (int32_t)r);
        int32_t* out = a.out + ((row0 + r) * a.kv.n_kv + head) * a.count;
        if (n_r > a.count) {
            choose<1, WAVE_BINS>(score_s + (size_t)r * a.spans, bins + r * WAVE_BINS, list[r], &listed[r], n_r, a.first, n_r - a.last, need, out);
        } else {
            for (uint32_t x = lane; x < a.count; x += 64) out[x] = x < n_r ? (int32_t)x : -1;
        }
    }
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

template <bool BF16, uint32_t WAVES, uint32_t KD>
static hipError_t launch_select(const SelectArgs& a, hipStream_t s) {
    const size_t lds = (size_t)a.rows_of * a.spans * 8;
    if (lds > 32768) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_select_kernel<BF16, WAVES, KD>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)(SELECT_SPANS * 8));
        if (e != hipSuccess) return e;
    }
    kv_select_kernel<BF16, WAVES, KD><<<a.places * a.kv.n_kv, 64 * WAVES, lds, s>>>(a);
    return hipGetLastError();
}
template <bool BF16, uint32_t WAVES>
static hipError_t launch_select(const SelectArgs& a, hipStream_t s) {
    switch ((a.kv.d + 63) / 64) {
        case 1: return launch_select<BF16, WAVES, 1>(a, s);
        case 2: return launch_select<BF16, WAVES, 2>(a, s);
        case 3: return launch_select<BF16, WAVES, 3>(a, s);
        default: return launch_select<BF16, WAVES, 4>(a, s);
    }
}
hipError_t launch_kv_select(const SelectArgs& args, bool bf16, hipStream_t s) {
    SelectArgs a = args;
    const uint64_t spans = ((uint64_t)a.b.max_pages << a.kv.shift) >> a.span_shift;
    if (spans > SELECT_SPANS) return hipErrorInvalidValue;
    a.spans = (uint32_t)spans;
    // (the scores of several rows at most 32 KiB, so that some workgroups share a CU)
    a.rows_of = a.b.row_start && a.g < 16 ? std::max<uint32_t>(1, std::min<uint32_t>({16 / a.g, 8, (uint32_t)(32768 / (spans * 8))})) : 1;
    const uint64_t places = a.b.row_start ? kv_places(a.b.rows, a.b.n_seqs, a.rows_of, 1) : a.b.n_seqs;
    if (!kv_launch_fits(places * a.kv.n_kv, 1024)) return hipErrorInvalidValue;
    a.places = (uint32_t)places;
    const bool wide = places * a.kv.n_kv <= 256 && spans >= 1024;  // (few rows, long ones)
    if (bf16) return wide ? launch_select<true, 16>(a, s) : launch_select<true, 8>(a, s);
    return wide ? launch_select<false, 16>(a, s) : launch_select<false, 8>(a, s);
}

}  // namespace oxhip
