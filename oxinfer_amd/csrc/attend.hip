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

#include "attend_split.hpp"

namespace oxhip {

AttendArgs attend_args(const KvView& kv, const KvBatchView& b, const AttendCall& call, const DecodeScratch& sc, bool* rules) {
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
    *rules = call.cap > 0.0f || call.slopes || !(call.scale >= 0x1p-10f && call.scale <= 0x1p40f);
    return a;
}

hipError_t launch_attend(const KvView& kv, const KvBatchView& b, const AttendCall& call, const DecodeScratch& sc, hipStream_t s) {
    bool rules;
    AttendArgs a = attend_args(kv, b, call, sc, &rules);
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
        return once ? launch_split<F32, RULES, true, PLAIN>(a, (unsigned)grid, s) : launch_split<F32, RULES, false, PLAIN>(a, (unsigned)grid, s);
    };
    const std::true_type yes;
    const std::false_type no;
    if (call.bf16) return rules ? go(no, yes) : go(no, no);
    return rules ? go(yes, yes) : go(yes, no);
}

}  // namespace oxhip
