// Attention over a prefix that a batch's sequences share, and over chosen spans of a cache: what attend.hip computes, over other lists of blocks.
//
// A tile is 16 query entries of one key head. Of a shared prefix they may come from several sequences, so that a shared block is read, and its codes are made
// f16 values, once for 16 entries; behind the shared tokens a tile's list names each sequence's own blocks, whose keys the other sequences' entries do not see.
// Of chosen spans a tile is one row's group of heads, for which the spans were chosen together.
//
// Shared: 64 sequences behind 8192 tokens and up to 1024 of their own, 8 key heads of 128 with 4 heads each, bf16, 40 us (68 MB from memory 13; `attend` over tables that
// name the shared pages 120); 128 behind 32768, f32, 197 (the products, twice for two planes, 117; `attend` 625). A block that 16 tiles of a key head take each comes from the L2
// all but once (93 % hits of the longer case), at 10 to 12 TB/s (the rate seen: that the L2 gives no more is not shown); a wave's step of 240 vector and 16 matrix instructions (32 of f32 rows) is a chain that four waves a SIMD do not quite
// fill. Chosen: 64 sequences, 64 spans of 64 each, 88 us: memory, 5.4 TB/s.
#include <cmath>

#include "attend_split.hpp"

namespace oxhip {

// How many tiles a batch has, and parts of each: `target` workgroups in all, where lists of `blocks` blocks at most (even: all as long) have parts of a.least blocks for them.
static hipError_t spread(AttendArgs& a, const DecodeScratch& sc, bool several, bool even, uint64_t blocks, uint32_t target, unsigned* grid) {
    const uint64_t units = kv_row_tiles(a.b.rows, a.g, several) * a.kv.n_kv;
    a.tile_rows = several && a.g < 16 ? 16 / a.g : 1;
    a.cols = std::min(16u, a.tile_rows * a.g);
    const uint64_t room = std::min<uint64_t>(sc.partial_floats / ((uint64_t)a.cols * (a.kv.d + 2)), sc.ncounters / CTR_STRIDE);  // parts that the scratch holds
    // A few workgroups more than the chip takes at once are a second round of them, so there are fewer then, and longer ones: of chosen spans, lists of one length, up to an eighth too many
    // (24 rows of 4 key heads of d = 256: 288 workgroups on 256 places 47.1 us, 192 of them 36.0; but 640 on 512 58.2, 320 of them 61.9). Of shared prefixes lists differ, and some have
    // fewer parts, so only where the fewer ones fill the chip all the same (288 34.9 us, 252 of them 27.8; 560 on 512 39.5, 480 of them 30.5; but 260 33.1, 208 of them 37.1).
    const uint64_t wanted = (target + units - 1) / units, fewer = std::max<uint64_t>(1, target / units);
    const bool round = even ? units * wanted * 8 <= target * 9 : units * fewer * 16 >= target * 15;
    uint64_t parts = std::max<uint64_t>(1, std::min<uint64_t>(round ? fewer : wanted, (blocks + a.least - 1) / a.least));
    parts = std::min<uint64_t>(parts, MOST_SPLITS);
    if (units * parts > room) parts = std::max<uint64_t>(1, room / units);
    if (!kv_launch_fits(units * parts, 64 * split_waves((int)a.kv.d / 32))) return hipErrorInvalidValue;
    a.units = (uint32_t)units;
    a.parts = (uint32_t)parts;
    *grid = (unsigned)(units * parts);
    return hipSuccess;
}
template <int KIND>
static hipError_t go(const AttendArgs& a, bool bf16, bool rules, unsigned grid, hipStream_t s) {
    if (bf16) return rules ? launch_split<false, true, false, KIND>(a, grid, s) : launch_split<false, false, false, KIND>(a, grid, s);
    return rules ? launch_split<true, true, false, KIND>(a, grid, s) : launch_split<true, false, false, KIND>(a, grid, s);
}

hipError_t launch_attend_shared(const KvView& kv, const KvBatchView& b, const SharedView& shared, const AttendCall& call, const DecodeScratch& sc, hipStream_t s) {
    bool rules;
    AttendArgs a = attend_args(kv, b, call, sc, &rules);
    a.least = kv.d > 128 ? KV_LEAST / 2 : KV_LEAST;
    a.group_start = shared.group_start;
    a.common = shared.common;
    a.n_groups = shared.n_groups;
    unsigned grid;
    // Rows share what they read where there is more of it than the chip takes at once. Fewer have tiles of their own, whose lists are shorter and whose workgroups have fewer entries
    // to join (8 key heads of 128, 4 heads each, f32: 4 sequences behind 700 tokens 11.1 us, 14.1 of four rows a tile; 32 of them 11.1 and 14.3; 8 behind 3000 tokens 16.2 and 20.4; and from the
    // border on 64 behind 700 tokens 16.2 and 14.5; 16 behind 3000 21.7 and 20.6; 16 behind 12000 43.0 and 27.7). The host knows the tables' room alone: four answers behind 700 tokens in
    // tables for 131072 share tiles, and take 13.8 us.
    const uint64_t blocks = (uint64_t)b.max_pages << kv.shift, alone = kv_row_tiles(b.rows, a.g, false) * kv.n_kv * ((blocks + a.least - 1) / a.least);
    const hipError_t e = spread(a, sc, alone > 256, false, blocks, 256 * split_places((int)kv.d / 32), &grid);
    return e != hipSuccess ? e : go<SHARED>(a, call.bf16, rules, grid, s);
}

constexpr uint64_t ROW_UNITS = 2048, ROW_ROWS = 32;

hipError_t launch_attend_selected(const KvView& kv, const KvBatchView& b, const ChosenView& chosen, const AttendCall& call, const DecodeScratch& sc, hipStream_t s) {
    bool rules;
    AttendArgs a = attend_args(kv, b, call, sc, &rules);
    a.least = kv.d > 128 ? KV_LEAST / 2 : KV_LEAST;
    a.chosen = chosen.chosen;
    a.count = chosen.count;
    while ((1u << a.span_shift) < chosen.span_blocks) a.span_shift++;
    // A wave a row and key head where these fill the chip and have a sequence's codes in common, so that they are bound by the L2 and by their own instructions
    // (64 spans of 64 of a prompt of 16384, 8 key heads of 128 with 4 heads each, bf16: 256 rows 126 us, 145 with a workgroup a row and key head, 512 rows 226 and 272, 2048 833 and
    // 1001; 128 rows 78 and 78; dense attention of 256, 512 and 2048 rows 163, 267 and 598). Rows of sequences of their own are bound by memory, and eight waves a list have more on its way (256 of them 236 and 209).
    const uint64_t units = (uint64_t)b.rows * kv.n_kv;
    if (a.g <= 8 && b.row_start && units >= ROW_UNITS && b.rows >= (uint64_t)b.n_seqs * ROW_ROWS) {
        if (!kv_launch_fits(units + 64, 64)) return hipErrorInvalidValue;
        a.units = (uint32_t)units;
        return launch_attend_rows(a, call.bf16, rules, s);
    }
    unsigned grid;
    const hipError_t e = spread(a, sc, false, true, std::min<uint64_t>((uint64_t)chosen.count << a.span_shift, (uint64_t)b.max_pages << kv.shift), 256 * split_places((int)kv.d / 32), &grid);
    return e != hipSuccess ? e : go<CHOSEN>(a, call.bf16, rules, grid, s);
}

}  // namespace oxhip
