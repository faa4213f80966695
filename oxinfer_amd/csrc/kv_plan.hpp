// Index arithmetic of the 8-bit key / value cache (oxhip_kv_cache) and of the launches that read and fill it: no device code of its own,
// so that a test compiles it for the CPU.
#pragma once
#include <cstddef>
#include <cstdint>

#ifdef __HIP__
#define OXHIP_HD __host__ __device__ inline
#else
#define OXHIP_HD inline
#endif

namespace oxhip {

// A block holds 32 tokens of one head: 32 d codes (d a multiple of 32) and one scale. Its bytes lie so that a wave's lane finds the
// operands of two matrix instructions (16x16x32, or 32x32x16) in 16 consecutive bytes, and the 64 lanes' 16 bytes in one KiB:
//   keys    KiB ks, lane 16 g + n: the channels 32 ks + 8 g .. + 7 of token n, then those of token 16 + n
//   values  KiB vs, lane 16 g + n: the tokens 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 of channel 32 vs + n, then those of channel 32 vs + 16 + n
// (the tokens of a value operand come in the order in which the product of keys and queries leaves its results in a lane's registers).
constexpr uint32_t KV_BLOCK = 32;
constexpr uint32_t KV_MAX_D = 256;
OXHIP_HD uint32_t kv_key_offset(uint32_t token, uint32_t c) {
    return c / 32 * 1024 + c % 32 / 8 * 256 + token % 16 * 16 + token / 16 * 8 + c % 8;
}
OXHIP_HD uint32_t kv_value_offset(uint32_t token, uint32_t c) {
    return c / 32 * 1024 + token % 16 / 4 * 256 + c % 16 * 16 + c % 32 / 16 * 8 + token / 16 * 4 + token % 4;
}

// The scale of a block stays within these, so that the logarithms, quotients and sums made of scales stay within f32.
constexpr float KV_SCALE_MIN = 0x1p-60f, KV_SCALE_MAX = 0x1p60f;

// Workgroups over ragged sequences, without a pass over them first. Sequence s has n = start[s + 1] - start[s] entries; it gets the places
// from kv_first_place(start[s], s, unit, more) on. For n > 0 the next sequence's are at least n / unit + more (rounded down) further:
//   more = 1: room for the tiles of `unit` entries, ceil(n / unit)
//   more = 2: room for the blocks of `unit` tokens that n consecutive tokens touch, wherever they begin: at most (n + 2 unit - 2) / unit
OXHIP_HD uint64_t kv_first_place(uint64_t start, uint64_t s, uint32_t unit, uint32_t more) { return start / unit + more * s; }
inline uint64_t kv_places(uint64_t entries, uint64_t n_seqs, uint32_t unit, uint32_t more) { return entries / unit + more * n_seqs; }

// A launch has fewer than 2^32 threads, and 65535 workgroups at most in its second direction.
inline bool kv_launch_fits(uint64_t workgroups, uint32_t threads, uint64_t second = 1) { return workgroups <= 0xFFFFFFFFu / threads && second <= 65535; }
// The workgroups along an append's launch: the blocks that its rows touch (and heads in the second direction), or, of single tokens, four heads each.
inline uint64_t kv_append_workgroups(bool ragged, uint64_t rows, uint64_t n_seqs, uint64_t heads) {
    return ragged ? kv_places(rows, n_seqs, KV_BLOCK, 2) : (n_seqs * heads + 3) / 4;
}
// The blocks that `count` consecutive tokens touch, wherever they begin.
inline uint64_t kv_read_blocks(uint64_t count) { return (count + 2 * KV_BLOCK - 2) / KV_BLOCK; }
// Tiles of 16 entries x key heads that the attention for few rows may have.
inline uint64_t kv_units(bool ragged, uint64_t rows, uint64_t n_seqs, uint64_t g, uint64_t n_kv) {
    return (ragged ? kv_places(rows * g, n_seqs, 16, 1) : n_seqs * ((g + 15) / 16)) * n_kv;
}
// Tiles of rows of a batch, whatever sequences they are of, for one key head: of 16 / g rows where several may share a tile, of one row otherwise, of 16 heads where
// a row's group has more.
inline uint64_t kv_row_tiles(uint64_t rows, uint64_t g, bool several) {
    const uint64_t of = several && g < 16 ? 16 / g : 1;
    return (rows + of - 1) / of * ((g + 15) / 16);
}

// A sequence's part of a batch, as far as it is sound: rows of the batch, tokens that a table of max_pages pages can hold.
struct KvSeq {
    int32_t s, row0, n, len;
};
OXHIP_HD KvSeq kv_part(int32_t s, int32_t row0, int32_t row1, int32_t len, uint32_t rows, uint32_t max_pages, uint32_t shift) {
    const int64_t most = (int64_t)max_pages * KV_BLOCK << shift;
    const int32_t first = row0 < 0 ? 0 : row0, end = row1 < (int32_t)rows ? row1 : (int32_t)rows;
    return KvSeq{s, first, end > first ? end - first : 0, (int32_t)(len < 0 ? 0 : len < most ? len : most)};
}
// The page that holds a block of a sequence, by its row of the table; -1 if the table names no page of the cache.
OXHIP_HD int32_t kv_page_of(const int32_t* table, uint32_t max_pages, uint32_t n_pages, uint32_t block, uint32_t shift) {
    const uint32_t p = block >> shift;
    if (p >= max_pages) return -1;
    const int32_t id = table[p];
    return id >= 0 && (uint32_t)id < n_pages ? id : -1;
}

// The blocks that a tile of query rows reads: those of the prefix (they see keys 0 .. prefix - 1), then those of [lo, hi), less the prefix's.
struct KvSpan {
    uint32_t pre, lo, count;  // blocks of the prefix; first block behind them; all blocks
};
OXHIP_HD KvSpan kv_span(int64_t prefix, int64_t lo, int64_t hi) {
    KvSpan s;
    s.pre = (uint32_t)((prefix + KV_BLOCK - 1) / KV_BLOCK);
    const uint32_t first = lo > 0 ? (uint32_t)(lo / KV_BLOCK) : 0u, end = hi > 0 ? (uint32_t)((hi + KV_BLOCK - 1) / KV_BLOCK) : 0u;
    s.lo = first > s.pre ? first : s.pre;
    s.count = s.pre + (hi > lo && end > s.lo ? end - s.lo : 0u);
    return s;
}
// The same of the blocks from `base` on alone: those of the prefix from there on are the first `pre` of them.
OXHIP_HD KvSpan kv_span_from(uint32_t base, int64_t prefix, int64_t lo, int64_t hi) {
    KvSpan s = kv_span(prefix, lo, hi);
    const uint32_t end = s.count > s.pre ? s.lo + (s.count - s.pre) : 0u, first = s.lo > base ? s.lo : base;
    s.pre = s.pre > base ? s.pre - base : 0u;
    s.lo = first;
    s.count = s.pre + (end > first ? end - first : 0u);
    return s;
}
OXHIP_HD uint32_t kv_span_block(const KvSpan& s, uint32_t i) { return i < s.pre ? i : s.lo + (i - s.pre); }

// A launch's workgroups over tiles of very different lengths: a tile of `blocks` blocks gets ceil(blocks / size) of them, size being all tiles'
// blocks over the workgroups that the chip holds, and KV_LEAST blocks at least (a tile's parts have to meet again, which takes longer than to
// read that many). A tile's blocks are here those that its sequence's last row can see; rules that go by the row are left out, and the parts
// are parts of what the tile really has. Counted in quanta of blocks, 1 unless 32 bits would not hold the sum.
constexpr uint32_t KV_LEAST = 32;
OXHIP_HD uint32_t kv_weight(const KvSeq& q, uint32_t window, int32_t prefix, uint32_t quantum) {
    const uint32_t all = ((uint32_t)q.len + KV_BLOCK - 1) / KV_BLOCK;
    uint32_t blocks = all;
    if (window && q.len - q.n >= 0 && (uint32_t)(q.len - q.n) >= window) {
        const uint32_t pre = prefix > 0 ? ((uint32_t)prefix + KV_BLOCK - 1) / KV_BLOCK : 0, out = ((uint32_t)(q.len - q.n) - window + 1) / KV_BLOCK;
        blocks = pre < out ? all - out + pre : all;
    }
    return blocks ? (quantum == 1 ? blocks : (blocks + quantum - 1) / quantum) : 1;
}
OXHIP_HD uint32_t kv_tiles(const KvSeq& q, uint32_t g) { return (uint32_t)(((uint64_t)(uint32_t)q.n * g + 15) / 16); }
// The quantum with which `tiles` tiles x heads of at most `blocks` blocks each come to less than 2^31 in all (0: none does).
inline uint32_t kv_quantum(uint64_t tiles, uint64_t blocks) {
    for (uint64_t q = 1; q < ((uint64_t)1 << 31); q *= 2)
        if (tiles < ((uint64_t)1 << 30) && tiles * ((blocks + q - 1) / q) < ((uint64_t)1 << 31)) return (uint32_t)q;
    return 0;
}

}  // namespace oxhip
