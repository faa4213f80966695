// What the kernels of the key / value cache share (kv_cache.hip, attend.hip): the views that a launch gets, finding a workgroup's sequence.
#pragma once
#include "internal.hpp"
#include "kv_plan.hpp"

namespace oxhip {

struct KvView {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    uint32_t n_pages, n_kv, d, shift;  // a page has 1 << shift blocks
};
struct KvBatchView {
    const int32_t *row_start, *kv_len, *pages;
    uint32_t n_seqs, rows, max_pages;
};
struct RopeView {
    const float* table;
    uint32_t n_pos, half;  // positions, pairs per head
    uint32_t interleaved;
};

__device__ __forceinline__ KvSeq kv_seq(const KvBatchView& b, int32_t s, uint32_t shift) {
    return kv_part(s, b.row_start ? b.row_start[s] : s, b.row_start ? b.row_start[s + 1] : s + 1, b.kv_len[s], b.rows, b.max_pages, shift);
}
// The sequence that has place w (kv_first_place with `scale` entries to a row), by one wave: the last s with its first place at most w. Up to
// 64 sequences take one request, up to 4096 two.
__device__ __forceinline__ int32_t kv_find(const KvBatchView& b, uint64_t w, uint32_t scale, uint32_t unit, uint32_t more) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0, n = b.n_seqs;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, s = base + lane * step;
        const bool below = lane * step < n && kv_first_place((uint64_t)(uint32_t)max(b.row_start[s], 0) * scale, s, unit, more) <= w;
        const uint64_t m = __ballot(below);
        const uint32_t at = m ? 63u - (uint32_t)__builtin_clzll(m) : 0u;
        base += at * step;
        n = min(step, n - at * step);
    }
    return (int32_t)base;
}
__device__ __forceinline__ int32_t kv_page(const KvBatchView& b, const KvView& kv, int32_t s, uint32_t block) {
    return kv_page_of(b.pages + (size_t)s * b.max_pages, b.max_pages, kv.n_pages, block, kv.shift);
}
// A block's number in the arrays of scales; its codes begin at 32 d times that.
__device__ __forceinline__ size_t kv_block_index(const KvView& kv, int32_t page, uint32_t head, uint32_t block) {
    return (((size_t)(uint32_t)page * kv.n_kv + head) << kv.shift) + (block & ((1u << kv.shift) - 1));
}

// a / b of values below 2^31, mostly small ones: by the hardware's reciprocal where its error is less than one (a lone wave takes a microsecond for
// four divisions of the general kind).
__device__ __forceinline__ uint32_t divide(uint32_t a, uint32_t b) {
    if (a >= 1u << 22) return a / b;
    const uint32_t q = (uint32_t)((float)a * __builtin_amdgcn_rcpf((float)b));
    const int32_t r = (int32_t)(a - q * b);
    return r < 0 ? q - 1 : r >= (int32_t)b ? q + 1 : q;
}

}  // namespace oxhip
