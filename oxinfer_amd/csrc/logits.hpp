// The arguments of the logits' launch (logits.hip).
#pragma once
#include "internal.hpp"

namespace oxhip {

struct LogitArgs {
    const void* x;
    void* out;      // or none
    int32_t* next;  // or none
    size_t x_stride, out_stride;
    uint32_t rows, vocab;
    const int32_t *history, *history_len, *prompt_len;
    size_t history_stride;
    const float *repetition, *presence, *frequency;
    const int32_t *bias_start, *bias_id;
    const float* bias;
    uint32_t n_bias, n_allowed;
    const uint32_t* allowed;
    size_t allowed_stride;  // words
    const int32_t* allowed_row;
    uint64_t* best;      // one per row and slice
    uint32_t* counters;  // one per row, zero between launches
    uint32_t slices, vec;
};

// Logits of a row that a workgroup takes.
inline uint32_t logit_slice(size_t rows, size_t vocab) { return rows * ((vocab + 4095) / 4096) >= 256 ? 4096 : 2048; }
inline size_t logit_slices(size_t rows, size_t vocab) { return (vocab + logit_slice(rows, vocab) - 1) / logit_slice(rows, vocab); }

}  // namespace oxhip
