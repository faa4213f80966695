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

// Logits of a row that a workgroup takes, and its threads. (Slices of 2048 by 256 threads, 4096 by 256, 4096 by 512 and 8192 by 1024: 64 rows of 151936 bf16
// with 2000 tokens of history 26.4, 28.0, 25.8 and 27.3 us a call, nine rows of 32003 with 9000 tokens 19.9, 21.4, 15.3 and 15.3, one of 128256 13.2 each.)
constexpr uint32_t LOGIT_SLICE = 4096, LOGIT_THREADS = 512;
// What a stream's scratch holds of rows and of their slices' best.
constexpr size_t LOGIT_NEXT_ROWS = 16384, LOGIT_NEXT_SLICES = (size_t)1 << 21;
inline size_t logit_slices(size_t vocab) { return (vocab + LOGIT_SLICE - 1) / LOGIT_SLICE; }

}  // namespace oxhip
