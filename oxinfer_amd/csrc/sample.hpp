// The arguments of the draw's launches (sample.hip).
#pragma once
#include "internal.hpp"

namespace oxhip {

// Logits of a row that a workgroup takes, eight of each thread; slices that a row's sums are kept of.
constexpr uint32_t SAMPLE_SLICE = 4096, SAMPLE_THREADS = 512, SAMPLE_SLICES = 256;
// Steps of weight, a quarter of an octave each, that the first pass counts tokens by: past them a weight is 0.
constexpr uint32_t SAMPLE_STEPS = 192;

// What the first pass finds out about a row: see sample_scan_kernel.
struct SampleRow {
    float top, low, high;  // the largest logit; steps of the tokens among which a limit falls
    uint32_t flags;
};
// What the second pass finds out about a slice.
struct SampleSlice {
    unsigned long long all, above, kept;  // weights: of all its tokens, of those above the limit's steps, of those of these that min-p leaves
    uint16_t n_above, n;                  // tokens above; tokens that are set apart
    uint32_t with;                        // those above are among these
};

struct SampleArgs {
    const void* x;
    size_t stride;
    uint32_t rows, vocab;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* next;
    float* logp;    // or none
    uint32_t unit;  // weights are whole numbers, 2^unit being the largest
    uint32_t slices, vec, row0;
    // scratch
    uint32_t* step;              // [rows][slices][SAMPLE_STEPS]: numbers of tokens, or (f32) their weights
    float* best;                 // [rows][slices]
    SampleRow* row;              // [rows]
    SampleSlice* slice;          // [rows][slices]
    unsigned long long* token;   // [rows][slices][room]: order_of a logit << 32 | id
    uint32_t room;
    uint32_t* counters;  // one of each row, zero between launches
};

}  // namespace oxhip
