// The arguments of the draw's launch (sample.hip).
#pragma once
#include "internal.hpp"

namespace oxhip {

struct SampleArgs {
    const void* x;
    size_t stride;
    uint32_t rows, vocab;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* next;
    float* logp;    // or none
    uint32_t unit;  // weights are whole numbers, 2^unit being the largest
    uint32_t vec;
};

}  // namespace oxhip
