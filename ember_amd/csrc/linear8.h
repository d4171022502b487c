// linear8.h -- what the products of 8-bit matrices are called with (not part of
// the public ABI).
#pragma once

#include "rows8.h"

namespace ember {

struct Linear8Args {
    Rows8 a, w;  // n x k and m x k; a gated layer's w is 2m x k, the gate's rows first
    const float *bias, *residual;
    float *out;   // n x m
    Rows8 h;      // a gated layer's output
    float *part;  // sums of parts of k (splits, n, m), or null
    int n, m, act;
    int chunk;    // groups of k to a part
    int aligned;  // out's and residual's rows can be moved 16 bytes at a time
};

}  // namespace ember
